// Rotary positions (kmi_rotary): pairs of a head's dims turned by the angle position *
// inv_freq, forward and (by the opposite angle) backward.
//
// Bound by memory: every value is read and written once, for three operations.  A thread
// owns V pairs (one 16-byte vector of each half; two adjacent vectors when interleaved) of one
// token, forms their sines and cosines once (about 45 instructions a pair, the angles in 64
// bits) and walks its share of the token's heads with them, four heads' loads in flight.
// Few tokens spread their heads over more threads instead, since nothing is gained by sharing
// angles when most of the chip idles.
#include "paged.hpp"

namespace kmi {
namespace rotary {
namespace {

struct Params {
    const void* x[2];
    void* y[2];
    int64_t xs[2][3], ys[2][3];
    int heads[2];
    int seq, d, rd;
    int64_t tokens;
    const void* positions;
    int64_t ps[2];
    int wide;  // int64 positions
    const float* freq;
    float scale;
    int inverse;
    int hg;       // threads that share a token's chunk, each with every hg-th head
    int chunks;   // of a head: rotated pairs of vectors, then copied vectors
    int tpt;      // threads of a token: hg * chunks
    int tpb;      // tokens of a workgroup
    fwd::FastDiv fd_tpt, fd_chunks;
};

template <typename T, int V>
struct Vec {
    T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
    Vec<T, V> v;
    if constexpr (V == 1)
        v.e[0] = *p;
    else
        __builtin_memcpy(&v, __builtin_assume_aligned(p, 16), 16);
    return v;
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const Vec<T, V>& v) {
    if constexpr (V == 1)
        *p = v.e[0];
    else
        __builtin_memcpy(__builtin_assume_aligned(p, 16), &v, 16);
}

constexpr int THREADS = 256;
constexpr int BATCH = 4;  // heads in flight

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(THREADS) void rotary_kernel(const Params p) {
    const int tl = fwd::fdiv(threadIdx.x, p.fd_tpt);
    if (tl >= p.tpb) return;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * p.tpb + tl;
    if (t >= p.tokens) return;
    const int rem = threadIdx.x - tl * p.tpt;
    const int hg = fwd::fdiv(rem, p.fd_chunks), c = rem - hg * p.chunks;
    const int64_t b = t / p.seq, s = t - b * p.seq;
    const int nrot = p.rd / (2 * V);
    const bool rot = c < nrot;
    // First and second vector of the chunk (a copied chunk has one).
    const int lo = rot ? (INTER ? 2 * V * c : V * c) : p.rd + V * (c - nrot);
    const int hi = rot ? (INTER ? lo + V : lo + p.rd / 2) : lo;
    const int heads = p.heads[0] + p.heads[1];
    auto src = [&](int h) {
        const int w = h >= p.heads[0];
        return static_cast<const T*>(p.x[w]) + b * p.xs[w][0] + (h - (w ? p.heads[0] : 0)) * p.xs[w][1] + s * p.xs[w][2];
    };
    auto dst = [&](int h) {
        const int w = h >= p.heads[0];
        return static_cast<T*>(p.y[w]) + b * p.ys[w][0] + (h - (w ? p.heads[0] : 0)) * p.ys[w][1] + s * p.ys[w][2];
    };
    Vec<T, V> a[BATCH], z[BATCH];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const int h = h0 + j * p.hg;
            if (h < heads) {
                const T* x = src(h);
                a[j] = load<T, V>(x + lo);
                if (rot) z[j] = load<T, V>(x + hi);
            }
        }
    };
    fetch(hg);  // (before the angles, whose latency it hides)
    float cs[V], sn[V];
    if (rot) {
        const int64_t at = b * p.ps[0] + s * p.ps[1];
        const double pos = p.wide ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                                  : static_cast<double>(static_cast<const int32_t*>(p.positions)[at]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            paged::turn(pos, p.freq[V * c + i], cs[i], sn[i]);
            cs[i] *= p.scale;
            sn[i] *= p.inverse ? -p.scale : p.scale;
        }
    }
    for (int h0 = hg; h0 < heads; h0 += BATCH * p.hg) {
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const int h = h0 + j * p.hg;
            if (h >= heads) break;
            T* y = dst(h);
            if (!rot) {
                store<T, V>(y + lo, a[j]);
                continue;
            }
            Vec<T, V> u, w;
            if constexpr (INTER && V > 1) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    Vec<T, V>& in = i < V / 2 ? a[j] : z[j];
                    Vec<T, V>& out = i < V / 2 ? u : w;
                    const int k = 2 * (i % (V / 2));
                    const float x1 = to_f32(in.e[k]), x2 = to_f32(in.e[k + 1]);
                    out.e[k] = from_f32<T>(x1 * cs[i] - x2 * sn[i]);
                    out.e[k + 1] = from_f32<T>(x2 * cs[i] + x1 * sn[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float x1 = to_f32(a[j].e[i]), x2 = to_f32(z[j].e[i]);
                    u.e[i] = from_f32<T>(x1 * cs[i] - x2 * sn[i]);
                    w.e[i] = from_f32<T>(x2 * cs[i] + x1 * sn[i]);
                }
            }
            store<T, V>(y + lo, u);
            store<T, V>(y + hi, w);
        }
        if (h0 + BATCH * p.hg < heads) fetch(h0 + BATCH * p.hg);
    }
}

const char* check_args(const kmi_rotary_args* a) {
    if (!a) return "null args";
    if (a->dtype != KMI_BF16 && a->dtype != KMI_F16 && a->dtype != KMI_F32) return "dtype must be BF16, F16 or F32";
    if (a->batch < 0 || a->seq < 0 || a->batch > (1 << 30) || a->seq > (1 << 30)) return "sizes out of range";
    if (a->head_dim < 1 || a->head_dim > 256) return "head_dim must be at most 256";
    if (a->rotary_dim < 2 || a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
        return "rotary_dim must be even, positive and at most head_dim";
    if (a->position_bits != 32 && a->position_bits != 64) return "position_bits must be 32 or 64";
    if (!a->x[0] || !a->y[0] || !a->positions || !a->inv_freq) return "null x, y, positions or inv_freq";
    if (a->x[1] && !a->y[1]) return "null second y";
    for (int w = 0; w < (a->x[1] ? 2 : 1); ++w)
        if (a->heads[w] < 1 || a->heads[w] > 65536) return "heads out of range";
    return nullptr;
}

template <typename T>
hipError_t launch(const kmi_rotary_args* a, hipStream_t stream) {
    constexpr int W = 16 / sizeof(T);
    Params p{};
    const int n = a->x[1] ? 2 : 1;
    // Whole 16-byte vectors, or element by element.
    bool vec = a->rotary_dim % (2 * W) == 0 && a->head_dim % W == 0;
    for (int w = 0; w < n; ++w) {
        p.x[w] = a->x[w];
        p.y[w] = a->y[w];
        p.heads[w] = static_cast<int>(a->heads[w]);
        vec = vec && reinterpret_cast<uintptr_t>(a->x[w]) % 16 == 0 && reinterpret_cast<uintptr_t>(a->y[w]) % 16 == 0;
        for (int i = 0; i < 3; ++i) {
            p.xs[w][i] = a->x_stride[w][i];
            p.ys[w][i] = a->y_stride[w][i];
            vec = vec && p.xs[w][i] % W == 0 && p.ys[w][i] % W == 0;
        }
    }
    p.seq = static_cast<int>(a->seq);
    p.d = static_cast<int>(a->head_dim);
    p.rd = static_cast<int>(a->rotary_dim);
    p.tokens = a->batch * a->seq;
    p.positions = a->positions;
    p.ps[0] = a->position_stride[0];
    p.ps[1] = a->position_stride[1];
    p.wide = a->position_bits == 64;
    p.freq = a->inv_freq;
    p.scale = static_cast<float>(a->scale);
    p.inverse = a->inverse ? 1 : 0;
    const int v = vec ? W : 1;
    p.chunks = p.rd / (2 * v) + (p.d - p.rd) / v;
    // Threads per token: enough for two wavefronts per SIMD over the chip when there are few
    // tokens, else one thread for all heads of a chunk.
    const int heads = p.heads[0] + p.heads[1];
    p.hg = 1;
    while (2 * p.hg * p.chunks <= THREADS && p.hg < heads && p.tokens * p.chunks * p.hg < (1 << 17)) p.hg *= 2;
    p.tpt = p.hg * p.chunks;
    p.tpb = THREADS / p.tpt;
    p.fd_tpt = fwd::fast_div(static_cast<uint32_t>(p.tpt));
    p.fd_chunks = fwd::fast_div(static_cast<uint32_t>(p.chunks));
    const dim3 grid(static_cast<unsigned>(ceil_div(p.tokens, p.tpb)));
    if (vec) {
        if (a->interleaved)
            hipLaunchKernelGGL((rotary_kernel<T, W, true>), grid, dim3(THREADS), 0, stream, p);
        else
            hipLaunchKernelGGL((rotary_kernel<T, W, false>), grid, dim3(THREADS), 0, stream, p);
    } else if (a->interleaved) {
        hipLaunchKernelGGL((rotary_kernel<T, 1, true>), grid, dim3(THREADS), 0, stream, p);
    } else {
        hipLaunchKernelGGL((rotary_kernel<T, 1, false>), grid, dim3(THREADS), 0, stream, p);
    }
    return hipGetLastError();
}

}  // namespace
}  // namespace rotary
}  // namespace kmi

extern "C" int kmi_rotary(const kmi_rotary_args* a, void* stream) {
    using namespace kmi;
    if (const char* why = rotary::check_args(a)) return fail(KMI_EINVAL, std::string("kmi_rotary: ") + why);
    if (a->batch * a->seq == 0) return KMI_OK;
    // (At least one token a workgroup; a launch holds fewer than 2^32 threads.)
    if (a->batch * a->seq >= (int64_t{1} << 24)) return fail(KMI_EINVAL, "kmi_rotary: 2^24 tokens or more");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t err = a->dtype == KMI_BF16  ? rotary::launch<bf16>(a, s)
                           : a->dtype == KMI_F16 ? rotary::launch<f16>(a, s)
                                                 : rotary::launch<float>(a, s);
    return hip_status(err, "kmi_rotary");
}
