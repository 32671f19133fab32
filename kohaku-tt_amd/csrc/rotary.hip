// Rotary positions (kmi_rotary): pairs of a head's dims turned by the angle position *
// inv_freq, forward and (by the opposite angle) backward.
//
// Bound by memory: every value is read and written once, for three operations.  A workgroup owns
// a few tokens.  Its threads first request their vectors (two of 16 bytes each, one of each half of
// a head's rotated dims), then form the tokens' sines and cosines into LDS, one pair a thread (about
// 45 instructions, the angles in 64 bits, behind the loads' latency), and then turn and store.
// Angles are so formed once per token and not per head, and no thread walks the heads one after the
// other.  Interleaved pairs lie within a vector; two adjacent vectors a thread, which leave gaps
// between a wavefront's lanes, took 43.8 us where the halves took 40.5.
//
// Measured: 4 x 4096 tokens of 16 and 8 heads x 128 (201 MB) 38.0 us, 5.3 TB/s (a large copy moves
// 5.1), interleaved 39.2; 8 tokens 2.8 us, one memory round trip behind the launch (the host's part
// of a call is 7).
#include <algorithm>

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
    int chunks;   // of a head: rotated pairs of vectors, then copied vectors
    int per;      // items (pairs of vectors, copied vectors) of a token: heads * chunks
    int tpb;      // tokens of a workgroup
    fwd::FastDiv fd_seq, fd_half, fd_chunks, fd_per;
};

template <typename T, int V>
struct Vec {
    T e[V];
};

template <typename T, int V, bool STREAM>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
    Vec<T, V> v;
    if constexpr (V == 1)
        v.e[0] = *p;
    else if constexpr (STREAM)
        v = __builtin_bit_cast(Vec<T, V>, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
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
constexpr int ITEMS = 4;       // of a thread, in flight together
constexpr int PAIRS = 2048;    // angles of a workgroup

template <typename T, int V, bool INTER, bool STREAM>
__global__ __launch_bounds__(THREADS) void rotary_kernel(const Params p) {
    __shared__ __align__(16) float cosine[PAIRS], sine[PAIRS];
    const int t0 = blockIdx.x * p.tpb;
    const int nt = min(p.tpb, static_cast<int>(p.tokens) - t0);
    const int half = p.rd / 2, nrot = half / V;
    const int items = nt * p.per;
    // An item's vectors and its first angle (negative: copied).
    Vec<T, V> a[ITEMS], z[ITEMS];
    T* dst[ITEMS];
    int lo[ITEMS], hi[ITEMS], at[ITEMS];
    auto fetch = [&](int base) {
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int i = base + j * THREADS + threadIdx.x;
            if (i >= items) continue;
            const int tl = fwd::fdiv(i, p.fd_per), r = i - tl * p.per;
            int h = fwd::fdiv(r, p.fd_chunks);
            const int c = r - h * p.chunks;
            const int w = h >= p.heads[0];
            h -= w ? p.heads[0] : 0;
            const int b = fwd::fdiv(t0 + tl, p.fd_seq), s = t0 + tl - b * p.seq;
            const T* x = static_cast<const T*>(p.x[w]) + b * p.xs[w][0] + h * p.xs[w][1] + s * p.xs[w][2];
            dst[j] = static_cast<T*>(p.y[w]) + b * p.ys[w][0] + h * p.ys[w][1] + s * p.ys[w][2];
            const bool rot = c < nrot;
            lo[j] = rot ? (INTER && V == 1 ? 2 * c : V * c) : p.rd + V * (c - nrot);
            hi[j] = INTER && V == 1 ? lo[j] + 1 : lo[j] + half;
            at[j] = rot ? tl * half + (INTER && V > 1 ? V / 2 : V) * c : -1;
            a[j] = load<T, V, STREAM>(x + lo[j]);
            if (rot) z[j] = load<T, V, STREAM>(x + hi[j]);
        }
    };
    fetch(0);
    for (int i = threadIdx.x; i < nt * half; i += THREADS) {
        const int tl = fwd::fdiv(i, p.fd_half), k = i - tl * half;
        const int b = fwd::fdiv(t0 + tl, p.fd_seq), s = t0 + tl - b * p.seq;
        const int64_t n = b * p.ps[0] + s * p.ps[1];
        const double pos = p.wide ? static_cast<double>(static_cast<const int64_t*>(p.positions)[n])
                                  : static_cast<double>(static_cast<const int32_t*>(p.positions)[n]);
        float c, sn;
        paged::turn(pos, p.freq[k], c, sn);
        cosine[i] = c * p.scale;
        sine[i] = sn * (p.inverse ? -p.scale : p.scale);
    }
    __syncthreads();
    for (int base = 0;;) {
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            if (base + j * THREADS + static_cast<int>(threadIdx.x) >= items) break;
            if (at[j] < 0) {
                store<T, V>(dst[j] + lo[j], a[j]);
                continue;
            }
            float cs[V], sn[V];
            if constexpr (INTER && V > 1) {
                // Pairs lie within a vector: the angles of the two vectors are half of all apart.
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int k = at[j] + i * (half / 2);
                    __builtin_memcpy(cs + i * (V / 2), __builtin_assume_aligned(cosine + k, V * 2), V * 2);
                    __builtin_memcpy(sn + i * (V / 2), __builtin_assume_aligned(sine + k, V * 2), V * 2);
                }
            } else {
                __builtin_memcpy(cs, __builtin_assume_aligned(cosine + at[j], V * 4), V * 4);
                __builtin_memcpy(sn, __builtin_assume_aligned(sine + at[j], V * 4), V * 4);
            }
            Vec<T, V> u, w;
            if constexpr (INTER && V > 1) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const Vec<T, V>& in = i < V / 2 ? a[j] : z[j];
                    Vec<T, V>& out = i < V / 2 ? u : w;
                    const int k = 2 * (i % (V / 2));
                    float y1, y2;
                    paged::turned(to_f32(in.e[k]), to_f32(in.e[k + 1]), cs[i], sn[i], y1, y2);
                    out.e[k] = from_f32<T>(y1);
                    out.e[k + 1] = from_f32<T>(y2);
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float y1, y2;
                    paged::turned(to_f32(a[j].e[i]), to_f32(z[j].e[i]), cs[i], sn[i], y1, y2);
                    u.e[i] = from_f32<T>(y1);
                    w.e[i] = from_f32<T>(y2);
                }
            }
            store<T, V>(dst[j] + lo[j], u);
            store<T, V>(dst[j] + hi[j], w);
        }
        base += ITEMS * THREADS;
        if (base >= items) break;
        fetch(base);
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
    p.per = (p.heads[0] + p.heads[1]) * p.chunks;
    // Tokens of a workgroup: a batch of items a thread, unless few tokens leave CUs idle.
    const int64_t fill = std::min<int64_t>(ITEMS * THREADS / p.per, PAIRS / (p.rd / 2));
    p.tpb = static_cast<int>(std::max<int64_t>(1, std::min(fill, p.tokens / 1024)));
    p.fd_seq = fwd::fast_div(static_cast<uint32_t>(p.seq));
    p.fd_half = fwd::fast_div(static_cast<uint32_t>(p.rd / 2));
    p.fd_chunks = fwd::fast_div(static_cast<uint32_t>(p.chunks));
    p.fd_per = fwd::fast_div(static_cast<uint32_t>(p.per));
    const dim3 grid(static_cast<unsigned>(ceil_div(p.tokens, p.tpb)));
    const bool past = p.tokens * (p.heads[0] + p.heads[1]) * p.d * static_cast<int64_t>(sizeof(T)) >= paged::kStreamBytes;
    auto enqueue = [&](void (*kernel)(Params)) { hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, stream, p); };
    if (vec && past)
        enqueue(a->interleaved ? rotary_kernel<T, W, true, true> : rotary_kernel<T, W, false, true>);
    else if (vec)
        enqueue(a->interleaved ? rotary_kernel<T, W, true, false> : rotary_kernel<T, W, false, false>);
    else
        enqueue(a->interleaved ? rotary_kernel<T, 1, true, false> : rotary_kernel<T, 1, false, false>);
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
