// The paged cache: its host checks, kmi_paged_append and kmi_paged_read.
//
// Append: a thread owns a chunk of dims of one token, turns its share of the token's query
// and key heads with sines and cosines formed once, and copies or quantises values.  16-bit
// rows move as 16-byte vectors (bound by memory); a 4-bit row's groups of 32 dims lie in four
// neighbouring lanes, eight dims each, which agree on the group's exponent by two lane
// exchanges.  Rotated keys are formed in 64 bits there: a value that 32 bits put on the wrong
// side of a border between two codes would come out a whole step off.
//
// Read: one 16-byte store per thread, its row found through the table.
#include "paged.hpp"

namespace kmi {
namespace paged {

const char* check_cache(const kmi_paged_cache& c, bool uses_tokens) {
    if (c.dtype != KMI_BF16 && c.dtype != KMI_F16) return "dtype must be BF16 or F16";
    if (c.bits != 16 && c.bits != 4) return "bits must be 16 or 4";
    const int step = c.bits == 16 ? 8 : 32;
    for (const int64_t d : {c.head_dim, c.head_dim_v})
        if (d < step || d > 256 || d % step)
            return c.bits == 16 ? "head dims must be multiples of 8 up to 256"
                                : "head dims of a 4-bit cache must be multiples of 32 up to 256";
    if (c.pages < 1 || c.pages > INT32_MAX) return "pages must be positive";
    if (c.page_size < 16 || c.page_size % 16 || c.page_size > (1 << 20)) return "page_size must be a multiple of 16";
    if (c.heads_kv < 1 || c.heads_kv > 65536) return "heads_kv out of range";
    if (!c.k || !c.v || !c.block_table || !c.key_lengths) return "null k, v, block_table or key_lengths";
    if (c.bits == 4 && (!c.k_scale || !c.v_scale)) return "a 4-bit cache needs k_scale and v_scale";
    for (const void* ptr : {c.k, c.v})
        if (reinterpret_cast<uintptr_t>(ptr) % 16) return "k and v must be 16-byte aligned";
    const int unit = c.bits == 16 ? 8 : 16;
    for (int i = 0; i < 3; ++i) {
        if (c.k_stride[i] % unit || c.v_stride[i] % unit)
            return c.bits == 16 ? "cache strides must be multiples of 8 elements"
                                : "code strides must be multiples of 16 bytes";
        if (c.k_stride[i] < 0 || c.v_stride[i] < 0) return "cache strides must not be negative";
        if (c.bits == 4 && (c.k_scale_stride[i] < 0 || c.v_scale_stride[i] < 0))
            return "cache strides must not be negative";
    }
    // (16 rows of a page are addressed with 32-bit offsets.)
    if (c.k_stride[2] > (1 << 24) || c.v_stride[2] > (1 << 24) ||
        (c.bits == 4 && (c.k_scale_stride[2] > (1 << 24) || c.v_scale_stride[2] > (1 << 24))))
        return "cache row strides must be at most 2^24";
    if (c.batch < 0 || c.batch > (1 << 24)) return "batch out of range";
    if (c.table_width < 0 || (c.table_width > 1 && c.table_stride < 0)) return "bad block_table strides";
    if (c.table_width > (int64_t{1} << 30) / c.page_size) return "block_table holds more than 2^30 keys a sequence";
    if (uses_tokens) {
        if (c.tokens < 0 || c.tokens > (1 << 24)) return "tokens out of range";
        if (!c.cu_seqlens && c.tokens != c.batch) return "without cu_seqlens there is one token per sequence";
    }
    return nullptr;
}

Cache device_cache(const kmi_paged_cache& c) {
    Cache d{};
    d.k = static_cast<char*>(c.k);
    d.v = static_cast<char*>(c.v);
    d.ksc = static_cast<uint8_t*>(c.k_scale);
    d.vsc = static_cast<uint8_t*>(c.v_scale);
    const int64_t es = c.bits == 16 ? 2 : 1;
    for (int i = 0; i < 3; ++i) {
        d.ks[i] = c.k_stride[i] * es;
        d.vs[i] = c.v_stride[i] * es;
        d.kss[i] = c.k_scale_stride[i];
        d.vss[i] = c.v_scale_stride[i];
    }
    d.table = c.block_table;
    d.table_stride = c.table_stride;
    d.klen = c.key_lengths;
    d.cu = c.cu_seqlens;
    d.pages = static_cast<int>(c.pages);
    d.page = static_cast<int>(c.page_size);
    d.hkv = static_cast<int>(c.heads_kv);
    d.d = static_cast<int>(c.head_dim);
    d.dv = static_cast<int>(c.head_dim_v);
    d.batch = static_cast<int>(c.batch);
    d.tokens = static_cast<int>(c.tokens);
    d.capacity = static_cast<int>(c.table_width * c.page_size);
    d.fd_page = fwd::fast_div(static_cast<uint32_t>(d.page));
    return d;
}

namespace {

constexpr int THREADS = 256;
constexpr int MOST = 512;  // threads of an append whose token needs more than 256

struct AppendParams {
    Cache c;
    const void* k;
    const void* v;
    const void* q;
    void* qo;
    int64_t ks[2], vs[2], qs[2], qos[2];  // elements: token, head
    int hq, rd, inter;
    const float* freq;
    double scale;
    int hg, nk, nv;  // threads that share a chunk's heads; chunks of a key (query) row, of a value row
    int tpt, tpb;
    fwd::FastDiv fd_tpt, fd_chunks;
};

template <typename T>
struct Vec8;
template <>
struct Vec8<bf16> {
    typedef bf16x8 type;
};
template <>
struct Vec8<f16> {
    typedef f16x8 type;
};
template <typename T>
using V8 = typename Vec8<T>::type;

// ---------------------------------------------------------------- 16 bits

// Key chunks of VW dims a half (both vectors of a rotated pair in one thread), value chunks of
// eight dims.  VW is 8, or 1 where the rotated dims are no whole pairs of vectors.
template <typename T, int VW>
__global__ __launch_bounds__(MOST) void append_kernel(const AppendParams p) {
    const int tl = fwd::fdiv(threadIdx.x, p.fd_tpt);
    const int t = blockIdx.x * p.tpb + tl;
    if (tl >= p.tpb || t >= p.c.tokens) return;
    const int rem = threadIdx.x - tl * p.tpt;
    const int hg = fwd::fdiv(rem, p.fd_chunks);
    int c = rem - hg * (p.nk + p.nv);
    const Place at = place_of(p.c, t);
    int row = 0;
    const int page = at.pos >= 0 ? page_of(p.c, at.seq, at.pos, row) : -1;
    if (c >= p.nk) {
        c -= p.nk;
        if (page < 0) return;
        for (int h = hg; h < p.c.hkv; h += p.hg) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const T*>(p.v) + t * p.vs[0] + h * p.vs[1] + 8 * c);
            *reinterpret_cast<u32x4*>(p.c.v + page * p.c.vs[0] + h * p.c.vs[1] + row * p.c.vs[2] + 16 * c) = x;
        }
        return;
    }
    const int nrot = p.rd / (2 * VW);
    const bool rot = c < nrot;
    const int lo = rot ? (p.inter ? 2 * VW * c : VW * c) : p.rd + VW * (c - nrot);
    const int hi = rot ? (p.inter ? lo + VW : lo + p.rd / 2) : lo;
    float cs[VW], sn[VW];
    if (rot) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            turn(static_cast<double>(at.pos), p.freq[VW * c + i], cs[i], sn[i]);
            cs[i] *= static_cast<float>(p.scale);
            sn[i] *= static_cast<float>(p.scale);
        }
    }
    for (int h = hg; h < p.hq + p.c.hkv; h += p.hg) {
        const bool query = h < p.hq;
        const T* src;
        T* dst;
        if (query) {
            src = static_cast<const T*>(p.q) + t * p.qs[0] + h * p.qs[1];
            dst = static_cast<T*>(p.qo) + t * p.qos[0] + h * p.qos[1];
        } else {
            if (page < 0) return;
            const int hk = h - p.hq;
            src = static_cast<const T*>(p.k) + t * p.ks[0] + hk * p.ks[1];
            dst = reinterpret_cast<T*>(p.c.k + page * p.c.ks[0] + hk * p.c.ks[1] + row * p.c.ks[2]);
        }
        T a[VW], z[VW];
        __builtin_memcpy(a, __builtin_assume_aligned(src + lo, VW * 2), VW * 2);
        __builtin_memcpy(z, __builtin_assume_aligned(src + hi, VW * 2), VW * 2);
        T u[VW], w[VW];
        if (query && at.pos < 0) {
            // A row of no sequence (or past the cache).
#pragma unroll
            for (int i = 0; i < VW; ++i) u[i] = w[i] = static_cast<T>(0.f);
        } else if (!rot) {
#pragma unroll
            for (int i = 0; i < VW; ++i) u[i] = w[i] = a[i];
        } else if (VW > 1 && p.inter) {
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const T* in = i < VW / 2 ? a : z;
                T* out = i < VW / 2 ? u : w;
                const int e = VW > 1 ? 2 * (i % (VW / 2 > 0 ? VW / 2 : 1)) : 0;
                const float x1 = to_f32(in[e]), x2 = to_f32(in[e + (VW > 1)]);
                out[e] = from_f32<T>(x1 * cs[i] - x2 * sn[i]);
                out[e + (VW > 1)] = from_f32<T>(x2 * cs[i] + x1 * sn[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                const float x1 = to_f32(a[i]), x2 = to_f32(z[i]);
                u[i] = from_f32<T>(x1 * cs[i] - x2 * sn[i]);
                w[i] = from_f32<T>(x2 * cs[i] + x1 * sn[i]);
            }
        }
        __builtin_memcpy(__builtin_assume_aligned(dst + lo, VW * 2), u, VW * 2);
        if (rot) __builtin_memcpy(__builtin_assume_aligned(dst + hi, VW * 2), w, VW * 2);
    }
}

// ---------------------------------------------------------------- 4 bits

// The largest of a value over the four lanes of a group.
__device__ __forceinline__ int max_of_four(int v) {
    v = max(v, __shfl_xor(v, 1, kWave));
    return max(v, __shfl_xor(v, 2, kWave));
}

// Eight values of a group of 32 (four neighbouring lanes hold it) as codes; `exponent`: the
// group's scale byte.  The codes are those nearest to y 2^-e in exact arithmetic: the product
// is exact in 64 bits and rounds to 32 toward zero with the last bit set where that drops
// anything, which no border between two codes has (nearest rounding could land on one).
__device__ __forceinline__ uint32_t quantise8(const double (&y)[8], int& exponent) {
    int top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, static_cast<int>(__double2hiint(y[i]) & 0x7fffffff));
    top = max_of_four(top);
    const int e64 = top >> 20;
    const int e = e64 == 0 ? -127 : min(max(e64 - 1023 - 2, -126), 127);
    exponent = e64 == 0x7ff ? 255 : e + 127;
    const double inv = __hiloint2double((1023 - e) << 20, 0);
    uint32_t codes = 0;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double s = y[i] * inv;
        f[i] = static_cast<float>(s);
        const double back = static_cast<double>(f[i]);
        if (back != s) {
            const uint32_t bits = __float_as_uint(f[i]);
            f[i] = __uint_as_float((fabs(back) > fabs(s) ? bits - 1 : bits) | 1u);
        }
    }
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[0], f[1], 1.f, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], 1.f, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], 1.f, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], 1.f, 3);
    return codes;
}

// Chunks of eight dims; head dims are whole groups, so a group's four chunks are four
// neighbouring lanes that run the same heads.
template <typename T>
__global__ __launch_bounds__(THREADS) void append4_kernel(const AppendParams p) {
    const int tl = fwd::fdiv(threadIdx.x, p.fd_tpt);
    const int t = blockIdx.x * p.tpb + tl;
    if (tl >= p.tpb || t >= p.c.tokens) return;
    const int rem = threadIdx.x - tl * p.tpt;
    const int hg = fwd::fdiv(rem, p.fd_chunks);
    int c = rem - hg * (p.nk + p.nv);
    const Place at = place_of(p.c, t);
    int row = 0;
    const int page = at.pos >= 0 ? page_of(p.c, at.seq, at.pos, row) : -1;
    typedef V8<T> v8;
    double y[8];
    int exponent;
    if (c >= p.nk) {
        c -= p.nk;
        if (page < 0) return;
        for (int h = hg; h < p.c.hkv; h += p.hg) {
            const v8 x = *reinterpret_cast<const v8*>(static_cast<const T*>(p.v) + t * p.vs[0] + h * p.vs[1] + 8 * c);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = static_cast<double>(to_f32(x[i]));
            const uint32_t codes = quantise8(y, exponent);
            *reinterpret_cast<uint32_t*>(p.c.v + page * p.c.vs[0] + h * p.c.vs[1] + row * p.c.vs[2] + 4 * c) = codes;
            if ((c & 3) == 0)
                p.c.vsc[page * p.c.vss[0] + h * p.c.vss[1] + row * p.c.vss[2] + (c >> 2)] = static_cast<uint8_t>(exponent);
        }
        return;
    }
    // Dim d = 8 c + i: its value times cs[i] plus its partner's times sn[i].
    const int half = p.rd / 2, d0 = 8 * c;
    double cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        cs[i] = 1.0;
        sn[i] = 0.0;
        if (d < p.rd) {
            const bool first = p.inter ? (d & 1) == 0 : d < half;
            // (An interleaved pair's angle is formed once.)
            if (p.inter && !first && i > 0) {
                cs[i] = cs[i - 1];
                sn[i] = -sn[i - 1];
                continue;
            }
            turn(static_cast<double>(at.pos), p.freq[p.inter ? d >> 1 : (first ? d : d - half)], cs[i], sn[i]);
            cs[i] *= p.scale;
            sn[i] *= first ? -p.scale : p.scale;
        }
    }
    // Half layout: whole partner vectors where a half is a number of chunks.
    const bool whole = half % 8 == 0;
    for (int h = hg; h < p.hq + p.c.hkv; h += p.hg) {
        const bool query = h < p.hq;
        if (!query && page < 0) return;
        const T* src = query ? static_cast<const T*>(p.q) + t * p.qs[0] + h * p.qs[1]
                             : static_cast<const T*>(p.k) + t * p.ks[0] + (h - p.hq) * p.ks[1];
        const v8 x = *reinterpret_cast<const v8*>(src + d0);
        v8 z = x;
        if (p.inter) {
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = x[i ^ 1];
        } else if (d0 < p.rd) {
            if (whole) {
                z = *reinterpret_cast<const v8*>(src + (d0 < half ? d0 + half : d0 - half));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = d0 + i;
                    if (d < p.rd) z[i] = src[d < half ? d + half : d - half];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double own = static_cast<double>(to_f32(x[i]));
            y[i] = d0 + i < p.rd ? own * cs[i] + static_cast<double>(to_f32(z[i])) * sn[i] : own;
        }
        if (query) {
            v8 w;
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = from_f32<T>(at.pos < 0 ? 0.f : static_cast<float>(y[i]));
            *reinterpret_cast<v8*>(static_cast<T*>(p.qo) + t * p.qos[0] + h * p.qos[1] + d0) = w;
        } else {
            const uint32_t codes = quantise8(y, exponent);
            const int hk = h - p.hq;
            *reinterpret_cast<uint32_t*>(p.c.k + page * p.c.ks[0] + hk * p.c.ks[1] + row * p.c.ks[2] + 4 * c) = codes;
            if ((c & 3) == 0)
                p.c.ksc[page * p.c.kss[0] + hk * p.c.kss[1] + row * p.c.kss[2] + (c >> 2)] = static_cast<uint8_t>(exponent);
        }
    }
}

const char* check_append(const kmi_paged_append_args* a) {
    if (!a) return "null args";
    if (const char* why = check_cache(a->cache, true)) return why;
    if (!a->k || !a->v) return "null k or v";
    if (a->rotary_dim != 0) {
        if (a->rotary_dim < 2 || a->rotary_dim % 2 || a->rotary_dim > a->cache.head_dim)
            return "rotary_dim must be even and at most head_dim";
        if (!a->inv_freq) return "rotary_dim without inv_freq";
    }
    if (a->q) {
        if (a->rotary_dim == 0) return "q is taken to be rotated: it needs rotary_dim";
        if (!a->q_out) return "q without q_out";
        if (a->heads_q < 1 || a->heads_q > 65536) return "heads_q out of range";
    }
    for (const void* ptr : {a->k, a->v, a->q, static_cast<const void*>(a->q ? a->q_out : nullptr)})
        if (reinterpret_cast<uintptr_t>(ptr) % 16) return "k, v, q and q_out must be 16-byte aligned";
    for (int i = 0; i < 2; ++i)
        if (a->k_stride[i] % 8 || a->v_stride[i] % 8 || (a->q && (a->q_stride[i] % 8 || a->q_out_stride[i] % 8)))
            return "strides must be multiples of 8 elements";
    return nullptr;
}

template <typename T>
hipError_t launch_append(const kmi_paged_append_args* a, hipStream_t stream) {
    AppendParams p{};
    p.c = device_cache(a->cache);
    p.k = a->k;
    p.v = a->v;
    p.q = a->q;
    p.qo = a->q_out;
    for (int i = 0; i < 2; ++i) {
        p.ks[i] = a->k_stride[i];
        p.vs[i] = a->v_stride[i];
        p.qs[i] = a->q_stride[i];
        p.qos[i] = a->q_out_stride[i];
    }
    p.hq = a->q ? static_cast<int>(a->heads_q) : 0;
    p.rd = static_cast<int>(a->rotary_dim);
    p.inter = a->interleaved ? 1 : 0;
    p.freq = a->inv_freq;
    p.scale = a->rotary_scale;
    const int64_t tokens = a->cache.tokens;
    const bool four = a->cache.bits == 4;
    const int vw = four ? 8 : (p.rd % 16 == 0 ? 8 : 1);
    p.nk = four ? p.c.d / 8 : p.rd / (2 * vw) + (p.c.d - p.rd) / vw;
    p.nv = p.c.dv / 8;
    // Threads of a token: as in kmi_rotary, more of them where tokens are few.
    const int heads = p.hq + p.c.hkv, per = p.nk + p.nv;
    p.hg = 1;
    while (2 * p.hg * per <= THREADS && p.hg < heads && tokens * per * p.hg < (1 << 17)) p.hg *= 2;
    p.tpt = p.hg * per;
    const int threads = p.tpt <= THREADS ? THREADS : MOST;
    p.tpb = threads / p.tpt;
    p.fd_tpt = fwd::fast_div(static_cast<uint32_t>(p.tpt));
    p.fd_chunks = fwd::fast_div(static_cast<uint32_t>(per));
    const dim3 grid(static_cast<unsigned>(ceil_div(tokens, p.tpb)));
    if (four)
        hipLaunchKernelGGL((append4_kernel<T>), grid, dim3(threads), 0, stream, p);
    else if (vw == 8)
        hipLaunchKernelGGL((append_kernel<T, 8>), grid, dim3(threads), 0, stream, p);
    else
        hipLaunchKernelGGL((append_kernel<T, 1>), grid, dim3(threads), 0, stream, p);
    return hipGetLastError();
}

// ---------------------------------------------------------------- read

struct ReadParams {
    Cache c;
    void* k;
    void* v;
    int max_k, nk, nv;  // chunks of eight dims
    int blocks;         // workgroups per (sequence, K/V head)
    fwd::FastDiv fd_chunks;
};

template <typename T, bool FOUR>
__global__ __launch_bounds__(THREADS) void read_kernel(const ReadParams p) {
    const int unit = blockIdx.x / p.blocks;
    const int b = unit / p.c.hkv, h = unit - b * p.c.hkv;
    const int i = (blockIdx.x - unit * p.blocks) * THREADS + threadIdx.x;
    const int pos = fwd::fdiv(i, p.fd_chunks);
    if (pos >= p.max_k) return;
    int c = i - pos * (p.nk + p.nv);
    const bool key = c < p.nk;
    if (!key) c -= p.nk;
    u32x4 out = u32x4{0u, 0u, 0u, 0u};
    if (pos < min(max(uniform_i32(p.c.klen + b), 0), p.c.capacity)) {
        int row = 0;
        const int page = max(page_of(p.c, b, pos, row), 0);
        const int64_t* st = key ? p.c.ks : p.c.vs;
        const char* src = (key ? p.c.k : p.c.v) + page * st[0] + h * st[1] + row * st[2];
        if constexpr (FOUR) {
            const int64_t* sst = key ? p.c.kss : p.c.vss;
            const uint8_t byte = (key ? p.c.ksc : p.c.vsc)[page * sst[0] + h * sst[1] + row * sst[2] + (c >> 2)];
            const uint32_t codes = *reinterpret_cast<const uint32_t*>(src + 4 * c);
            const float s = scale_of(byte);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = fp4_pair<T>(codes, s, j);
        } else {
            out = *reinterpret_cast<const u32x4*>(src + 16 * c);
        }
    }
    char* dst = static_cast<char*>(key ? p.k : p.v);
    const int n = key ? p.nk : p.nv;
    *reinterpret_cast<u32x4*>(dst + ((static_cast<int64_t>(unit) * p.max_k + pos) * n + c) * 16) = out;
}

}  // namespace

hipError_t launch_read(const kmi_paged_cache& cache, void* k, void* v, int64_t max_k, hipStream_t stream) {
    ReadParams p{};
    p.c = device_cache(cache);
    p.k = k;
    p.v = v;
    p.max_k = static_cast<int>(max_k);
    p.nk = p.c.d / 8;
    p.nv = p.c.dv / 8;
    p.fd_chunks = fwd::fast_div(static_cast<uint32_t>(p.nk + p.nv));
    p.blocks = static_cast<int>(ceil_div(max_k * (p.nk + p.nv), THREADS));
    const dim3 grid(static_cast<unsigned>(p.blocks * cache.batch * cache.heads_kv));
    const bool bf = cache.dtype == KMI_BF16;
    if (cache.bits == 4) {
        if (bf)
            hipLaunchKernelGGL((read_kernel<bf16, true>), grid, dim3(THREADS), 0, stream, p);
        else
            hipLaunchKernelGGL((read_kernel<f16, true>), grid, dim3(THREADS), 0, stream, p);
    } else if (bf) {
        hipLaunchKernelGGL((read_kernel<bf16, false>), grid, dim3(THREADS), 0, stream, p);
    } else {
        hipLaunchKernelGGL((read_kernel<f16, false>), grid, dim3(THREADS), 0, stream, p);
    }
    return hipGetLastError();
}

// The most keys a dense copy of the cache can hold a sequence: its workgroups stay below 2^24
// (HIP's limit of 2^32 threads) and a unit's chunks below 2^31.
bool read_fits(const kmi_paged_cache& c, int64_t max_k) {
    const int64_t per = c.head_dim / 8 + c.head_dim_v / 8;
    if (max_k > ((int64_t{1} << 31) - THREADS) / per) return false;
    const int64_t units = c.batch * c.heads_kv;
    return units == 0 || ceil_div(max_k * per, THREADS) < (int64_t{1} << 24) / units;
}

}  // namespace paged
}  // namespace kmi

extern "C" int kmi_paged_append(const kmi_paged_append_args* a, void* stream) {
    using namespace kmi;
    if (const char* why = paged::check_append(a)) return fail(KMI_EINVAL, std::string("kmi_paged_append: ") + why);
    if (a->cache.tokens == 0) return KMI_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t err =
        a->cache.dtype == KMI_BF16 ? paged::launch_append<bf16>(a, s) : paged::launch_append<f16>(a, s);
    return hip_status(err, "kmi_paged_append");
}

extern "C" int kmi_paged_read(const kmi_paged_cache* c, void* k_out, void* v_out, int64_t max_k, void* stream) {
    using namespace kmi;
    if (!c) return fail(KMI_EINVAL, "kmi_paged_read: null cache");
    if (const char* why = paged::check_cache(*c, false)) return fail(KMI_EINVAL, std::string("kmi_paged_read: ") + why);
    if (!k_out || !v_out || reinterpret_cast<uintptr_t>(k_out) % 16 || reinterpret_cast<uintptr_t>(v_out) % 16)
        return fail(KMI_EINVAL, "kmi_paged_read: k_out and v_out must be 16-byte aligned and not null");
    if (max_k < 0 || !paged::read_fits(*c, max_k)) return fail(KMI_EINVAL, "kmi_paged_read: max_k out of range");
    if (max_k == 0 || c->batch == 0) return KMI_OK;
    return hip_status(paged::launch_read(*c, k_out, v_out, max_k, static_cast<hipStream_t>(stream)), "kmi_paged_read");
}
