// The paged cache: its host checks, kmi_paged_append and kmi_paged_read.
//
// Append: a workgroup owns a few tokens.  Its threads request their vectors of queries, keys and
// values, find the tokens' places (one thread a token) and form their sines and cosines into LDS
// behind those loads' latency, and then turn, quantise and store, so that nothing waits for a
// token's chain of lengths, table entry and angle but the stores.  16-bit rows move as 16-byte
// vectors (bound by memory: 8 x up to 2048 tokens of 16/8 heads x 128, 182 MB, 39.2 us, 4.6 TB/s;
// 64 single tokens 3.6 us).  A 4-bit row's groups of 32 dims lie in four neighbouring lanes, eight
// dims each, which agree on the group's exponent by two lane exchanges.  A value that 32 bits put on
// the wrong side of a border between two codes would come out a whole step off, so codes are those
// of exact arithmetic: keys are rotated in 32 bits, and once more in 64 where one of a group lies
// next to a border.
//
// Read: four 16-byte stores a thread, their rows found through the table (16 x up to 1001 keys of
// 2 x 64 4.3 us; 4 x up to 2048 keys of 8 x 128 out of 4 bits, 40 MB, 8.1 us, 4.9 TB/s).
#include <algorithm>
#include <cmath>

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
    // (A page's offset is the product of two 32-bit numbers.)
    for (const int64_t* st : {c.k_stride, c.v_stride, c.k_scale_stride, c.v_scale_stride})
        if ((c.bits == 4 || (st != c.k_scale_stride && st != c.v_scale_stride)) && st[0] > INT32_MAX / 2)
            return "cache page strides must be below 2^30";
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
constexpr int ITEMS = 4;    // of a thread, in flight together
constexpr int TOKENS = 64;  // of a workgroup, at most
constexpr int PAIRS = 1024; // angles of a workgroup, at most

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
    float slack;  // 2^-21 |scale|: what rotated values are off in 32 bits, of their pair's sizes
    int nk, nv;    // chunks of a query or key row, of a value row
    // Workgroups of queries and keys come first, those of values behind them: items (vectors, or
    // pairs of them) of a token and tokens of a workgroup for each.
    int per_qk, per_v, tpb_qk, tpb_v, blocks_qk;
    fwd::FastDiv fd_qk, fd_v, fd_nk, fd_nv, fd_half;
};

// A token's row in head 0 of the cache and its scales there, in bytes (-1: none), and its position
// (-1: none).
struct Held {
    int64_t at, scale;
    int pos, pad;
};

// The places of a workgroup's tokens and, for rotated calls, their angles' cosines and sines (F:
// float, or double, then in both), into LDS.  Tokens of one sequence (nearly every workgroup's) find
// it by scalar loads, which do not queue behind the vectors in flight, and wait for one vector load,
// the table's; a workgroup across sequences searches per token.
template <typename F>
__device__ __forceinline__ void place_tokens(const AppendParams& p, const int64_t (&st)[3], const int64_t (&ss)[3],
                                             int t0, int nt, Held* held, float* cosine,
                                             float* sine, F* cosine_f = nullptr, F* sine_f = nullptr) {
    const Cache& c = p.c;
    const int half = cosine ? p.rd / 2 : 0;
    int seq = t0, first = 0, lq = 1;
    bool one = nt == 1;
    if (c.cu) {
        int lo = 0, hi = c.batch;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (uniform_i32(c.cu + mid) <= t0)
                lo = mid;
            else
                hi = mid - 1;
        }
        seq = min(lo, max(c.batch - 1, 0));
        const int start = uniform_i32(c.cu + seq), end = uniform_i32(c.cu + min(seq + 1, c.batch));
        one = start >= 0 && start <= t0 && t0 + nt <= end && end <= c.tokens;
        first = t0 - start;
        lq = end - start;
    }
    int64_t pos0 = 0;
    if (one) pos0 = static_cast<int64_t>(uniform_i32(c.klen + seq)) - lq + first;
    if (static_cast<int>(threadIdx.x) < nt) {
        Place at{seq, -1};
        if (!one)
            at = place_of(c, t0 + threadIdx.x);
        else if (pos0 + threadIdx.x >= 0 && pos0 + threadIdx.x < c.capacity)
            at.pos = static_cast<int>(pos0 + threadIdx.x);
        Held h{-1, -1, at.pos, 0};
        int row;
        const int64_t page = at.pos >= 0 ? page_of(c, at.seq, at.pos, row) : -1;
        if (page >= 0) {
            h.at = page * st[0] + row * st[2];
            h.scale = page * ss[0] + row * ss[2];
        }
        held[threadIdx.x] = h;
    }
    if (!one) __syncthreads();  // (uniform)
    for (int i = threadIdx.x; i < nt * half; i += THREADS) {
        const int tl = fwd::fdiv(i, p.fd_half);
        const double pos = one ? static_cast<double>(pos0 + tl) : static_cast<double>(held[tl].pos);
        F cs, sn;
        turn(pos, p.freq[i - tl * half], cs, sn);
        cs *= static_cast<F>(p.scale);
        sn *= static_cast<F>(p.scale);
        cosine[i] = static_cast<float>(cs);
        sine[i] = static_cast<float>(sn);
        if constexpr (std::is_same<F, double>::value) {
            cosine_f[i] = cs;
            sine_f[i] = sn;
        }
    }
    __syncthreads();
}

// An item of a workgroup: its token, head and chunk.  Query heads come before key heads.
struct Item {
    int tl, h, c;
};
__device__ __forceinline__ Item item_of(int i, int per, fwd::FastDiv fd_per, int chunks, fwd::FastDiv fd_chunks) {
    Item m;
    m.tl = fwd::fdiv(i, fd_per);
    const int r = i - m.tl * per;
    m.h = fwd::fdiv(r, fd_chunks);
    m.c = r - m.h * chunks;
    return m;
}
__device__ __forceinline__ Item qk_item(const AppendParams& p, int i) { return item_of(i, p.per_qk, p.fd_qk, p.nk, p.fd_nk); }
__device__ __forceinline__ Item v_item(const AppendParams& p, int i) { return item_of(i, p.per_v, p.fd_v, p.nv, p.fd_nv); }

// The source row of a query or key head, and the place of a cache row (codes, or 16-bit values).
template <typename T>
__device__ __forceinline__ const T* qk_row(const AppendParams& p, int64_t t, int h) {
    return h < p.hq ? static_cast<const T*>(p.q) + t * p.qs[0] + h * p.qs[1]
                    : static_cast<const T*>(p.k) + t * p.ks[0] + (h - p.hq) * p.ks[1];
}
__device__ __forceinline__ char* k_place(const AppendParams& p, const Held& at, int h) {
    return p.c.k + at.at + h * p.c.ks[1];
}
__device__ __forceinline__ char* v_place(const AppendParams& p, const Held& at, int h) {
    return p.c.v + at.at + h * p.c.vs[1];
}

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

// A workgroup of values: `out` stores a chunk of eight dims at its place.
template <typename T, bool STREAM, typename F>
__device__ __forceinline__ void append_values(const AppendParams& p, int block, Held* held, F out) {
    const int t0 = block * p.tpb_v;
    const int nt = min(p.tpb_v, p.c.tokens - t0);
    const int items = nt * p.per_v;
    for (int base = 0; base < items; base += ITEMS * THREADS) {
        V8<T> x[ITEMS];
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int i = base + j * THREADS + threadIdx.x;
            if (i >= items) continue;
            const Item m = v_item(p, i);
            const V8<T>* const src = reinterpret_cast<const V8<T>*>(
                static_cast<const T*>(p.v) + static_cast<int64_t>(t0 + m.tl) * p.vs[0] + m.h * p.vs[1] + 8 * m.c);
            x[j] = STREAM ? __builtin_nontemporal_load(src) : *src;
        }
        if (base == 0) place_tokens<float>(p, p.c.vs, p.c.vss, t0, nt, held, nullptr, nullptr);
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int i = base + j * THREADS + threadIdx.x;
            if (i >= items) break;
            const Item m = v_item(p, i);
            const Held at = held[m.tl];
            if (at.at >= 0) out(at, m.h, m.c, x[j]);
        }
    }
}

// Query and key chunks of VW dims a half: both vectors of a rotated pair in one thread.  VW is 8,
// or 1 where the rotated dims are no whole pairs of vectors.
template <typename T, int VW, bool INTER, bool STREAM>
__global__ __launch_bounds__(THREADS) void append_kernel(const AppendParams p) {
    __shared__ __align__(16) float cosine[PAIRS], sine[PAIRS];
    __shared__ Held held[TOKENS];
    if (static_cast<int>(blockIdx.x) >= p.blocks_qk) {
        append_values<T, STREAM>(p, blockIdx.x - p.blocks_qk, held, [&](const Held& at, int h, int c, const V8<T>& x) {
            *reinterpret_cast<V8<T>*>(v_place(p, at, h) + 16 * c) = x;
        });
        return;
    }
    const int t0 = blockIdx.x * p.tpb_qk;
    const int nt = min(p.tpb_qk, p.c.tokens - t0);
    const int items = nt * p.per_qk;
    const int half = p.rd / 2, nrot = half / VW;
    struct Vec {
        T e[VW];
    };
    // A pair of vectors is one of each half of the rotated dims in either layout, so that a
    // wavefront's loads are of one piece (as in rotary.hip).
    constexpr bool NEXT = INTER && VW == 1;
    auto first_dim = [&](int c) { return c < nrot ? (NEXT ? 2 * c : VW * c) : p.rd + VW * (c - nrot); };
    auto load = [&](const T* from) {
        Vec v;
        if constexpr (STREAM && VW == 8)
            v = __builtin_bit_cast(Vec, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from)));
        else
            __builtin_memcpy(&v, __builtin_assume_aligned(from, VW * 2), VW * 2);
        return v;
    };
    auto store = [&](T* to, const Vec& v) { __builtin_memcpy(__builtin_assume_aligned(to, VW * 2), &v, VW * 2); };
    const int apart = NEXT ? 1 : half;
    Vec a[ITEMS], z[ITEMS];
    auto fetch = [&](int base) {
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int i = base + j * THREADS + threadIdx.x;
            if (i >= items) continue;
            const Item m = qk_item(p, i);
            const T* src = qk_row<T>(p, t0 + m.tl, m.h) + first_dim(m.c);
            a[j] = load(src);
            if (m.c < nrot) z[j] = load(src + apart);
        }
    };
    fetch(0);
    place_tokens<float>(p, p.c.ks, p.c.kss, t0, nt, held, cosine, sine);
    for (int base = 0;;) {
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int i = base + j * THREADS + threadIdx.x;
            if (i >= items) break;
            const Item m = qk_item(p, i);
            const Held at = held[m.tl];
            T* dst;
            if (m.h < p.hq) {
                dst = static_cast<T*>(p.qo) + static_cast<int64_t>(t0 + m.tl) * p.qos[0] + m.h * p.qos[1];
                // A query of no sequence (or past the cache) is zero.
                if (at.pos < 0) a[j] = z[j] = Vec{};
            } else {
                if (at.at < 0) continue;
                dst = reinterpret_cast<T*>(k_place(p, at, m.h - p.hq));
            }
            dst += first_dim(m.c);
            if (m.c >= nrot) {
                store(dst, a[j]);
                continue;
            }
            float cs[VW], sn[VW];
            if constexpr (INTER && VW > 1) {
                // (Pairs lie within a vector: the angles of the two are half of all apart.)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int k = m.tl * half + VW / 2 * m.c + i * (half / 2);
                    __builtin_memcpy(cs + i * (VW / 2), __builtin_assume_aligned(cosine + k, VW * 2), VW * 2);
                    __builtin_memcpy(sn + i * (VW / 2), __builtin_assume_aligned(sine + k, VW * 2), VW * 2);
                }
            } else {
                __builtin_memcpy(cs, __builtin_assume_aligned(cosine + m.tl * half + VW * m.c, VW * 4), VW * 4);
                __builtin_memcpy(sn, __builtin_assume_aligned(sine + m.tl * half + VW * m.c, VW * 4), VW * 4);
            }
            Vec u, w;
            auto pair = [&](T p1, T p2, int e, T& y1, T& y2) {
                float f1, f2;
                turned(to_f32(p1), to_f32(p2), cs[e], sn[e], f1, f2);
                y1 = from_f32<T>(f1);
                y2 = from_f32<T>(f2);
            };
            if constexpr (INTER && VW > 1) {
#pragma unroll
                for (int e = 0; e < VW / 2; ++e) {
                    pair(a[j].e[2 * e], a[j].e[2 * e + 1], e, u.e[2 * e], u.e[2 * e + 1]);
                    pair(z[j].e[2 * e], z[j].e[2 * e + 1], VW / 2 + e, w.e[2 * e], w.e[2 * e + 1]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < VW; ++e) pair(a[j].e[e], z[j].e[e], e, u.e[e], w.e[e]);
            }
            store(dst, u);
            store(dst + apart, w);
        }
        base += ITEMS * THREADS;
        if (base >= items) break;
        fetch(base);
    }
}

// ---------------------------------------------------------------- 4 bits

// The largest of a value (not negative) over the four lanes of a group: a quad's exchanges.
__device__ __forceinline__ int max_of_four(int v) {
    v = max(v, __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true));  // lanes 1, 0, 3, 2
    return max(v, __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true));  // lanes 2, 3, 0, 1
}

// The group's scale byte and exponent e from the largest exponent field of its 64-bit values.
struct Scale {
    int byte, e;
};
__device__ __forceinline__ Scale group_scale(int field) {
    field = max_of_four(field);
    const int e = field == 0 ? -127 : min(max(field - 1025, -126), 127);
    return Scale{field == 0x7ff ? 255 : e + 127, e};
}

// Eight values over a power of two as codes: nearest, ties to even, saturating.
__device__ __forceinline__ uint32_t codes_of(const float (&f)[8], float unit) {
    uint32_t codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, f[0], f[1], unit, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], unit, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], unit, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], unit, 3);
}
// (Through a dword of its own: a vector's element in a bit cast stands for the first one.)
__device__ __forceinline__ uint32_t codes_of(const bf16x8& x, float unit) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, x);
    const uint32_t a = w[0], b = w[1], c = w[2], d = w[3];
    uint32_t codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(pair, a), unit, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(pair, b), unit, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(pair, c), unit, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(pair, d), unit, 3);
}
__device__ __forceinline__ uint32_t codes_of(const f16x8& x, float unit) {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, x);
    const uint32_t a = w[0], b = w[1], c = w[2], d = w[3];
    uint32_t codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(0u, __builtin_bit_cast(pair, a), unit, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(pair, b), unit, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(pair, c), unit, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(pair, d), unit, 3);
}

// Values of 16 bits, converted as they are: their largest by its bits, two at a time.
template <typename T>
__device__ __forceinline__ uint32_t quantise(const V8<T>& x, int& byte) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const u32x4 w = __builtin_bit_cast(u32x4, x) & 0x7fff7fffu;
    const uint32_t a = w[0], b = w[1], c = w[2], d = w[3];
    const u16x2 two = __builtin_elementwise_max(
        __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)),
        __builtin_elementwise_max(__builtin_bit_cast(u16x2, c), __builtin_bit_cast(u16x2, d)));
    const int top = max_of_four(max(static_cast<int>(two[0]), static_cast<int>(two[1])));
    const float largest = to_f32(__builtin_bit_cast(T, static_cast<uint16_t>(top)));
    // (A subnormal bf16's exponent is below the smallest scale's, as a field of zero says; only
    // zero itself keeps the byte 0.)
    const int field = static_cast<int>(__float_as_uint(largest) >> 23);
    byte = field == 255 ? 255 : max(field - 2, top == 0 ? 0 : 1);
    return codes_of(x, scale_of(max(byte, 1)));
}

// A value of 64 bits in 32, toward zero with the last bit set where that drops anything: no border
// between two codes has that bit (nearest rounding could land on one), so codes stay those of the
// value as it was.
__device__ __forceinline__ float to_odd(double x) {
    const float f = static_cast<float>(x);
    const double back = static_cast<double>(f);
    const uint32_t bits = __float_as_uint(f);
    return back == x ? f : __uint_as_float((fabs(back) > fabs(x) ? bits - 1 : bits) | 1u);
}

// Rotated values in 32 bits, each at most `slack` off the exact one: their codes, should they be
// those of every value that near (`sure`, the same for the lanes of a group), so that the nearest
// codes in exact arithmetic cost 64 bits only next to a border (one group in some thousands).
__device__ __forceinline__ uint32_t quantise(const float (&y)[8], float slack, int& byte, bool& sure) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(y[i]) & 0x7fffffffu));
    // The group's largest lies between these two.
    const int most = max_of_four(__float_as_int(top + slack)), least = max_of_four(__float_as_int(fmaxf(top - slack, 0.f)));
    const int field = most >> 23;
    // (Within them nothing that counts is subnormal, scale and slack included.)
    const bool plain = field == least >> 23 && ((field >= 60 && field <= 150) || most == 0);
    byte = most == 0 ? 0 : field - 2;
    const float unit = scale_of(max(byte, 1));
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo[i] = y[i] - slack;
        hi[i] = y[i] + slack;
    }
    const uint32_t codes = codes_of(lo, unit);
    // (A slack of zero leaves the sign of zeros alone in lo.)
    sure = max_of_four(plain && (codes == codes_of(hi, unit) || slack == 0.f) ? 0 : 1) == 0;
    return codes;
}

// Chunks of eight dims; head dims are whole groups, so a group's four chunks are four
// neighbouring lanes with items of one token and head.
//
// Bound by issue (the vector unit was busy 78% of the time) until keys were rotated and converted in
// 32 bits, values converted as they are, and rows' places formed once a token: 4 x up to 2048 tokens
// of 8 heads x 128 18.3 to 14.3 us in a graph, 4 x 4096 36.4 to 26.0 (3.3 TB/s).  The 64-bit groups
// read their vectors at once: value after value they took the call back to 20 us.
template <typename T, bool INTER>
__global__ __launch_bounds__(THREADS) void append4_kernel(const AppendParams p) {
    __shared__ __align__(32) float cosine[PAIRS], sine[PAIRS];
    __shared__ __align__(16) double cosine64[PAIRS], sine64[PAIRS];
    __shared__ Held held[TOKENS];
    typedef V8<T> v8;
    if (static_cast<int>(blockIdx.x) >= p.blocks_qk) {
        append_values<T, false>(p, blockIdx.x - p.blocks_qk, held, [&](const Held& at, int h, int c, const v8& x) {
            int byte;
            *reinterpret_cast<uint32_t*>(v_place(p, at, h) + 4 * c) = quantise<T>(x, byte);
            if ((c & 3) == 0) p.c.vsc[at.scale + h * p.c.vss[1] + (c >> 2)] = static_cast<uint8_t>(byte);
        });
        return;
    }
    const int t0 = blockIdx.x * p.tpb_qk;
    const int nt = min(p.tpb_qk, p.c.tokens - t0);
    const int items = nt * p.per_qk;
    const int half = p.rd / 2;
    // Rotated dims that are whole chunks (their halves, unless pairs are neighbours): a chunk's
    // partners are one then too, and all of it is rotated, or none.
    const bool whole = INTER ? p.rd % 8 == 0 : half % 8 == 0;
    v8 x[ITEMS], z[ITEMS];
    auto fetch = [&](int base) {
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int i = base + j * THREADS + threadIdx.x;
            if (i >= items) continue;
            const Item m = qk_item(p, i);
            const T* src = qk_row<T>(p, t0 + m.tl, m.h);
            const int d0 = 8 * m.c;
            x[j] = *reinterpret_cast<const v8*>(src + d0);
            if (!INTER && whole && d0 < p.rd) z[j] = *reinterpret_cast<const v8*>(src + (d0 < half ? d0 + half : d0 - half));
        }
    };
    const auto keep = [&](const Item& m, const Held& at, uint32_t codes, int byte) {
        const int h = m.h - p.hq;
        *reinterpret_cast<uint32_t*>(k_place(p, at, h) + 4 * m.c) = codes;
        if ((m.c & 3) == 0) p.c.ksc[at.scale + h * p.c.kss[1] + (m.c >> 2)] = static_cast<uint8_t>(byte);
    };
    const auto q_place = [&](const Item& m) {
        return static_cast<T*>(p.qo) + static_cast<int64_t>(t0 + m.tl) * p.qos[0] + m.h * p.qos[1] + 8 * m.c;
    };
    fetch(0);
    place_tokens<double>(p, p.c.ks, p.c.kss, t0, nt, held, cosine, sine, cosine64, sine64);
    for (int base = 0;;) {
        uint32_t again = 0;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int i = base + j * THREADS + threadIdx.x;
            if (i >= items) break;
            const Item m = qk_item(p, i);
            const Held at = held[m.tl];
            if (m.h >= p.hq && at.at < 0) continue;  // (all four lanes of a group)
            if (!whole) {
                again |= 1u << j;
                continue;
            }
            const int d0 = 8 * m.c;
            float y[8], size = 0.f;
            if (d0 < p.rd) {
                constexpr int N = INTER ? 4 : 8;  // angles
                const bool front = d0 < half;
                const int k = m.tl * half + (INTER ? d0 / 2 : (front ? d0 : d0 - half));
                float c[N], s[N];
                __builtin_memcpy(c, __builtin_assume_aligned(cosine + k, 4 * N), 4 * N);
                __builtin_memcpy(s, __builtin_assume_aligned(sine + k, 4 * N), 4 * N);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float own = to_f32(x[j][e]), other = to_f32(INTER ? x[j][e ^ 1] : z[j][e]);
                    const float t = other * s[INTER ? e >> 1 : e];
                    const bool minus = INTER ? (e & 1) == 0 : front;
                    y[e] = __builtin_fmaf(own, c[INTER ? e >> 1 : e], minus ? -t : t);
                    size = fmaxf(size, fabsf(own) + fabsf(other));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = to_f32(x[j][e]);
            }
            if (m.h < p.hq) {
                v8 w;
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = from_f32<T>(at.pos < 0 ? 0.f : y[e]);
                *reinterpret_cast<v8*>(q_place(m)) = w;
                continue;
            }
            // Off by the cosine's and sine's rounding, the product's and the sum's, each 2^-24 of
            // (|x| + |other|) scale at most, doubled for what the test itself rounds.
            int byte;
            bool sure;
            const uint32_t codes = quantise(y, size == 0.f ? 0.f : fmaxf(size * p.slack, 0x1p-100f), byte, sure);
            if (sure)
                keep(m, at, codes, byte);
            else
                again |= 1u << j;
        }
        // Groups next to a border, and rotated dims that are no whole chunks: in 64 bits, value by
        // value from memory.
#pragma unroll 1
        for (int j = 0; again != 0; ++j, again >>= 1) {
            if ((again & 1u) == 0) continue;
            const Item m = qk_item(p, base + j * THREADS + threadIdx.x);
            const Held at = held[m.tl];
            const T* const src = qk_row<T>(p, t0 + m.tl, m.h);
            const auto value = [&](int d) {
                const double own = static_cast<double>(to_f32(src[d]));
                if (d >= p.rd) return own;
                const bool first = INTER ? (d & 1) == 0 : d < half;
                const double other = static_cast<double>(to_f32(src[INTER ? d ^ 1 : (first ? d + half : d - half)]));
                const int k = m.tl * half + (INTER ? d >> 1 : (first ? d : d - half));
                return own * cosine64[k] + other * (first ? -sine64[k] : sine64[k]);
            };
            double y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = value(8 * m.c + e);
            if (m.h < p.hq) {
                v8 w;
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = from_f32<T>(at.pos < 0 ? 0.f : static_cast<float>(y[e]));
                *reinterpret_cast<v8*>(q_place(m)) = w;
                continue;
            }
            int top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, static_cast<int>(__double2hiint(y[e]) & 0x7fffffff));
            const Scale scale = group_scale(top >> 20);
            const double inv = __hiloint2double((1023 - scale.e) << 20, 0);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = to_odd(y[e] * inv);
            keep(m, at, codes_of(f, 1.f), scale.byte);
        }
        base += ITEMS * THREADS;
        if (base >= items) break;
        fetch(base);
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
    p.slack = static_cast<float>(std::fabs(a->rotary_scale) * 0x1p-21);
    const int64_t tokens = a->cache.tokens;
    const bool four = a->cache.bits == 4;
    const int vw = four ? 8 : (p.rd % 16 == 0 ? 8 : 1);
    p.nk = four ? p.c.d / 8 : p.rd / (2 * vw) + (p.c.d - p.rd) / vw;
    p.nv = p.c.dv / 8;
    p.per_qk = (p.hq + p.c.hkv) * p.nk;
    p.per_v = p.c.hkv * p.nv;
    // Tokens of a workgroup: a batch of items a thread, unless few tokens leave CUs idle.
    const auto tokens_of = [&](int per, int64_t most) {
        return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({ITEMS * THREADS / per, most, tokens / 1024})));
    };
    p.tpb_qk = tokens_of(p.per_qk, p.rd > 0 ? std::min(TOKENS, PAIRS / (p.rd / 2)) : TOKENS);
    p.tpb_v = tokens_of(p.per_v, TOKENS);
    p.blocks_qk = static_cast<int>(ceil_div(tokens, p.tpb_qk));
    p.fd_qk = fwd::fast_div(static_cast<uint32_t>(p.per_qk));
    p.fd_v = fwd::fast_div(static_cast<uint32_t>(p.per_v));
    p.fd_nk = fwd::fast_div(static_cast<uint32_t>(p.nk));
    p.fd_nv = fwd::fast_div(static_cast<uint32_t>(p.nv));
    p.fd_half = fwd::fast_div(static_cast<uint32_t>(p.rd / 2));
    const dim3 grid(static_cast<unsigned>(p.blocks_qk + ceil_div(tokens, p.tpb_v)));
    auto enqueue = [&](void (*kernel)(AppendParams)) { hipLaunchKernelGGL(kernel, grid, dim3(THREADS), 0, stream, p); };
    if (four)
        enqueue(p.inter ? append4_kernel<T, true> : append4_kernel<T, false>);
    else if (vw == 8 && tokens * (static_cast<int64_t>(p.hq + p.c.hkv) * p.c.d + p.c.hkv * p.c.dv) * 2 >= kStreamBytes)
        enqueue(p.inter ? append_kernel<T, 8, true, true> : append_kernel<T, 8, false, true>);
    else if (vw == 8)
        enqueue(p.inter ? append_kernel<T, 8, true, false> : append_kernel<T, 8, false, false>);
    else
        enqueue(p.inter ? append_kernel<T, 1, true, false> : append_kernel<T, 1, false, false>);
    return hipGetLastError();
}

// ---------------------------------------------------------------- read

// Keys or values: where they lie, and the dense copy.
struct Side {
    const char* rows;
    const uint8_t* scales;
    int64_t stride[3], scale_stride[3];
    char* out;
    int chunks;  // of eight dims, of a row
    int blocks;  // workgroups per (sequence, K/V head)
    fwd::FastDiv fd_chunks;
};

struct ReadParams {
    Cache c;
    Side side[2];
    int max_k;
    int end;  // 1: rows past a sequence's length are zeroed, 0: left out
};

// A workgroup copies chunks of one unit's keys or values.
template <typename T, bool FOUR>
__global__ __launch_bounds__(THREADS) void read_kernel(const ReadParams p) {
    const int per = p.side[0].blocks + p.side[1].blocks;
    const int unit = blockIdx.x / per;
    const int b = unit / p.c.hkv, h = unit - b * p.c.hkv;
    int block = blockIdx.x - unit * per;
    const bool values = block >= p.side[0].blocks;
    const Side& side = p.side[values ? 1 : 0];
    if (values) block -= p.side[0].blocks;
    const int first = block * (THREADS * ITEMS) + threadIdx.x;
    const int lk = min(max(uniform_i32(p.c.klen + b), 0), p.c.capacity);
    const int rows_out = p.end ? p.max_k : min(lk, p.max_k);
    if (fwd::fdiv(block * (THREADS * ITEMS), side.fd_chunks) >= rows_out) return;
    u32x4 x[ITEMS];
    uint32_t byte[ITEMS];
    int pos[ITEMS], c[ITEMS], entry[ITEMS], row[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        pos[j] = fwd::fdiv(first + j * THREADS, side.fd_chunks);
        c[j] = first + j * THREADS - pos[j] * side.chunks;
        x[j] = u32x4{0u, 0u, 0u, 0u};
        byte[j] = 0;
    }
    if (lk > 0) {
        // Every table entry, then every row (keys past the last repeat its, unused), so that a
        // thread's items wait for memory together.
        const int32_t* const table = p.c.table + b * p.c.table_stride;
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int at = min(pos[j], lk - 1), n = fwd::fdiv(at, p.c.fd_page);
            row[j] = at - n * p.c.page;
            entry[j] = table[n];
        }
        const char* const rows = side.rows + h * side.stride[1];
        const uint8_t* const scales = side.scales + h * side.scale_stride[1];
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            // (Page strides are below 2^32 bytes, row strides below 2^26.)
            const uint32_t page = static_cast<uint32_t>(clamp_page(entry[j], p.c.pages)), r = static_cast<uint32_t>(row[j]);
            const auto at = [&](const int64_t(&st)[3], uint32_t inner) {
                return static_cast<uint64_t>(page) * static_cast<uint32_t>(st[0]) +
                       static_cast<uint64_t>(r) * static_cast<uint32_t>(st[2]) + inner;
            };
            const uint32_t chunk = static_cast<uint32_t>(c[j]);
            if constexpr (FOUR) {
                byte[j] = scales[at(side.scale_stride, chunk >> 2)];
                x[j][0] = *reinterpret_cast<const uint32_t*>(rows + at(side.stride, 4 * chunk));
            } else {
                x[j] = *reinterpret_cast<const u32x4*>(rows + at(side.stride, 16 * chunk));
            }
        }
    }
    char* const out = side.out + static_cast<int64_t>(unit) * p.max_k * (side.chunks * 16);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        if (pos[j] >= rows_out) continue;
        if constexpr (FOUR) {
            const uint32_t codes = x[j][0];
            const float s = scale_of(byte[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[j][e] = fp4_pair<T>(codes, s, e);
        }
        if (pos[j] >= lk) x[j] = u32x4{0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4*>(out + static_cast<uint64_t>(static_cast<uint32_t>(first + j * THREADS)) * 16) = x[j];
    }
}

}  // namespace

hipError_t launch_read(const kmi_paged_cache& c, void* k, void* v, int64_t max_k, bool end, hipStream_t stream) {
    ReadParams p{};
    p.end = end;
    p.c = device_cache(c);
    p.max_k = static_cast<int>(max_k);
    for (int w = 0; w < 2; ++w) {
        Side& s = p.side[w];
        s.rows = w ? p.c.v : p.c.k;
        s.scales = w ? p.c.vsc : p.c.ksc;
        for (int i = 0; i < 3; ++i) {
            s.stride[i] = w ? p.c.vs[i] : p.c.ks[i];
            s.scale_stride[i] = w ? p.c.vss[i] : p.c.kss[i];
        }
        s.out = static_cast<char*>(w ? v : k);
        s.chunks = (w ? p.c.dv : p.c.d) / 8;
        s.blocks = static_cast<int>(ceil_div(max_k * s.chunks, THREADS * ITEMS));
        s.fd_chunks = fwd::fast_div(static_cast<uint32_t>(s.chunks));
    }
    const dim3 grid(static_cast<unsigned>((p.side[0].blocks + p.side[1].blocks) * c.batch * c.heads_kv));
    const bool bf = c.dtype == KMI_BF16;
    if (c.bits == 4) {
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
    if (max_k > ((int64_t{1} << 31) - THREADS * ITEMS) / per) return false;
    const int64_t units = c.batch * c.heads_kv;
    return units == 0 || ceil_div(max_k * per, THREADS * ITEMS) + 1 < (int64_t{1} << 24) / units;
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
    return hip_status(paged::launch_read(*c, k_out, v_out, max_k, true, static_cast<hipStream_t>(stream)), "kmi_paged_read");
}
