// What the paged-cache kernels share: the cache as the kernels see it, its host checks, the
// angles of the position rotation and the 4-bit conversions.
#pragma once

#include "attention_params.hpp"

namespace kmi {
namespace paged {

// A kmi_paged_cache on the device side (strides in bytes).
struct Cache {
    char* k;
    char* v;
    uint8_t* ksc;
    uint8_t* vsc;
    int64_t ks[3], vs[3], kss[3], vss[3];
    const int32_t* table;
    int64_t table_stride;
    const int32_t* klen;
    const int32_t* cu;  // null: one token per sequence
    int pages, page, hkv, d, dv, batch, tokens;
    int capacity;  // keys a table row can hold
    fwd::FastDiv fd_page;
};

// Table entries, lengths and offsets are read with scalar loads where the address is uniform
// (no kernel writes them).
__device__ __forceinline__ int uniform_i32(const int32_t* p) {
    return *(const __attribute__((address_space(4))) int32_t*)(reinterpret_cast<uintptr_t>(p));
}

__device__ __forceinline__ int clamp_page(int e, int pages) {
    return static_cast<uint32_t>(e) < static_cast<uint32_t>(pages) ? e : 0;
}

// Sequence b's first token, token count and keys (as clamped by the header's rules).
struct Span {
    int q0, lq, lk;
};
__device__ __forceinline__ Span span_of(const Cache& c, int b) {
    Span s;
    s.lk = min(max(uniform_i32(c.klen + b), 0), c.capacity);
    if (c.cu) {
        s.q0 = min(max(uniform_i32(c.cu + b), 0), c.tokens);
        s.lq = min(max(uniform_i32(c.cu + b + 1), s.q0), c.tokens) - s.q0;
    } else {
        s.q0 = b;
        s.lq = 1;
    }
    return s;
}

// A token's sequence and key position; seq is -1 for a token of no sequence and pos -1 for
// a key outside the cache.
struct Place {
    int seq, pos;
};
__device__ __forceinline__ Place place_of(const Cache& c, int t) {
    Place at{t, -1};
    int r = 0, lq = 1;
    if (c.cu) {
        // The last offset at or below t (offsets do not decrease).
        int lo = 0, hi = c.batch;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (c.cu[mid] <= t)
                lo = mid;
            else
                hi = mid - 1;
        }
        if (lo >= c.batch || c.cu[lo] > t) return Place{-1, -1};
        const int end = c.cu[lo + 1];
        if (t >= end) return Place{-1, -1};
        at.seq = lo;
        r = t - max(c.cu[lo], 0);
        lq = min(end, c.tokens) - max(c.cu[lo], 0);
    }
    const int64_t pos = static_cast<int64_t>(c.klen[at.seq]) - lq + r;
    if (pos >= 0 && pos < c.capacity) at.pos = static_cast<int>(pos);
    return at;
}

// The page of a key, or -1 where the table names none.
__device__ __forceinline__ int page_of(const Cache& c, int seq, int pos, int& row) {
    const int i = fwd::fdiv(pos, c.fd_page);
    row = pos - i * c.page;
    const int e = c.table[seq * c.table_stride + i];
    return static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages) ? e : -1;
}

// ---------------------------------------------------------------- rotation

// cos and sin of pos * freq.  The angle is formed and reduced to turns in 64 bits: in 32 a
// position of 10^6 would leave it 0.03 radians off.  sincospif is exact to two units in the
// last place of its (reduced) argument.
__device__ __forceinline__ void turn(double pos, float freq, float& c, float& s) {
    double r = pos * static_cast<double>(freq) * 0.15915494309189535;
    r -= rint(r);
    sincospif(static_cast<float>(r + r), &s, &c);
}
// The same in 64 bits, for values that are compared with a border between two codes.
__device__ __forceinline__ void turn(double pos, float freq, double& c, double& s) {
    double r = pos * static_cast<double>(freq) * 0.15915494309189535;
    r -= rint(r);
    sincospi(r + r, &s, &c);
}

// A pair turned, with its products and sums in one order everywhere (left to the compiler, which
// of the two products is fused differs from kernel to kernel).
__device__ __forceinline__ void turned(float x1, float x2, float c, float s, float& y1, float& y2) {
    y1 = __builtin_fmaf(x1, c, -(x2 * s));
    y2 = __builtin_fmaf(x2, c, x1 * s);
}

// Inputs that a kernel reads once are read past the caches (non-temporal loads) from this size on, a
// quarter of the last-level cache: the results then stay there instead.  Measured on the rotation
// (us, through the caches / past them; after the product that writes its input): 25 MB 9.7 / 10.2
// (19.5 / 19.4), 50 MB 18.6 / 21.1 (34.1 / 34.1), 75 MB 30.1 / 30.6 (51.1 / 50.6), 101 MB 39.6 / 38.3
// (68.4 / 66.0), 201 MB 77.9 / 67.1 (144.7 / 136.8).  Results written past them cost what reads
// them next more than they save (201 MB 78.0 / 73.3, with a sum over them 119.4 / 126.7).
constexpr int64_t kStreamBytes = int64_t{64} << 20;

// ---------------------------------------------------------------- 4 bits

// Two of the values a dword of eight codes stands for (codes 2 sel and 2 sel + 1) times the
// power of two in `scale` (its exponent alone counts), as a packed pair of T: exact in bf16; in
// fp16 exact down to 2^-24.
template <typename T>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t codes, float scale, int sel);
#define KMI_FP4_PAIR(T, fn)                                                                     \
    template <>                                                                                 \
    __device__ __forceinline__ uint32_t fp4_pair<T>(uint32_t codes, float scale, int sel) {     \
        switch (sel) {                                                                          \
            case 0: return __builtin_bit_cast(uint32_t, fn(codes, scale, 0));                   \
            case 1: return __builtin_bit_cast(uint32_t, fn(codes, scale, 1));                   \
            case 2: return __builtin_bit_cast(uint32_t, fn(codes, scale, 2));                   \
            default: return __builtin_bit_cast(uint32_t, fn(codes, scale, 3));                  \
        }                                                                                       \
    }
KMI_FP4_PAIR(bf16, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4)
KMI_FP4_PAIR(f16, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4)
#undef KMI_FP4_PAIR

// The scale a byte stands for, as the conversions take it (byte 255: NaN; byte 0 is only written
// for groups of zeros).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// ---------------------------------------------------------------- host side

// Why a cache is refused, or null.  writes: an append (k / v are written).
const char* check_cache(const kmi_paged_cache& c, bool uses_tokens);
Cache device_cache(const kmi_paged_cache& c);
// Whether a dense copy of max_k keys a sequence can be launched, and the launch (kmi_paged_read;
// end: rows past a sequence's length are zeroed and not left out).
bool read_fits(const kmi_paged_cache& c, int64_t max_k);
hipError_t launch_read(const kmi_paged_cache& c, void* k, void* v, int64_t max_k, bool end, hipStream_t stream);

}  // namespace paged
}  // namespace kmi
