// Attention over a paged cache for few query rows: single tokens and short drafts, at most 32
// "virtual rows" (query tokens x GQA group) per (sequence, K/V head).
//
// Bound by the cache's bytes.  A unit's keys are dealt in tiles of 32 to the wavefronts of its
// splits in turn.  Each tile is two halves of 16 rows (page sizes are multiples of 16), read through
// a buffer resource that ends with the sequence: rows past the last key read as zeros, so nothing
// stale in a page is ever touched.  The wavefronts share nothing until the end and so need no
// barrier: K goes straight into MFMA operand registers, V through a private LDS tile read
// transposed; the next tile's loads and the table entries of the one after are in flight during a
// tile's softmax and PV.  S^T = K Q^T leaves a query row per lane, its softmax state is scalar; P
// feeds O^T += V^T P^T as it stands, in two 16-bit parts (a second product, hidden behind the
// loads: 64 sequences x 2 heads x 8192 keys x 128 100.2 against 100.4 us, in 4 bits 35.5 against
// 35.1, when both took that long), so that results are as close to 64-bit ones as their own
// rounding (0.0017 relative where one part gave 0.0023).
//
// 16-bit caches: 16x16x32 MFMAs.  4-bit caches: the codes of K are the operand of the scaled
// 16x16x128 MFMA as they lie in memory, with the cache's own scale bytes; no key is ever
// widened.  Its other operand, Q, is the sum of two (bf16) or three (fp16) e4m3 parts of four
// significant bits, 2^-4 apart, on one power of two per row: bf16's eight bits fit two parts
// exactly (elements below 2^-13 of the row's largest to within 2^-17 of it), fp16's eleven fit
// three.  V's codes are widened by the packed conversions on their way into the LDS tile.
//
// Measured: that 16-bit call takes 83 us with its merge, 6.5 TB/s (a copy moves 5.13, the dense
// decode kernel takes 97 us), the 4-bit one (143 MB) 30.6, 4.7 TB/s, and 54.5 with twice the
// sequences, 5.2: start, first latencies and the merge are fixed.  What made it so, in 4 bits: entries and lengths read
// side by side, table entries clamped and scale bytes widened where they are used (a widening left
// where the byte was loaded waited for the whole next tile: 38.4 -> 35.5 us), ranges computed and
// keys hidden in a sequence's last tile alone.  Two or three tiles in flight were no faster (35.5,
// 37.1), nor eight wavefronts a workgroup.
#pragma once

#include "paged_attn.hpp"

namespace kmi {
namespace paged {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mfma16;
template <>
struct Mfma16<bf16> {
    typedef bf16x8 v8;
    static __device__ __forceinline__ f32x4 run(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mfma16<f16> {
    typedef f16x8 v8;
    static __device__ __forceinline__ f32x4 run(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// gfx950's transposed LDS read (see mfma_tile.hpp).
template <typename T>
__device__ __forceinline__ u32x2 tr_read(const T* p) {
    if constexpr (std::is_same<T, bf16>::value) {
        typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 x4;
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                                             (__attribute__((address_space(3))) x4*)(reinterpret_cast<uintptr_t>(p))));
    } else {
        typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 x4;
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                                             (__attribute__((address_space(3))) x4*)(reinterpret_cast<uintptr_t>(p))));
    }
}

// Keys and values are read once, past the caches (auxiliary bit 1): 64 x 8192 keys of 2 x 128 98.9
// us through them, 86.8 so, 16 x 8192 31.5, 27.9, in 4 bits 34.7, 32.0, up to 50 MB alike (three
// caches in turn, as a model's layers are; one cache of 134 to 268 MB that stays in the last level
// is 4 to 11% slower so).
template <typename R>
__device__ __forceinline__ u32x4 load_once(R rsrc, uint32_t offset) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset, 0, 2));
}

// Reductions over the four lanes that hold a row (lane, lane ^ 16, lane ^ 32, lane ^ 48).
__device__ __forceinline__ float max4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

constexpr int WAVES = 4;
constexpr int THREADS = WAVES * kWave;
constexpr int TK = 32;                // keys of a tile
constexpr float kLazy = 8.f;          // log2 units a row max may grow before O is rescaled
constexpr float kLn2f = 0.6931471805599453f;
constexpr uint32_t kOpen = 0x7fffffffu;  // the range of a resource whose rows are all there
constexpr uint32_t kNone = 0x80000000u;  // an offset past every range: reads as zeros

// Parts of a 4-bit call's Q.
template <typename T>
constexpr int kParts = std::is_same<T, bf16>::value ? 2 : 3;

// LDS row pitch of the V tile: 16 elements of padding spread the rows over the banks.
constexpr int v_pitch(int dp) { return dp + 16; }

template <typename T, int DP, int NQ>
constexpr size_t decode_lds() {
    const size_t v = static_cast<size_t>(WAVES) * TK * v_pitch(DP) * sizeof(T);
    const size_t merge = static_cast<size_t>(WAVES) * 16 * (DP + 4 + 2) * sizeof(float);
    return v > merge ? v : merge;
}

// Wavefronts per SIMD the kernel is held to: four for 16 rows of a 4-bit cache, whose tiles are
// small and which is bound by how many wavefronts work at once.
constexpr int decode_occupancy(int dp, int nq, bool four) { return four && nq == 1 && dp <= 128 ? 4 : 1; }

template <typename T, int DP, int NQ, bool FOUR>
__global__ __launch_bounds__(THREADS, decode_occupancy(DP, NQ, FOUR)) void paged_decode_kernel(const AttnParams p) {
    typedef typename Mfma16<T>::v8 v8;
    constexpr int DC = DP / 32;                // K fragments of a key row (16 bits)
    constexpr int KC = (DP + 127) / 128;       // the same at 4 bits
    constexpr int DB = DP / 16;                // output blocks
    constexpr int VP = v_pitch(DP);
    constexpr int CP = DP + 4;
    // V staging, 16 bits: VPS lanes a row (a power of two; those past the padded row idle).
    constexpr int NCH = DP / 8;
    constexpr int VPS = NCH <= 4 ? 4 : NCH <= 8 ? 8 : NCH <= 16 ? 16 : 32;
    constexpr int RPP = kWave / VPS, KIT = 16 / RPP;  // rows a pass, passes of a half
    // V staging, 4 bits: chunks of 32 dims (one scale byte), N4 a row, R4 rounds of a half.
    constexpr int N4 = DP / 32, R4 = (16 * N4 + kWave - 1) / kWave;

    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g4 = lane >> 4, l16 = lane & 15;
    const int units = p.batch * p.hkv;
    const int lin = static_cast<int>(blockIdx.x) - p.tail_blocks;
    if (lin < 0) {
        zero_tail<T>(p, blockIdx.x);
        return;
    }
    const int bh = fwd::fdiv(lin, p.fd_splits);
    const int split = lin - bh * p.splits;
    const int seq = fwd::fdiv(bh, p.fd_hkv), kvh = bh - seq * p.hkv;
    const int G = p.group;
    // Tiles are dealt to a unit's wavefronts in turn: tile slot, slot + nslots, ...  A wavefront's
    // first table entries are so known before the sequence's length, and read beside it.
    const int slot = split * WAVES + wave, nslots = p.splits * WAVES;

    // A tile in registers.
    struct TileRegs {
        v8 k[FOUR ? 1 : 2][FOUR ? 1 : DC];
        u32x4 v[FOUR ? 1 : 2][FOUR ? 1 : KIT];
        u32x4 k4[FOUR ? 2 : 1][FOUR ? KC : 1], v4[FOUR ? 2 : 1][FOUR ? R4 : 1];
        uint8_t k4s[FOUR ? 2 : 1][FOUR ? KC : 1], v4s[FOUR ? 2 : 1][FOUR ? R4 : 1];
    };
    TileRegs x;
    T* const vl = reinterpret_cast<T*>(smem) + wave * TK * VP;
    const int krow = lane / VPS, dg = lane % VPS;
    const uint32_t kst = static_cast<uint32_t>(p.c.ks[2]), vst = static_cast<uint32_t>(p.c.vs[2]);
    const uint32_t kss = FOUR ? static_cast<uint32_t>(p.c.kss[2]) : 0, vss = FOUR ? static_cast<uint32_t>(p.c.vss[2]) : 0;
    // The unit's head within a page.
    const char* const kh = p.c.k + kvh * p.c.ks[1];
    const char* const vh = p.c.v + kvh * p.c.vs[1];
    const uint8_t* const ksh = FOUR ? p.c.ksc + kvh * p.c.kss[1] : nullptr;
    const uint8_t* const vsh = FOUR ? p.c.vsc + kvh * p.c.vss[1] : nullptr;

    // The page and row of a half tile (keys past what the table holds repeat its last).
    struct Entry {
        int page, row;
    };
    auto entry = [&](int key) {
        Entry e;
        e.page = p.entry_at(seq, max(min(key, p.c.capacity - 1), 0), e.row);
        return e;
    };
    // (Page strides are below 2^32 bytes.)
    auto at = [](const auto* base, const Entry& e, int64_t page_stride, uint32_t row_stride) {
        return base + static_cast<uint64_t>(static_cast<uint32_t>(e.page)) * static_cast<uint32_t>(page_stride) +
               static_cast<uint32_t>(e.row) * static_cast<uint64_t>(row_stride);
    };
    // The lane's byte offsets within a half (past every range for dims that are none).
    uint32_t koff[FOUR ? KC : DC], voff[FOUR ? R4 : 1], ksoff[FOUR ? KC : 1], vsoff[FOUR ? R4 : 1];
    if constexpr (!FOUR) {
#pragma unroll
        for (int c = 0; c < DC; ++c) koff[c] = 32 * c + 8 * g4 < p.d ? l16 * kst + 16 * g4 + 64 * c : kNone;
        voff[0] = 8 * dg < p.dv ? krow * vst + 16 * dg : kNone;
    } else {
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const bool in = 128 * c + 32 * g4 < p.d;
            koff[c] = in ? l16 * kst + 64 * c + 16 * g4 : kNone;
            ksoff[c] = in ? l16 * kss + 4 * c + g4 : kNone;
        }
#pragma unroll
        for (int i = 0; i < R4; ++i) {
            const int ci = lane + kWave * i, r = ci / N4, ch = ci % N4;
            const bool in = r < 16 && 32 * ch < p.dv;
            voff[i] = in ? r * vst + 16 * ch : kNone;
            vsoff[i] = in ? r * vss + ch : kNone;
        }
    }
    // Requests `rows` rows (16 n at most) from an entry on into halves h .. h + n - 1.
    auto request = [&](Entry e, int rows, int h0, int n) __attribute__((always_inline)) {
        e.page = clamp_page(e.page, p.c.pages);
        // (Ranges matter at the sequence's end alone.)
        uint32_t ek = kOpen, ev = kOpen, eks = kOpen, evs = kOpen;
        if (rows < 16 * n) {
            ek = rows_extent(rows, kst, FOUR ? p.d / 2 : 2 * p.d);
            ev = rows_extent(rows, vst, FOUR ? p.dv / 2 : 2 * p.dv);
            if (FOUR) {
                eks = rows_extent(rows, kss, p.d / 32);
                evs = rows_extent(rows, vss, p.dv / 32);
            }
        }
        const auto rk = buffer_rsrc(at(kh, e, p.c.ks[0], kst), ek);
        const auto rv = buffer_rsrc(at(vh, e, p.c.vs[0], vst), ev);
        if constexpr (!FOUR) {
#pragma unroll
            for (int h = 0; h < n; ++h) {
#pragma unroll
                for (int c = 0; c < DC; ++c)
                    x.k[h0 + h][c] = __builtin_bit_cast(v8, load_once(rk, koff[c] + 16 * h * kst));
#pragma unroll
                for (int i = 0; i < KIT; ++i) x.v[h0 + h][i] = load_once(rv, voff[0] + (16 * h + i * RPP) * vst);
            }
        } else {
            const auto rks = buffer_rsrc(at(ksh, e, p.c.kss[0], kss), eks);
            const auto rvs = buffer_rsrc(at(vsh, e, p.c.vss[0], vss), evs);
#pragma unroll
            for (int h = 0; h < n; ++h) {
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    x.k4[h0 + h][c] = load_once(rk, koff[c] + 16 * h * kst);
                    x.k4s[h0 + h][c] = __builtin_amdgcn_raw_buffer_load_b8(rks, ksoff[c] + 16 * h * kss, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < R4; ++i) {
                    x.v4[h0 + h][i] = load_once(rv, voff[i] + 16 * h * vst);
                    x.v4s[h0 + h][i] = __builtin_amdgcn_raw_buffer_load_b8(rvs, vsoff[i] + 16 * h * vss, 0, 0);
                }
            }
        }
    };
    // A tile lies in one page where pages are whole tiles, else its halves each in one.
    const bool whole = p.c.page % TK == 0;  // (uniform)
    struct Entries {
        Entry half[2];
    };
    auto look_up = [&](int t) __attribute__((always_inline)) {
        Entries e;
        e.half[0] = entry(TK * t);
        e.half[1] = whole ? e.half[0] : entry(TK * t + 16);
        return e;
    };
    Entries next = look_up(slot);  // of the tile to request next
    const Span sp = p.span(seq);
    const int vrows = min(min(sp.lq, p.seq_q) * G, 16 * NQ);
    const int lk = sp.lk;
    if (vrows <= 0) return;  // (uniform)
    const int nt = (lk + TK - 1) / TK;
    auto load_tile = [&](int t) __attribute__((always_inline)) {
        const int rows = lk - TK * t;
        if (whole) {
            request(next.half[0], rows, 0, 2);
        } else {
            request(next.half[0], rows, 0, 1);
            request(next.half[1], rows - 16, 1, 1);
        }
    };

    // This lane's rows: query position and head, and the keys they see.
    int pos[NQ], head[NQ], lim[NQ];
    bool valid[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = 16 * n + l16;
        valid[n] = r < vrows;
        const int rr = valid[n] ? r : 0;
        pos[n] = fwd::fdiv(rr, p.fd_group);
        head[n] = kvh * G + (rr - pos[n] * G);
        lim[n] = p.causal ? min(lk, lk - sp.lq + pos[n] + 1) : lk;
    }
    const int every = p.causal ? min(lk, lk - sp.lq + 1) : lk;  // keys below it are seen by every row
    // A negative scale flips Q's sign, so that the row maximum of the products is that of the
    // logits; a zero one becomes a factor that finite products vanish under.
    const float c2 = fmaxf(fabsf(p.scale_log2), 1e-30f);
    const bool flip = p.scale_log2 < 0.f;
    auto q_row = [&](int n) {
        return static_cast<const T*>(p.q) + head[n] * p.qs[1] + static_cast<int64_t>(sp.q0 + pos[n]) * p.qs[2];
    };
    v8 qf[FOUR ? 1 : NQ][FOUR ? 1 : DC];
    i32x8 q8[FOUR ? NQ : 1][FOUR ? KC : 1][FOUR ? kParts<T> : 1];
    int qsc[FOUR ? NQ : 1];  // scale byte of the first part
    if constexpr (!FOUR) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const int col = 32 * c + 8 * g4;
                const u32x4 x = *reinterpret_cast<const u32x4*>(q_row(n) + min(col, p.d - 8)) ^ (flip ? 0x80008000u : 0u);
                qf[n][c] = __builtin_bit_cast(v8, col < p.d ? x : u32x4{0u, 0u, 0u, 0u});
            }
    } else {
        // The scaled MFMA's B operand: bytes 0 .. 15 of lane (g4, l16) are dims 16 g4 .., bytes
        // 16 .. 31 dims 64 + 16 g4 .. of its 128.
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            v8 x[KC][4];
            float top = 0.f;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int col = 128 * c + 64 * (j >> 1) + 16 * g4 + 8 * (j & 1);
                    const u32x4 raw = *reinterpret_cast<const u32x4*>(q_row(n) + min(col, p.d - 8));
                    x[c][j] = __builtin_bit_cast(v8, col < p.d ? raw : u32x4{0u, 0u, 0u, 0u});
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(to_f32(x[c][j][e])));
                }
            top = max4(top);
            // 2^(E - 7), E the exponent of the row's largest: parts below 256 in magnitude.
            const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 7, 16), 240);
            qsc[n] = e;
            const float inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23) * (flip ? -1.f : 1.f);
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = to_f32(x[c][j][i]) * inv;
#pragma unroll
                    for (int w = 0; w < kParts<T>; ++w) {
#pragma unroll
                        for (int i = 0; i < 8; i += 4) {
                            int b = __builtin_amdgcn_cvt_pk_fp8_f32(y[i], y[i + 1], 0, false);
                            b = __builtin_amdgcn_cvt_pk_fp8_f32(y[i + 2], y[i + 3], b, true);
                            q8[n][c][w][2 * j + i / 4] = b;
                            y[i] = 16.f * (y[i] - __builtin_amdgcn_cvt_f32_fp8(b, 0));
                            y[i + 1] = 16.f * (y[i + 1] - __builtin_amdgcn_cvt_f32_fp8(b, 1));
                            y[i + 2] = 16.f * (y[i + 2] - __builtin_amdgcn_cvt_f32_fp8(b, 2));
                            y[i + 3] = 16.f * (y[i + 3] - __builtin_amdgcn_cvt_f32_fp8(b, 3));
                        }
                    }
                }
        }
    }

    // The first tile, and the entries of the one behind it.
    int t = slot;
    if (t < nt) {
        load_tile(t);
        next = look_up(t + nslots);
    }

    // The tile's V rows into the wavefront's LDS.
    auto stage = [&] {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (!FOUR) {
                if (dg < NCH) {
#pragma unroll
                    for (int i = 0; i < KIT; ++i)
                        *reinterpret_cast<u32x4*>(vl + (16 * h + krow + i * RPP) * VP + 8 * dg) = x.v[h][i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < R4; ++i) {
                    const int ci = lane + kWave * i, r = ci / N4, ch = ci % N4;
                    if (16 * N4 % kWave != 0 && r >= 16) continue;
                    const float s = scale_of(x.v4s[h][i]);
                    T* dst = vl + (16 * h + r) * VP + 32 * ch;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        u32x4 w;
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = fp4_pair<T>(x.v4[h][i][j], s, e);
                        *reinterpret_cast<u32x4*>(dst + 8 * j) = w;
                    }
                }
            }
        }
    };

    f32x4 o[NQ][DB];
    float m[NQ], thr[NQ], neg_m[NQ], lsum[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int d = 0; d < DB; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        m[n] = thr[n] = -INFINITY;
        neg_m[n] = lsum[n] = 0.f;
    }

    for (; t < nt; t += nslots) {
        // LDS keeps one wavefront's accesses in order (the previous tile's reads, these writes,
        // this tile's reads): only the compiler must keep it.
        __asm__ volatile("" ::: "memory");
        stage();
        f32x4 s[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (!FOUR) {
#pragma unroll
                    for (int c = 0; c < DC; ++c) s[n][h] = Mfma16<T>::run(x.k[h][c], qf[n][c], s[n][h]);
                } else {
#pragma unroll
                    for (int w = 0; w < kParts<T>; ++w)
#pragma unroll
                        for (int c = 0; c < KC; ++c) {
                            const i32x4 a = __builtin_bit_cast(i32x4, x.k4[h][c]);
                            // (Format 4: e2m1, its operand in the first four registers; 0: e4m3.)
                            s[n][h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                                __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1), q8[n][c][w], s[n][h], 4, 0, 0,
                                static_cast<int>(x.k4s[h][c]), 0, qsc[n] - 4 * w);
                        }
                }
            }
        // The K operands are consumed and V is in LDS: the next tile's loads overlap the softmax and
        // PV.
        if (t + nslots < nt) {
            load_tile(t + nslots);
            next = look_up(t + 2 * nslots);
        }
        v8 pf[NQ], rest[NQ];  // the weights' two parts
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            // Lane (g4, l16), register i of half h: key 16 h + 4 g4 + i of row l16.
            if (TK * t + TK > every) {
                const int rel = lim[n] - TK * t - 4 * g4;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (16 * h + i >= rel) s[n][h][i] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                             fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
            if (__builtin_amdgcn_ballot_w64(mx * c2 > thr[n])) {
                const float mt = max4(mx) * c2;
                const bool move = mt > thr[n];
                const float alpha = move ? __builtin_amdgcn_exp2f(m[n] - mt) : 1.f;  // 0 while m was -inf
                if (move) {
                    m[n] = mt;
                    thr[n] = mt + kLazy;
                    neg_m[n] = -mt;
                }
                lsum[n] *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[n][d] *= alpha;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][h][i], c2, neg_m[n]));
                    lsum[n] += e;
                    pf[n][4 * h + i] = static_cast<T>(e);
                    rest[n][4 * h + i] = static_cast<T>(e - static_cast<float>(pf[n][4 * h + i]));
                }
        }
        const T* vsrc = vl + (4 * g4 + (l16 >> 2)) * VP + 4 * (l16 & 3);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const u32x2 lo = tr_read(vsrc + 16 * d), hi = tr_read(vsrc + 16 * VP + 16 * d);
            const v8 vf = __builtin_bit_cast(v8, u32x4{lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
            for (int n = 0; n < NQ; ++n) o[n][d] = Mfma16<T>::run(vf, rest[n], Mfma16<T>::run(vf, pf[n], o[n][d]));
        }
    }

    // The wavefronts merge in LDS (the V tiles are done with), 16 rows at a time: every one leaves
    // its state there and combines a share of the dims.
    float* const ex = reinterpret_cast<float*>(smem);
    float* const st = ex + WAVES * 16 * CP;
    constexpr int PER = DP / (4 * WAVES);  // dims of a lane: PER at PER (4 wave + g4) of row l16
    typedef float fper __attribute__((ext_vector_type(PER % 4 == 0 ? 4 : 2)));
    constexpr int VE = PER % 4 == 0 ? 4 : 2;
    const int c0 = PER * (4 * wave + g4);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float l = sum4(lsum[n]);
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DB; ++d) *reinterpret_cast<f32x4*>(ex + (wave * 16 + l16) * CP + 16 * d + 4 * g4) = o[n][d];
        if (g4 == 0) *reinterpret_cast<f32x2*>(st + (wave * 16 + l16) * 2) = f32x2{m[n], l};
        __syncthreads();
        if (!valid[n]) continue;
        f32x2 state[WAVES];
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            state[w] = *reinterpret_cast<const f32x2*>(st + (w * 16 + l16) * 2);
            top = fmaxf(top, state[w][0]);
        }
        float total = 0.f, acc[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            // (By the sum, not the maximum: logits that are all NaN leave that at minus infinity.)
            const float wt = state[w][1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(state[w][0] - top);
            total += wt * state[w][1];
#pragma unroll
            for (int i = 0; i < PER; i += VE) {
                const fper x = *reinterpret_cast<const fper*>(ex + (w * 16 + l16) * CP + c0 + i);
#pragma unroll
                for (int e = 0; e < VE; ++e) acc[i + e] += wt * x[e];
            }
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const int64_t tok = sp.q0 + pos[n];
        if (p.splits == 1) {
            T* dst = static_cast<T*>(p.out) + head[n] * p.os[1] + tok * p.os[2] + c0;
            typedef T tper __attribute__((ext_vector_type(VE)));
#pragma unroll
            for (int i = 0; i < PER; i += VE) {
                tper y;
#pragma unroll
                for (int e = 0; e < VE; ++e) y[e] = from_f32<T>(acc[i + e] * inv);
                if (c0 + i < p.dv) *reinterpret_cast<tper*>(dst + i) = y;
            }
            if (p.lse && wave == 0 && g4 == 0)
                p.lse[head[n] * p.ls[1] + tok * p.ls[2]] = total == 0.f ? -INFINITY : (top + log2f(total)) * kLn2f;
        } else {
            const int64_t at = (static_cast<int64_t>(split) * p.rows_total + tok) * p.hq + head[n];
#pragma unroll
            for (int i = 0; i < PER; i += VE) {
                fper y;
#pragma unroll
                for (int e = 0; e < VE; ++e) y[e] = acc[i + e] * inv;
                if (c0 + i < p.dv) *reinterpret_cast<fper*>(p.part_o + at * DP + c0 + i) = y;
            }
            if (wave == 0 && g4 == 0) p.part_lse[at] = total == 0.f ? -INFINITY : top + log2f(total);
        }
    }
}

template <typename T, int DP, int NQ, bool FOUR>
hipError_t launch_decode_as(const AttnParams& p, hipStream_t stream) {
    constexpr size_t lds = decode_lds<T, DP, NQ>();
    if constexpr (lds > 64 * 1024) {
        const hipError_t attr =
            hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_decode_kernel<T, DP, NQ, FOUR>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        if (attr != hipSuccess) return attr;
    }
    hipLaunchKernelGGL((paged_decode_kernel<T, DP, NQ, FOUR>),
                       dim3(static_cast<unsigned>(p.batch * p.hkv * p.splits + p.tail_blocks)), dim3(THREADS), lds, stream, p);
    return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch_decode(const AttnParams& p, int rows, bool four, hipStream_t stream) {
    if (four) return rows == 16 ? launch_decode_as<T, DP, 1, true>(p, stream) : launch_decode_as<T, DP, 2, true>(p, stream);
    return rows == 16 ? launch_decode_as<T, DP, 1, false>(p, stream) : launch_decode_as<T, DP, 2, false>(p, stream);
}

}  // namespace paged
}  // namespace kmi
