// Attention over a paged cache, host side: argument checks, the launch plan, the merge of key
// splits and the C ABI entry points.  The kernels are in paged_decode.hpp (at most 32 virtual
// rows per K/V head) and attention_tile.hpp through paged_tile.hpp (more).
//
// A 4-bit cache under the tile kernel is widened once into a dense copy in the workspace
// (kmi_paged_read's kernel): its rows are read by many row tiles, and the copy's bytes are a few
// percent of what the products take.
#include <algorithm>
#include <cstdlib>

#include "paged_attn.hpp"

namespace kmi {
namespace paged {
namespace {

constexpr int kDecodeTile = 32;

struct Plan {
    bool decode;
    int rows;        // virtual rows of a workgroup
    int row_groups;  // tile kernel: 4 or 2
    int nx;          // row tiles of a unit
    int splits, min_split;
    int dp;
    size_t copy_bytes, part_bytes;
};

int pad_dim(const kmi_paged_attn_args* a) {
    return padded_head_dim(std::max(a->cache.head_dim, a->cache.head_dim_v));
}

// KMI_PAGED_SPLITS=n (read once) pins the key splits.
int splits_override() {
    static const int v = [] {
        const char* e = std::getenv("KMI_PAGED_SPLITS");
        return e ? std::atoi(e) : 0;
    }();
    return v;
}

int64_t capacity_of(const kmi_paged_attn_args* a) {
    return std::min(a->cache.table_width * a->cache.page_size, a->max_k);
}

const char* check_attn(const kmi_paged_attn_args* a) {
    if (!a) return "null args";
    if (const char* why = check_cache(a->cache, true)) return why;
    if (!a->q || !a->out) return "null q or out";
    if (reinterpret_cast<uintptr_t>(a->q) % 16) return "q must be 16-byte aligned";
    if (reinterpret_cast<uintptr_t>(a->out) % 8) return "out must be 8-byte aligned";
    for (int i = 0; i < 2; ++i) {
        if (a->q_stride[i] % 8) return "q strides must be multiples of 8 elements";
        if (a->o_stride[i] % 4) return "out strides must be multiples of 4 elements";
    }
    if (a->heads_q < 1 || a->heads_q > 65536 || a->heads_q % a->cache.heads_kv) return "heads_kv must divide heads_q";
    if (a->max_q < 0 || a->max_q > a->cache.tokens) return "max_q must be at most the token count";
    if (a->max_k < 0) return "max_k must not be negative";
    if (a->max_q * (a->heads_q / a->cache.heads_kv) > (1 << 30)) return "sizes too large";
    return nullptr;
}

// Splits of a decode call over a 16-bit cache: the fewest that keep CUs and wavefronts 85% at work, else
// those that come nearest.  The cache's bytes bound such a call, and a CU with one workgroup more than
// the others, or a wavefront with one tile more, is its end.  Measured (us, in brackets as many splits
// as make two workgroups a CU, rounded up), heads of 128 dims: 48 units (sequences x K/V heads) of 8192
// keys 37.2 (46.6), 80 59.6 (70.8), 24 24.3 (28.8), 16 17.8 (19.6), 128 85.7 (87.0), 250 157 (167), 28
// of 16384 42.7 (53.3), 160 of 4096 57.9 (62.2), 200 77.2 (82.2), 32 17.0 (18.5), 300 of 2048 59.0
// (62.6), 64 16.7 (18.6), 128 of 1024 16.5 (18.1).
int64_t even_splits(int64_t units, int64_t keys, int64_t most) {
    // How much of `slots` is at work while n things take them in rounds.
    const auto share = [](int64_t n, int64_t slots) {
        return n == 0 ? 0. : static_cast<double>(n) / static_cast<double>(slots * ceil_div(n, slots));
    };
    int64_t best = 1;
    double fullest = 0.;
    for (int64_t s = 1; s <= std::min<int64_t>(most, kMaxSplits); ++s) {
        const double full = share(units * s, 256) * share(ceil_div(keys, kDecodeTile), 4 * s);
        if (full > fullest) {
            best = s;
            fullest = full;
        }
        if (full >= 0.85) break;
    }
    return best;
}

// Over a 4-bit cache, whose tiles are small: as near to two workgroups a CU as splits come (us at that,
// at even_splits' where that is another): 48 units of 8192 keys 20.2, 21.6, 80 23.9, 31.7, 24 15.1,
// 15.6, 128 34.5, 43.8, 28 of 16384 21, 26, 160 of 4096 23.5 both, 200 28.4, 28.5, 300 of 2048 23.0,
// 26.0.
int64_t four_bit_splits(int64_t units, int64_t most) {
    return std::min(std::max<int64_t>(1, (512 + units / 2) / std::max<int64_t>(1, units)), most);
}

Plan make_plan(const kmi_paged_attn_args* a) {
    Plan pl{};
    pl.dp = pad_dim(a);
    const int64_t G = a->heads_q / a->cache.heads_kv;
    const int64_t vrows = std::max<int64_t>(1, a->max_q * G), units = a->cache.batch * a->cache.heads_kv;
    const int64_t keys = capacity_of(a);
    int64_t splits;
    if (vrows <= 32) {
        pl.decode = true;
        pl.rows = vrows <= 16 ? 16 : 32;
        pl.nx = 1;
        pl.min_split = kDecodeTile;
        // At most a tile for each of a split's wavefronts, two where there are many splits.
        const int64_t most = std::max(std::min<int64_t>(ceil_div(keys, 4 * kDecodeTile), 8), keys / (8 * kDecodeTile));
        // Splits cost a second launch, 2.7 us of the GPU and 3 of the host; seven tiles a
        // wavefront at head dim 64, the time of three and a half at 128, cost less in one (777
        // keys of 14/2 heads x 64: 7.3 us in a graph, 6.6 in seven, but from the host 8 against 11).
        if (ceil_div(keys, 4 * kDecodeTile) * pl.dp <= 7 * 64)
            splits = 1;
        else
            splits = a->cache.bits == 4 ? four_bit_splits(units, most) : even_splits(units, keys, most);
    } else {
        // Row tiles of the call, from its tokens (a tile begun per unit counts half).
        const auto tiles = [&](int64_t rows) {
            return std::min(ceil_div(vrows, rows) * units,
                            ceil_div(a->cache.tokens * G, rows) * a->cache.heads_kv + units / 2);
        };
        const int64_t t4 = tiles(128), t2 = std::max<int64_t>(1, tiles(64));
        // 128-row workgroups where they fill two thirds of the chip (two a CU, of which head dim 64 takes
        // twice as many; one past 128, of 64 rows).  Prompts from their start do not pay for a merge and take 64
        // rows below a full chip.  Over longer keys splits fill it, of 128 rows unless those are few:
        // as many as make one round, or, where that leaves a quarter of it idle, a round and a half.
        // Measured (us, tiles, whole and in 2, 3, 4, 5, 6, 8, 12 splits; * as planned):
        //   128 rows, head dim 128: 4 x up to 1024 tokens of 32/8 heads over 8192 keys (744) 335*, 353,
        //     358, 371; 5 x 600 of 16/8 over 2100 (400) 70*, 87, 95; 4 x 700 over 3700 (352) 114*, 127,
        //     125; 5 x 500 over 3500 (320) 109, 121, 112*, 118, over 12500 361, 340, 303*, 308; 1 x 1024 of
        //     32/8 over 2048 (256) 56, 53*, 64; 3 x 640 of 16/8 over 8640 (240) 195, 162*, 184, 174, 186;
        //     2 x 777 of 16/8 over 4500 (208) 107, 84*, 105, 97; 1 x 700 of 32/8 over 8700 (176) 195,
        //     139, 160, 143, 137*, 146, over 30700 672, 444, 516, 439, 405*, 427, 400; 2 x 300 of 32/8
        //     over 8300 (160) 186, 133, 105*, 129, 123; 512 of 16/2 over 4600 (64) 106, 63, 49, 44, 48, 44,
        //     44*, 53; 256 of 32/8 over 30256 (64) 657, 339, 233, 182, 188, 172, 154*, 177
        //   of head dim 64: 9 x 500 of 14/2 over 3500 (504) 126, 96*, 111, 107; 6 x 400 over 3400 (264) 78,
        //     73, 67*, 71; 2 x 400 over 3400 (88) 63, 38, 35, 33, 29*, 37, 35, 40
        //   64 rows: 3 x 100 of 16/2 x 128 over 9100 (78) 139, 77, 57, 54, 47, 44*, 58, 52; 8 x 32 over
        //     8224 (64) 127, 71, 53, 45, 46, 43, 40*, 50; 4 x 64 over 4160 (64) 68, 41, 33, 29, 30, 28,
        //     27*, 34; 16 x 16 over 2064 (64) 37, 26, 22, 20*, 22, 22, 23, 29; 300 of 16/2 x 256 over 4300
        //     (76) 107, 65, 51*, 75; 4 x 200 of 16/4 x 192 over 2200 (208) 54*, 67
        //   prompts (64 rows / 128 rows, whole and in 2, 4, 8): 2048 of 14/2 x 64 (224 of 128) 26, 39, 42,
        //     42 / 38, 38, 39, 39; 2 x 700 of 16/2 x 128 (176) 20, 33, 33, 33 / 23, 36, 35, 35; 4 x 2048
        //     of 32/8 x 128 231, 366, .. / 197, 323, ..; 512 of 14/2 x 64 (56 of 64 rows) 10.0, 13.2
        const bool own = a->causal && 2 * a->max_q > keys;
        const int64_t slots = pl.dp <= 128 ? 512 : 256;
        pl.row_groups = 2;
        pl.min_split = 256;
        splits = std::min(slots / t2, std::max(keys / 512, slots / 2 / t2));
        if (own) {
            splits = t2 >= slots / 8 ? 1 : slots / 4 / t2;
            if (pl.dp <= 128 && t4 >= 448) {
                pl.row_groups = 4;
                splits = 1;
            }
        } else if (pl.dp <= 128 && t4 >= 48) {
            pl.row_groups = 4;
            const int64_t more = (840 + t4 / 2) / t4;  // a round and a half
            splits = slots / t4;
            if (pl.dp <= 64)
                splits = std::max(splits, std::min(2 * slots / t4, keys / 1000));
            else if (t4 < slots * 2 / 3 && splits * t4 < slots * 3 / 4 && keys >= 1000 * more)
                splits = more;
        }
        splits = std::max<int64_t>(1, splits);
        pl.rows = 32 * pl.row_groups;
        pl.nx = static_cast<int>(ceil_div(vrows, pl.rows));
    }
    if (splits_override() > 0) splits = splits_override();
    pl.splits = static_cast<int>(
        std::max<int64_t>(1, std::min<int64_t>({splits, int64_t{kMaxSplits}, ceil_div(keys, pl.min_split)})));
    if (a->cache.bits == 4 && !pl.decode)
        pl.copy_bytes = static_cast<size_t>(units) * keys * (a->cache.head_dim + a->cache.head_dim_v) * 2;
    if (pl.splits > 1)
        pl.part_bytes = static_cast<size_t>(pl.splits) * a->cache.tokens * a->heads_q * (pl.dp + 4) * sizeof(float);
    return pl;
}

// The splits' normalised rows weighted by their sums, a (query token, query head) to as many lanes as
// it has vectors of four dims.  Nothing is looked up (every split of every row wrote its
// log-sum-exp), so the first rows are requested beside the sums: one memory round trip.  Rows of
// empty splits are read and dropped.  2 x 777 tokens of 16 x 128 in two splits (26 MB) 6.8 us; a
// wavefront a row with two dims a lane 9.7, with room for eight splits 12.0 (BATCH: in flight).
constexpr int merge_lanes(int dp) { return dp <= 32 ? 8 : dp <= 64 ? 16 : dp <= 128 ? 32 : 64; }
constexpr int MERGE_THREADS = 256;
template <typename T, int DP, int BATCH>
__global__ __launch_bounds__(MERGE_THREADS) void merge_kernel(const AttnParams p) {
    constexpr int LANES = merge_lanes(DP), ROWS = MERGE_THREADS / LANES;
    const int64_t step = p.rows_total * p.hq;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / LANES;
    if (row >= step) return;
    const int lane = threadIdx.x % LANES, d0 = 4 * lane;
    const float* const src = p.part_o + row * DP + min(d0, p.dv - 4);
    float top = -INFINITY, total = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.splits; s0 += BATCH) {
        f32x4 x[BATCH];
        float lse[BATCH];
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
            const int64_t at = min(s0 + s, p.splits - 1) * step;
            x[s] = *reinterpret_cast<const f32x4*>(src + at * DP);
            lse[s] = p.part_lse[at + row];
        }
        float most = top;
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
            if (s0 + s >= p.splits) lse[s] = -INFINITY;
            most = fmaxf(most, lse[s]);
        }
        const float shrink = most == top ? 1.f : __builtin_amdgcn_exp2f(top - most);
        acc *= shrink;
        total *= shrink;
        top = most;
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
            const float w = lse[s] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lse[s] - top);
            total += w;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += w > 0.f ? w * x[s][e] : 0.f;  // (never written where 0)
        }
    }
    const int tok = static_cast<int>(row / p.hq), head = static_cast<int>(row - static_cast<int64_t>(tok) * p.hq);
    if (d0 < p.dv) {
        const float inv = total == 0.f ? 0.f : 1.f / total;
        typedef T t4 __attribute__((ext_vector_type(4)));
        t4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(acc[e] * inv);
        *reinterpret_cast<t4*>(static_cast<T*>(p.out) + head * p.os[1] + tok * p.os[2] + d0) = y;
    }
    if (p.lse && lane == 0)
        p.lse[head * p.ls[1] + tok * p.ls[2]] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
}

template <typename T, int DP>
hipError_t run(const AttnParams& p, const Plan& pl, bool four, hipStream_t stream) {
    const hipError_t err = pl.decode ? launch_decode<T, DP>(p, pl.rows, four, stream)
                                     : launch_tile<T, DP>(p, pl.row_groups, stream);
    if (err != hipSuccess || pl.splits == 1) return err;
    const int64_t rows = p.rows_total * p.hq;
    hipLaunchKernelGGL((pl.splits == 2 ? merge_kernel<T, DP, 2> : merge_kernel<T, DP, 8>),
                       dim3(static_cast<unsigned>(ceil_div(rows, MERGE_THREADS / merge_lanes(DP)))), dim3(MERGE_THREADS), 0,
                       stream, p);
    return hipGetLastError();
}

template <typename T>
hipError_t run_dim(const AttnParams& p, const Plan& pl, bool four, hipStream_t stream) {
    switch (pl.dp) {
        case 32: return run<T, 32>(p, pl, four, stream);
        case 64: return run<T, 64>(p, pl, four, stream);
        case 96: return run<T, 96>(p, pl, four, stream);
        case 128: return run<T, 128>(p, pl, four, stream);
        case 192: return run<T, 192>(p, pl, four, stream);
        default: return run<T, 256>(p, pl, four, stream);
    }
}

// Workgroups that zero the rows behind the last sequence, should there be any: one per 64 KB of
// output (none without offsets, where every row has a sequence).
int tail_blocks(const kmi_paged_attn_args* a) {
    if (!a->cache.cu_seqlens) return 0;
    return static_cast<int>(std::min<int64_t>(512, ceil_div(a->cache.tokens * a->heads_q * a->cache.head_dim_v, 1 << 15)));
}

// Launches hold fewer than 2^32 threads (2^24 workgroups); the tile kernel's rounds its row tiles
// of a unit up to groups of at most 32, fewer than twice as many.
bool grid_fits(const kmi_paged_attn_args* a, const Plan& pl) {
    const double units = static_cast<double>(a->cache.batch) * a->cache.heads_kv;
    const double blocks = units * pl.nx * pl.splits;
    const double rows = static_cast<double>(a->cache.tokens) * a->heads_q;
    return blocks < (1 << 23) - (1 << 15) && (pl.splits == 1 || rows < (1 << 26));
}

}  // namespace
}  // namespace paged
}  // namespace kmi

extern "C" int kmi_paged_attn_workspace_bytes(const kmi_paged_attn_args* a, size_t* bytes) {
    using namespace kmi;
    if (!bytes) return fail(KMI_EINVAL, "kmi_paged_attn_workspace_bytes: null bytes");
    if (const char* why = paged::check_attn(a))
        return fail(KMI_EINVAL, std::string("kmi_paged_attn_workspace_bytes: ") + why);
    const paged::Plan pl = paged::make_plan(a);
    *bytes = pl.copy_bytes + pl.part_bytes;
    return KMI_OK;
}

extern "C" int kmi_paged_attn_kernel(const kmi_paged_attn_args* a, const char** name) {
    using namespace kmi;
    if (!name) return fail(KMI_EINVAL, "kmi_paged_attn_kernel: null name");
    if (const char* why = paged::check_attn(a)) return fail(KMI_EINVAL, std::string("kmi_paged_attn_kernel: ") + why);
    const paged::Plan pl = paged::make_plan(a);
    *name = pl.decode ? (pl.rows == 16 ? "decode16" : "decode32") : (pl.row_groups == 4 ? "tile128" : "tile64");
    return KMI_OK;
}

extern "C" int kmi_paged_attn(const kmi_paged_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace kmi;
    using namespace kmi::paged;
    if (const char* why = check_attn(a)) return fail(KMI_EINVAL, std::string("kmi_paged_attn: ") + why);
    if (a->cache.tokens == 0 || a->cache.batch == 0) return KMI_OK;
    const Plan pl = make_plan(a);
    const size_t need = pl.copy_bytes + pl.part_bytes;
    if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
        return fail(KMI_EWORKSPACE,
                    "kmi_paged_attn: workspace missing, misaligned or smaller than kmi_paged_attn_workspace_bytes");
    if (!grid_fits(a, pl)) return fail(KMI_EINVAL, "kmi_paged_attn: too many workgroups");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t keys = capacity_of(a);
    AttnParams p{};
    p.c = device_cache(a->cache);
    p.c.capacity = static_cast<int>(keys);
    if (keys == 0) {
        // No table entry can be read: any int32 stands for the first one, and no key is.
        p.c.table = a->cache.key_lengths;
        p.c.table_stride = 0;
    }
    const bool copy = pl.copy_bytes > 0;
    if (copy) {
        if (!read_fits(a->cache, keys)) return fail(KMI_EINVAL, "kmi_paged_attn: max_k out of range");
        const int64_t units = a->cache.batch * a->cache.heads_kv;
        char* const kc = static_cast<char*>(workspace);
        char* const vc = kc + static_cast<size_t>(units) * keys * a->cache.head_dim * 2;
        const hipError_t err = launch_read(a->cache, kc, vc, keys, false, s);
        if (err != hipSuccess) return hip_status(err, "kmi_paged_attn");
        p.head_pages = 1;
        p.c.k = kc;
        p.c.v = vc;
        const int64_t d[2] = {a->cache.head_dim, a->cache.head_dim_v};
        for (int w = 0; w < 2; ++w) {
            int64_t* st = w ? p.c.vs : p.c.ks;
            st[2] = d[w] * 2;
            st[1] = keys * st[2];
            st[0] = a->cache.heads_kv * st[1];
        }
    }
    p.q = a->q;
    p.out = a->out;
    p.lse = a->lse;
    p.qs[1] = a->q_stride[1];
    p.qs[2] = a->q_stride[0];
    p.os[1] = a->o_stride[1];
    p.os[2] = a->o_stride[0];
    p.ls[1] = a->lse_stride[0];
    p.ls[2] = a->lse_stride[1];
    // (The tile kernel takes row strides in elements.)
    p.ks[2] = p.c.ks[2] / 2;
    p.vs[2] = p.c.vs[2] / 2;
    p.batch = static_cast<int>(a->cache.batch);
    p.hq = static_cast<int>(a->heads_q);
    p.hkv = static_cast<int>(a->cache.heads_kv);
    p.group = p.hq / p.hkv;
    p.seq_q = static_cast<int>(a->max_q);
    p.d = static_cast<int>(a->cache.head_dim);
    p.dv = static_cast<int>(a->cache.head_dim_v);
    p.causal = a->causal ? 1 : 0;
    p.scale_log2 = static_cast<float>(a->scale * 1.4426950408889634);
    p.splits = pl.splits;
    p.min_split = pl.min_split;
    p.nx = pl.nx;
    p.tail_blocks = tail_blocks(a);
    p.rows_total = a->cache.tokens;
    p.fd_splits = fwd::fast_div(static_cast<uint32_t>(p.splits));
    p.fd_hkv = fwd::fast_div(static_cast<uint32_t>(p.hkv));
    p.fd_group = fwd::fast_div(static_cast<uint32_t>(p.group));
    if (pl.splits > 1) {
        p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.copy_bytes);
        p.part_lse = p.part_o + static_cast<size_t>(pl.splits) * p.rows_total * p.hq * pl.dp;
    }
    const bool four = a->cache.bits == 4;
    const hipError_t err = a->cache.dtype == KMI_BF16 ? run_dim<bf16>(p, pl, four, s) : run_dim<f16>(p, pl, four, s);
    return hip_status(err, "kmi_paged_attn");
}
