// attn_tile over a paged cache: chunks of prompts and drafts of more than 32 virtual rows.
//
// The tile kernel's own pipeline (attention_tile.hpp); a wavefront's rows of a tile come in
// pieces of 16 that each lie in one page, so paging costs a scalar table load per piece.  A call
// with few row tiles splits the keys over workgroups (fp32 partials, merged by a second launch).
//
// Bound as the dense kernel is, by the matrix unit's issue beside the softmax: 4 x up to 1024 tokens
// of 32/8 heads over 8192 keys x 128 335 us (835 TFLOP/s; the packed kernel over the same keys in one
// piece 372, whose order of workgroups shares less in the L2s).
#pragma once

#include "attention_tile.hpp"
#include "paged_attn.hpp"

namespace kmi {
namespace fwd {

template <>
inline constexpr bool kPagedKeys<paged::AttnParams> = true;

// The sequence with the `nth` most keys (the lower index first among equals), found by every
// wavefront for itself: a lane a sequence, up to 64 of them.
__device__ __forceinline__ int sorted_sequence(const paged::AttnParams& p, int nth) {
    const int lane = threadIdx.x & 63;
    const int lk = lane < p.batch ? min(max(p.c.klen[lane], 0), p.c.capacity) : -1;
    int before = 0;
    for (int j = 0; j < p.batch; ++j) {
        const int other = __builtin_amdgcn_readlane(lk, j);
        before += other > lk || (other == lk && j < lane) ? 1 : 0;
    }
    const uint64_t found = __builtin_amdgcn_ballot_w64(lane < p.batch && before == nth);
    return __builtin_amdgcn_readfirstlane(found ? __builtin_ctzll(found) : 0);
}

// Workgroup order.  Row tiles of a unit (sequence, K/V head) read the same keys of a split, so a group
// of them lies on one XCD (block b runs on XCD b % 8), its tiles next to each other, and shares its L2.
// Groups of one size go round the XCDs there and back, each split's on its own (a unit's splits
// together on one XCD left others idle: 3 x 640 tokens of 16/8 heads over 8640 keys x 128 215 us, so
// 162), those with most keys first: the longest sequence's heads, then the next one's; where a causal
// call's keys are mostly its own queries (prompts from their start) the last row tiles of every unit,
// then those before them.  The last workgroups zero the rows behind the last sequence.
template <typename T, int DP, int RG>
__global__ __launch_bounds__(NTHREADS, tile_waves(DP)) void paged_attn_tile_kernel(const paged::AttnParams p) {
    constexpr size_t TILES = 4 * sizeof(T) * Tile<T, DP, tile_keys(DP, RG)>::ELEMS;
    __shared__ __align__(1024) unsigned char smem[TILES];
    const int lin = blockIdx.x;
    if (lin >= static_cast<int>(gridDim.x) - p.tail_blocks) {
        paged::zero_tail<T>(p, gridDim.x - 1 - lin);
        return;
    }
    const int x = lin & 7, s = lin >> 3;
    const int round = s / p.tile_group, i = s - round * p.tile_group;
    const int item = 8 * round + (round & 1 ? 7 - x : x);
    const int units = p.batch * p.hkv, parts = p.tile_groups * p.splits;
    const int unit = p.rows_first ? item % units : item / parts, part = p.rows_first ? item / units : item - unit * parts;
    const int xg = fdiv(part, p.fd_splits), split = part - xg * p.splits;
    const int xi = xg * p.tile_group + i;
    if (unit >= units || part >= parts || xi >= p.nx) return;
    int bh = unit;
    if (p.sorted) {
        const int nth = fdiv(unit, p.fd_hkv);
        bh = sorted_sequence(p, nth) * p.hkv + (unit - nth * p.hkv);
    }
    attn_tile<T, DP, MK_NONE, RG>(p, smem, bh, p.causal ? p.nx - 1 - xi : xi, split);
}

}  // namespace fwd

namespace paged {

template <typename T, int DP>
hipError_t launch_tile(const AttnParams& p_in, int rg, hipStream_t stream) {
    AttnParams p = p_in;
    const int units = p.batch * p.hkv;
    // All row tiles of a unit (32 at most), fewer where that leaves less than 32 groups to deal
    // (4x1024 tokens of 32/8 heads over 8192 keys x 128: groups of 8, 16, 32 tiles 387, 363, 345 us;
    // 512 tokens of 14/2 heads over 8192 keys x 64, 4, 16, 32 tiles 47, 48, 70).
    p.tile_group = 32;
    while (p.tile_group > 1 && (p.tile_group >= 2 * p.nx || units * ((p.nx + p.tile_group - 1) / p.tile_group) < 32))
        p.tile_group /= 2;
    p.rows_first = p.causal && 2 * static_cast<int64_t>(p.seq_q) > p.c.capacity;
    p.tile_groups = (p.nx + p.tile_group - 1) / p.tile_group;
    p.tile_group = (p.nx + p.tile_groups - 1) / p.tile_groups;  // (of one size)
    p.sorted = p.batch > 1 && p.batch <= 64 && static_cast<int64_t>(units) * p.nx * p.splits > 256;
    const int rounds = (units * p.tile_groups * p.splits + 7) / 8;
    const dim3 grid(static_cast<unsigned>(8 * rounds * p.tile_group + p.tail_blocks));
    if constexpr (DP <= 128) {
        if (rg == 4) {
            hipLaunchKernelGGL((fwd::paged_attn_tile_kernel<T, DP, 4>), grid, dim3(fwd::NTHREADS), 0, stream, p);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((fwd::paged_attn_tile_kernel<T, DP, 2>), grid, dim3(fwd::NTHREADS), 0, stream, p);
    return hipGetLastError();
}

}  // namespace paged
}  // namespace kmi
