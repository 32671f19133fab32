// attn_tile over a paged cache: chunks of prompts and drafts of more than 32 virtual rows.
//
// The tile kernel's own pipeline (attention_tile.hpp); a wavefront's rows of a tile come in
// pieces of 16 that each lie in one page, so paging costs a scalar table load per piece.  A call
// with few row tiles splits the keys over workgroups (fp32 partials, merged by a second launch).
#pragma once

#include "attention_tile.hpp"
#include "paged_attn.hpp"

namespace kmi {
namespace fwd {

template <>
inline constexpr bool kPagedKeys<paged::AttnParams> = true;

// Workgroups: row tiles heaviest first, the splits of a row tile next to each other.  From eight
// units (sequence, K/V head) on, unit u's lie on XCD u % 8 (block b runs on XCD b % 8), so that its
// keys stay in one L2, with each row of tiles' units rotated by the row (ragged sequences would
// otherwise meet the same few units' work row after row).  One more workgroup zeroes the rows
// behind the last sequence.
template <typename T, int DP, int RG>
__global__ __launch_bounds__(NTHREADS, tile_waves(DP)) void paged_attn_tile_kernel(const paged::AttnParams p) {
    constexpr size_t TILES = 4 * sizeof(T) * Tile<T, DP, tile_keys(DP, RG)>::ELEMS;
    __shared__ __align__(1024) unsigned char smem[TILES];
    const int units = p.batch * p.hkv;
    const int lin = blockIdx.x;
    if (lin == static_cast<int>(gridDim.x) - 1) {
        paged::zero_tail<T>(p);
        return;
    }
    int bh, row;  // row: row tile and split
    if (p.xcd_map == 3) {
        const int x = lin & 7, s = lin >> 3;
        const int nxu = (units - x + 7) >> 3;
        if (nxu <= 0) return;
        row = s / nxu;
        if (row >= p.nx * p.splits) return;
        bh = x + 8 * ((s - row * nxu + row) % nxu);
    } else {
        row = fdiv(lin, p.fd_units);
        bh = lin - row * units;
    }
    const int xi = fdiv(row, p.fd_splits), split = row - xi * p.splits;
    attn_tile<T, DP, MK_NONE, RG>(p, smem, bh, p.causal ? p.nx - 1 - xi : xi, split);
}

}  // namespace fwd

namespace paged {

template <typename T, int DP>
hipError_t launch_tile(const AttnParams& p_in, int rg, hipStream_t stream) {
    AttnParams p = p_in;
    const int units = p.batch * p.hkv;
    p.xcd_map = units >= 8 ? 3 : 0;
    const dim3 grid(static_cast<unsigned>((p.xcd_map == 3 ? 8 * ((units + 7) / 8) : units) * p.nx * p.splits + 1));
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
