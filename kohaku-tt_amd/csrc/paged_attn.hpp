// Parameters shared by the host side of attention over a paged cache (paged_attention.hip) and
// its kernels (paged_decode.hpp and attention_tile.hpp's, instantiated per padded head dim).
#pragma once

#include "paged.hpp"

namespace kmi {
namespace paged {

constexpr int kMaxSplits = 64;

struct AttnParams : fwd::AttnParams {
    Cache c;
    int min_split;     // the fewest keys of a split
    // Tile kernel's order: row tiles of a group, groups of a unit, sequences longest first.
    int tile_group, tile_groups, sorted, rows_first;
    int tail_blocks;   // workgroups that zero the rows behind the last sequence
    int head_pages;    // 1: c.k / c.v are dense copies [batch, heads_kv, capacity, dim] (no table)
    __device__ __forceinline__ Span span(int seq) const { return span_of(c, seq); }
    // Keys of a split of a sequence with `lk` keys, a multiple of `unit`: the sequence in at most
    // `splits` parts of at least min_split; splits past the last key write empty partials.
    __device__ __forceinline__ int split_keys(int lk, int unit) const {
        const int per = fwd::fdiv(lk + splits - 1, fd_splits);
        return max((max(per, min_split) + unit - 1) / unit * unit, unit);
    }
    // The table entry of a key of a sequence and its row there (uniform; not yet clamp_page'd, so
    // that nothing waits for it before it is used).
    __device__ __forceinline__ int entry_at(int seq, int key, int& row) const {
        const int i = fwd::fdiv(key, c.fd_page);
        row = key - i * c.page;
        return uniform_i32(c.table + seq * c.table_stride + i);
    }
    // A unit's keys and values, for the tile kernel: where rows from a key on lie (uniform).  Page
    // strides are below 2^32 bytes.
    struct Rows {
        const char* k;
        const char* v;
        const int32_t* table;  // null: a dense copy, one page a sequence
        uint32_t k_page, v_page, k_row, v_row;
        int seq, pages, page;
        fwd::FastDiv fd_page;
        __device__ __forceinline__ int page_at(int key, int& row) const {
            if (!table) {
                row = key;
                return seq;
            }
            const int i = fwd::fdiv(key, fd_page);
            row = key - i * page;
            return clamp_page(uniform_i32(table + i), pages);
        }
        __device__ __forceinline__ const char* k_rows(int key) const {
            int row;
            const uint64_t at = static_cast<uint32_t>(page_at(key, row));
            return k + at * k_page + static_cast<uint64_t>(static_cast<uint32_t>(row)) * k_row;
        }
        __device__ __forceinline__ const char* v_rows(int key) const {
            int row;
            const uint64_t at = static_cast<uint32_t>(page_at(key, row));
            return v + at * v_page + static_cast<uint64_t>(static_cast<uint32_t>(row)) * v_row;
        }
    };
    __device__ __forceinline__ Rows rows(int seq, int kvh) const {
        // (A dense copy's sequences may lie further apart than a page stride says.)
        const int64_t base = head_pages ? seq : 0;
        return Rows{c.k + base * c.ks[0] + kvh * c.ks[1],
                    c.v + base * c.vs[0] + kvh * c.vs[1],
                    head_pages ? nullptr : c.table + seq * c.table_stride,
                    head_pages ? 0u : static_cast<uint32_t>(c.ks[0]),
                    head_pages ? 0u : static_cast<uint32_t>(c.vs[0]),
                    static_cast<uint32_t>(c.ks[2]),
                    static_cast<uint32_t>(c.vs[2]),
                    seq,
                    c.pages,
                    c.page,
                    c.fd_page};
    }
};

// Zeros (and log-sum-exps of minus infinity) for the rows behind the last sequence, in a split
// call through the merge, by tail_blocks workgroups of the call.
template <typename T>
__device__ __forceinline__ void zero_tail(const AttnParams& p, int block) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const int vec = p.dv / 4;
    for (int t = min(max(uniform_i32(p.c.cu + p.c.batch), 0), p.c.tokens) + block; t < p.c.tokens; t += p.tail_blocks) {
        if (p.splits > 1) {
            for (int i = threadIdx.x; i < p.hq * p.splits; i += blockDim.x) {
                const int s = i / p.hq;
                p.part_lse[(s * p.rows_total + t) * p.hq + (i - s * p.hq)] = -INFINITY;
            }
            continue;
        }
        T* const row = static_cast<T*>(p.out) + t * p.os[2];
        for (int i = threadIdx.x; i < p.hq * vec; i += blockDim.x) {
            const int h = i / vec;
            *reinterpret_cast<t4*>(row + h * p.os[1] + 4 * (i - h * vec)) = t4{};
        }
        if (p.lse)
            for (int h = threadIdx.x; h < p.hq; h += blockDim.x) p.lse[t * p.ls[2] + h * p.ls[1]] = -INFINITY;
    }
}

// Enqueues a call's kernel (the merge is paged_attention.hip's).  rows: 16 or 32 virtual rows a
// workgroup for the decode kernel.
template <typename T, int DP>
hipError_t launch_decode(const AttnParams& p, int rows, bool four, hipStream_t stream);
template <typename T, int DP>
hipError_t launch_tile(const AttnParams& p, int row_groups, hipStream_t stream);

}  // namespace paged
}  // namespace kmi
