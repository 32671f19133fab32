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
    // The page of a key of a sequence and its row there (uniform).
    __device__ __forceinline__ int page_at(int seq, int key, int& row) const {
        if (head_pages) {
            row = key;
            return seq;
        }
        return clamp_page(entry_at(seq, key, row), c.pages);
    }
    __device__ __forceinline__ const char* k_rows(int seq, int kvh, int key) const {
        int row;
        const int page = page_at(seq, key, row);
        return c.k + page * c.ks[0] + kvh * c.ks[1] + row * c.ks[2];
    }
    __device__ __forceinline__ const char* v_rows(int seq, int kvh, int key) const {
        int row;
        const int page = page_at(seq, key, row);
        return c.v + page * c.vs[0] + kvh * c.vs[1] + row * c.vs[2];
    }
};

// Zeros (and log-sum-exps of minus infinity) for the rows behind the last sequence, in a split
// call through the merge: one workgroup of a call does it.
template <typename T>
__device__ __forceinline__ void zero_tail(const AttnParams& p) {
    if (!p.c.cu) return;
    const int t0 = min(max(uniform_i32(p.c.cu + p.c.batch), 0), p.c.tokens);
    const int vec = p.dv / 4;
    const int64_t n = static_cast<int64_t>(p.c.tokens - t0) * p.hq;
    if (p.splits > 1) {
        for (int64_t i = threadIdx.x; i < n * p.splits; i += blockDim.x) {
            const int64_t s = i / n;
            p.part_lse[(s * p.rows_total + t0) * p.hq + (i - s * n)] = -INFINITY;
        }
        return;
    }
    typedef T t4 __attribute__((ext_vector_type(4)));
    for (int64_t i = threadIdx.x; i < n * vec; i += blockDim.x) {
        const int64_t r = i / vec, t = t0 + r / p.hq, h = r % p.hq;
        *reinterpret_cast<t4*>(static_cast<T*>(p.out) + t * p.os[2] + h * p.os[1] + 4 * (i - r * vec)) = t4{};
    }
    if (p.lse)
        for (int64_t r = threadIdx.x; r < n; r += blockDim.x)
            p.lse[(t0 + r / p.hq) * p.ls[2] + (r % p.hq) * p.ls[1]] = -INFINITY;
}

// Enqueues a call's kernel (the merge is paged_attention.hip's).  rows: 16 or 32 virtual rows a
// workgroup for the decode kernel.
template <typename T, int DP>
hipError_t launch_decode(const AttnParams& p, int rows, bool four, hipStream_t stream);
template <typename T, int DP>
hipError_t launch_tile(const AttnParams& p, int row_groups, hipStream_t stream);

}  // namespace paged
}  // namespace kmi
