// The paged 4-bit key/value cache's layout (declared in include/l3m_kernels.h), shared by the kernels
// that write it (kv4.cu) and read it (kv4_attend.cu).
//
// Why this layout: one tile of 16 tokens of one head is one contiguous piece (2304 bytes for q4_0 at
// head_dim 128), so a warp fetches it with 16-byte copies side by side and a page of one head is a run of tiles.
// Inside it the codes of one token are contiguous, so appending a token writes whole bytes of its own
// and never shares one with a neighbour. The order within a token's row is the order in which the
// tensor-core fragments of m16n8k16 want them: lane 4*g + t of a warp reads, for the key row of its
// token, the contiguous part t (one 32-bit word of 8 dims per block), and for a value row the
// contiguous part g (16 bits of 4 dims per block), with no shuffles between lanes.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>
#include "../../include/l3m_kernels.h"

namespace l3m {

constexpr int kKvTile = 16;      // tokens per cache tile
constexpr int kKvBlock = 32;     // values per quantisation block

struct Kv4Dev {
    uint8_t *data;
    int n_pages, page, tiles, n_kv, dim, ng, sb;      // tiles per page, blocks per row, bytes per scale
    int tile_bytes;
    __host__ __device__ size_t tile_at(int page_id, int head, int tile) const {
        return (((size_t)page_id * n_kv + head) * tiles + tile) * tile_bytes;
    }
    __host__ __device__ int k_scales() const { return 512 * ng; }
    __host__ __device__ int v_scales() const { return 512 * ng + kKvTile * ng * sb; }
};

inline const char *kv4_shape_error(const l3m_kv4 *c) {
    if (!c) return "a cache is required";
    if (c->dtype != L3M_DT_Q4_0 && c->dtype != L3M_DT_MXFP4) return "the cache's dtype is q4_0 or mxfp4";
    if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8) return "head_dim must be a multiple of 8 from 8 to 256";
    if (c->n_kv_heads < 1 || c->n_kv_heads > 65535) return "n_kv_heads must be 1 to 65535";
    if (c->page < kKvTile || c->page > 4096 || c->page % kKvTile) return "page must be a multiple of 16 from 16 to 4096";
    if (c->n_pages < 0 || (int64_t)c->n_pages * c->page > 0x7fffffff) return "n_pages * page must be below 2^31";
    return nullptr;
}

inline const char *kv4_error(const l3m_kv4 *c) {
    if (const char *e = kv4_shape_error(c)) return e;
    if (!c->data || ((uintptr_t)c->data & 15)) return "the cache's data must be 16-byte aligned device memory";
    if ((int64_t)c->n_pages * c->n_kv_heads * (c->page / kKvTile) > 0x7fffffff) return "the cache must have fewer than 2^31 tiles";
    return nullptr;
}

inline Kv4Dev kv4_dev(const l3m_kv4 *c) {
    Kv4Dev d;
    d.data = (uint8_t *)c->data;
    d.n_pages = c->n_pages;
    d.page = c->page;
    d.tiles = c->page / kKvTile;
    d.n_kv = c->n_kv_heads;
    d.dim = c->head_dim;
    d.ng = (c->head_dim + kKvBlock - 1) / kKvBlock;
    d.sb = c->dtype == L3M_DT_Q4_0 ? 2 : 1;
    d.tile_bytes = d.ng * (512 + 2 * kKvTile * d.sb);
    return d;
}

// What request r asks of an attention call: its first row of q, how many of its rows are looked at, its cached tokens, and its
// first query's position. Rows are cut off at max_q and at the end of q; positions count from the request's own number of them.
struct Queries { int start, nq, kv, at; };
__device__ __forceinline__ Queries queries_of(const l3m_kv4_attend &a, int r) {
    Queries q;
    q.start = a.q_start[r];
    const int count = min(max(a.q_start[r + 1] - q.start, 0), 1 << 30);
    q.nq = min(count, a.max_q);
    if (a.max_rows) q.nq = min(q.nq, max(a.max_rows - q.start, 0));
    q.kv = min(max(a.kv_len[r], 0), a.max_kv);
    q.at = q.kv - count;
    return q;
}

}  // namespace l3m
