// What the kernels on a KV cache in pages share (pages.cu, attention_pages.cu).
#pragma once

#include "common.cuh"

namespace sbvr {

constexpr int PG_D = 128;                          // head_dim

struct PgCache {                                   // sbvr_pages_t as the kernels take it
    __half* pool;
    int* table;
    int* lengths;
    int* refs;
    int* status;
    int* scratch;
    int layers, pages, page, page_shift, n_kv, max_seqs, max_pages;
};

// Fills `out` from the caller's description, or says what is wrong with it.
int pg_cache(const sbvr_pages_t* c, PgCache* out);

inline bool pg_overlap(const void* a, size_t an, const void* b, size_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + bn && y < x + an;
}

// Elements of one layer's K (or V): the pages of K lie in front of those of V.
__host__ __device__ inline size_t pg_plane(const PgCache& c) { return (size_t)c.pages * c.n_kv * c.page * PG_D; }

}  // namespace sbvr
