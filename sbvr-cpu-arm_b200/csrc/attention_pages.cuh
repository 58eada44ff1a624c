// What the attention kernels on a paged cache share: their parameters, how the rows of a group are cut into blocks and the keys of all blocks
// into equal shares (attention_pages.cu, attention_shared.cu).
#pragma once

#include "common.cuh"
#include "pages.cuh"

namespace sbvr {

constexpr int AO_D = PG_D;
// Weights become fp16 for the second product: half a step, 2^-11, of each.  They are multiplied by 2^10 first, so that what is 2^-24 and more of
// the largest keeps all of its bits; the reference a weight is taken from may lag 2^5 behind the largest: at most 2^15.
constexpr float AO_LIFT = 10.0f;

struct AoParams {
    PgCache c;
    const __half* k;                               // this layer's planes
    const __half* v;
    const __half* q;
    const int* slots;
    const int* positions;
    const int* starts;                             // [groups + 1], NULL: nothing is shared
    const int* shared;                             // [groups]
    __half* out;
    float* part;                                   // [slots of parts][rows][130]
    long long q_pitch;
    int seqs, tps, n_heads, R, groups;
    float sl2;                                     // scale * log2(e)
    int rows, per_block;                           // first kernel: rows of a block, sequences whose rows share one
    int ctas;                                      // ... CTAs, shares of the keys at most
};

__device__ __forceinline__ float ao_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ int ao_slot(const AoParams& p, int seq) {
    const int s = p.slots ? __ldg(p.slots + seq) : seq;
    return s >= 0 && s < p.c.max_seqs ? s : -1;
}
// tokens that a row of a position attends to: none below zero, no more than a slot can hold
__device__ __forceinline__ int ao_limit(const AoParams& p, int position) { return max(0, min(position + 1, p.c.max_pages * p.c.page)); }
// the page of tokens k * page .. of a slot, -1 where the table names none
__device__ __forceinline__ int ao_page(const AoParams& p, int slot, int k) {
    const int e = slot >= 0 ? __ldg(p.c.table + (size_t)slot * p.c.max_pages + k) : -1;
    return e >= 0 && e < p.c.pages ? e : -1;
}
__device__ __forceinline__ int ao_shared(const AoParams& p, int g) {
    const int s = max(0, min(__ldg(p.shared + g), p.c.max_pages * p.c.page));
    return s & ~(p.c.page - 1);
}


// Keys of a tile of the first kernel.
constexpr int AS_KEYS = 64;
constexpr int AS_LEAST = 4;                        // tiles that are worth a CTA of their own

struct AoGroup {
    int s0, s1;                                    // its sequences
    int keys;                                      // shared tokens that are multiplied out in common
    int blocks, tiles;                             // blocks of rows; tiles of a block's keys
};
__device__ __forceinline__ AoGroup ao_group(const AoParams& p, int g) {
    AoGroup r;
    r.s0 = max(0, min(__ldg(p.starts + g), p.seqs)), r.s1 = max(r.s0, min(__ldg(p.starts + g + 1), p.seqs));
    r.keys = r.s1 - r.s0 > 1 ? ao_shared(p, g) : 0;            // (one sequence: its own kernel reads them as well)
    r.blocks = r.keys ? (r.s1 - r.s0 + p.per_block - 1) / p.per_block : 0;
    r.tiles = (r.keys + AS_KEYS - 1) / AS_KEYS;
    return r;
}
// All tiles in order: groups, KV heads, blocks, tiles.  `find` looks for a tile (x) or for the group of a sequence (seq >= 0), a warp together.
struct AoFind {
    AoGroup group;
    int g;                                         // -1: there is none
    long long tile0;                               // first tile of the group
    int seg0;                                      // first (KV head, block) of the group
};
__device__ __forceinline__ long long ao_warp_add(long long v, int lane) {      // inclusive prefix sums
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}
__device__ __forceinline__ AoFind ao_find(const AoParams& p, long long x, int seq, long long* total) {
    const int lane = threadIdx.x & 31;
    AoFind f = {};
    f.g = -1;
    long long tiles = 0;
    int segs = 0;
    for (int base = 0; base < p.groups; base += 32) {
        AoGroup gr = {};
        if (base + lane < p.groups) gr = ao_group(p, base + lane);
        const int segs_of = gr.blocks * p.c.n_kv;
        const long long mine = (long long)segs_of * gr.tiles;
        const long long up = ao_warp_add(mine, lane), sup = ao_warp_add(segs_of, lane);
        const bool hit = base + lane < p.groups && (seq >= 0 ? gr.s0 <= seq && seq < gr.s1 : tiles + up - mine <= x && x < tiles + up);
        const unsigned int any = __ballot_sync(0xffffffffu, hit);
        if (any && f.g < 0) {
            const int l = __ffs(any) - 1;
            f.g = base + l;
            f.group.s0 = __shfl_sync(0xffffffffu, gr.s0, l), f.group.s1 = __shfl_sync(0xffffffffu, gr.s1, l);
            f.group.keys = __shfl_sync(0xffffffffu, gr.keys, l);
            f.group.blocks = __shfl_sync(0xffffffffu, gr.blocks, l), f.group.tiles = __shfl_sync(0xffffffffu, gr.tiles, l);
            f.tile0 = tiles + __shfl_sync(0xffffffffu, up - mine, l);
            f.seg0 = segs + (int)__shfl_sync(0xffffffffu, sup - segs_of, l);
        }
        tiles += __shfl_sync(0xffffffffu, up, 31);
        segs += (int)__shfl_sync(0xffffffffu, sup, 31);
    }
    *total = tiles;
    return f;
}
// CTAs that share `total` tiles, the first tile of one of them, and the CTA of a tile
__device__ __forceinline__ int ao_shares(const AoParams& p, long long total) { return (int)max(1LL, min((long long)p.ctas, total / AS_LEAST)); }
__device__ __forceinline__ long long ao_first(long long total, int shares, int c) { return total * c / shares; }
__device__ __forceinline__ int ao_share_of(long long total, int shares, long long x) { return (int)(((x + 1) * shares - 1) / total); }

// The part that share c leaves of block `seg`: segments and shares only grow along the tiles, so their sum names a place of its own.
// [place]: O [32 fours of dims][rows][4], then (m, l) [rows][2]
__host__ __device__ inline size_t ao_place_floats(int rows) { return (size_t)rows * (AO_D + 2); }

// prompt: nsplit CTAs per block of a sequence's rows, else `grid` CTAs on what groups share
int launch_attention_shared(const AoParams& p, bool prompt, int nsplit, int grid, cudaStream_t st);

}  // namespace sbvr
