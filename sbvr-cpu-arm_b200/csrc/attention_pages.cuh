// What the attention kernels on a paged cache share: their parameters, how the rows of a group are cut into blocks and the keys of all blocks
// into equal shares (attention_pages.cu, attention_shared.cu).
#pragma once

#include <climits>

#include "common.cuh"
#include "pages.cuh"

namespace sbvr {

constexpr int AO_D = PG_D;
// Weights become fp16 for the second product: half a step, 2^-11, of each.  They are multiplied by 2^10 first, so that what is 2^-24 and more of
// the largest keeps all of its bits; the reference a weight is taken from may lag 2^5 behind the largest: at most 2^15.  The 2^10 stays in the sums of
// every part and cancels in the end.  It is added to the difference of score and reference, never to the reference alone: from 2^24 on that loses it, and
// from 2^26 on fma(score, scale, -reference) keeps more of the largest score than the reference did: weights that fp16 does not hold.
constexpr float AO_LIFT = 10.0f, AO_LIFTED = 1024.0f;

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
    int ctas, places;                              // ... CTAs of a round, parts there is room for
};

__device__ __forceinline__ float ao_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Keys and values that are read once leave L2 first: what every launch needs again (its instructions above all, tables, queries) stays.  With them in
// the way, 64 sequences on 4 x 8000 shared tokens took 60.0 us instead of 54.6: instructions came from DRAM behind the keys.
__device__ __forceinline__ uint64_t ao_read_once() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ uint64_t ao_read_again() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
    return policy;
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
// Every block's tiles are cut evenly into pieces, as many per block as its share of the tiles is of `rounds` times the CTAs: one round unless another
// number of them ends sooner by AS_EXTRA, what a piece costs on top of its own tiles (queries, the first keys, sums).  A warp works it out together, a lane
// per group; all of this runs once per CTA on a cold instruction cache, so it is kept short (a search for the longest piece, in 64 bits, took 4 us).
constexpr int AS_EXTRA = 6, AS_ROUNDS = 3;
struct AoPiece {
    AoGroup group;
    int g;                                         // -1: there is none
    int n;                                         // pieces of a block
    int piece0;                                    // first piece of the group: its KV heads, blocks, pieces
};
__device__ __forceinline__ AoGroup ao_lane_group(const AoParams& p, int base) {
    AoGroup r = {};
    if (base + (int)(threadIdx.x & 31) < p.groups) r = ao_group(p, base + (threadIdx.x & 31));
    return r;
}
// pieces of a block, for `density` pieces per tile
__device__ __forceinline__ int ao_pieces(const AoGroup& g, float density) {
    return max(1, min((int)(g.tiles * density), (g.tiles + AS_LEAST - 1) / AS_LEAST));
}
__device__ __forceinline__ float ao_density(const AoParams& p) {
    float tiles = 0.0f;
    for (int base = 0; base < p.groups; base += 32) {
        const AoGroup g = ao_lane_group(p, base);
        tiles += (float)g.tiles * (float)(g.blocks * p.c.n_kv);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    const float one = (float)p.ctas / fmaxf(tiles, 1.0f);
    int pieces[AS_ROUNDS] = {}, most[AS_ROUNDS] = {};
    for (int base = 0; base < p.groups; base += 32) {
        const AoGroup g = ao_lane_group(p, base);
#pragma unroll
        for (int r = 0; r < AS_ROUNDS; ++r) {
            const int n = ao_pieces(g, one * (r + 1));
            pieces[r] += n * g.blocks * p.c.n_kv;
            most[r] = max(most[r], (g.tiles + n - 1) / n);
        }
    }
    int best = INT_MAX, rounds = 1;
#pragma unroll
    for (int r = 0; r < AS_ROUNDS; ++r) {
        const int sum = (int)__reduce_add_sync(0xffffffffu, (unsigned int)pieces[r]), top = __reduce_max_sync(0xffffffffu, most[r]);
        const int cost = (sum + p.ctas - 1) / p.ctas * (top + AS_EXTRA);
        if (cost < best) best = cost, rounds = r + 1;
    }
    return one * rounds;
}
// the group of a piece, or (piece < 0) of a sequence
__device__ __forceinline__ AoPiece ao_find(const AoParams& p, float density, int piece, int seq) {
    const int lane = threadIdx.x & 31;
    AoPiece f = {};
    f.g = -1;
    int sum = 0;
#pragma unroll 1
    for (int base = 0; base < p.groups && f.g < 0; base += 32) {
        const AoGroup gr = ao_lane_group(p, base);
        const int n = ao_pieces(gr, density), mine = n * gr.blocks * p.c.n_kv;
        int up = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += y;
        }
        up += sum;
        const unsigned int any = __ballot_sync(0xffffffffu, piece >= 0 ? up - mine <= piece && piece < up : gr.s0 <= seq && seq < gr.s1);
        if (any) {
            const int l = __ffs(any) - 1;
            f.g = base + l;
            f.group.s0 = __shfl_sync(0xffffffffu, gr.s0, l), f.group.s1 = __shfl_sync(0xffffffffu, gr.s1, l);
            f.group.keys = __shfl_sync(0xffffffffu, gr.keys, l);
            f.group.blocks = __shfl_sync(0xffffffffu, gr.blocks, l), f.group.tiles = __shfl_sync(0xffffffffu, gr.tiles, l);
            f.n = __shfl_sync(0xffffffffu, n, l), f.piece0 = __shfl_sync(0xffffffffu, up - mine, l);
        }
        sum = __shfl_sync(0xffffffffu, up, 31);
    }
    return f;
}

// The part that a piece leaves: O [32 fours of dims][rows][4], then (m, l) [rows][2].
__host__ __device__ inline size_t ao_place_floats(int rows) { return (size_t)rows * (AO_D + 2); }

// prompt: nsplit CTAs per block of a sequence's rows, else `grid` CTAs on what groups share
int launch_attention_shared(const AoParams& p, bool prompt, int nsplit, int grid, cudaStream_t st);

}  // namespace sbvr
