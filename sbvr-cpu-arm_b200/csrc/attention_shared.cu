// Attention of blocks of 128 or 256 rows over a paged cache on the fifth-generation tensor cores: keys that a group's sequences share, for the rows of
// all of them, or a prompt's rows over all keys they attend to.  Leaves parts (attention_pages.cuh), or the output where a CTA has all of a block's keys.
//
// A tile is 64 keys:
//   scores   S[128 rows, 64 keys] = q . k, both from shared memory (128-byte swizzle), fp32 in tensor memory
//   weights  a thread per row: 2^(s - reference + 10) in fp32, rounded to fp16 once, stored over S
//   output   O[128 rows, 128 dims] += weights . V, weights from tensor memory, V as it lies in the cache
// The reference of a row is the largest score it has met, but follows it only when that has grown by more than 2^5: then its sums are scaled.
//
// Shared keys: the tiles of all blocks in one list, cut into equal shares, one per CTA; a share may end one block and begin the next.
// Prompts: a CTA per block and part of its tiles, longest blocks first.
//
// Warps: four per 128 rows form weights; one issues the MMAs (one lane); two bring K and V, boxes of a page by TMA (places past the last page: a box
// behind the end, which TMA fills with zeros).  Blocks of 128 rows: two CTAs per SM.  256 rows (two sets of S and O in tensor memory, a tile of K and V
// for both): one.  Every wait is bounded; a CTA in which one runs out, or among whose keys values are not finite that only some rows attend to, multiplies its
// rows out without the tensor cores.
#include <cuda.h>

#include "attention_pages.cuh"
#include "attention_tc.cuh"
#include "tc_stream.cuh"

namespace sbvr {

constexpr uint32_t AS_QBOX = 128 * 128, AS_KBOX = AS_KEYS * 128, AS_TILE = 2 * AS_KBOX;        // boxes of 64 dims, a tile of K or V
constexpr int AS_HDR = 3072;

template <int NT>
struct AsShape {
    static constexpr int ROWS = 128 * NT, STAGES = NT == 1 ? 2 : 5;
    static constexpr int IWARP = 4 * NT, KWARP = IWARP + 1, VWARP = IWARP + 2, THREADS = (4 * NT + 3) * 32;
    static constexpr int SMEM = AS_HDR + NT * 2 * (int)AS_QBOX + STAGES * 2 * (int)AS_TILE;
    static constexpr uint32_t COLS = 256 * NT;
};

struct AsSeg {                                     // what a CTA works on at a time
    int seq0, seq1;                                // sequences whose rows it has (prompt: one)
    int row0;                                      // prompt: first row of the sequence
    int kvh, slot;                                 // slot whose table is read
    int ta, tb;                                    // tiles
    int keys;                                      // 0: as many as its rows attend to (prompt)
    int place;                                     // of its part, -1: the output
};

// row i of the block -> token, query head; false where there is none
__device__ __forceinline__ bool as_row(const AoParams& p, const AsSeg& s, bool prompt, int i, int* token, int* head) {
    const int rps = p.tps * p.R;
    if (prompt) {
        const int r = s.row0 + i, t = r / p.R;
        *token = s.seq0 * p.tps + t, *head = s.kvh * p.R + (r - t * p.R);
        return t < p.tps;
    }
    const int q = i / rps, r = i - q * rps, t = r / p.R;
    *token = (s.seq0 + q) * p.tps + t, *head = s.kvh * p.R + (r - t * p.R);
    return s.seq0 + q < s.seq1;
}

__device__ __forceinline__ void as_store(const AoParams& p, int place, int rows, int row, int dim4, const float4& v) {
    *reinterpret_cast<float4*>(p.part + (size_t)place * ao_place_floats(rows) + ((size_t)dim4 * rows + row) * 4) = v;
}
__device__ __forceinline__ void as_store_ml(const AoParams& p, int place, int rows, int row, float m, float l) {
    *reinterpret_cast<float2*>(p.part + (size_t)place * ao_place_floats(rows) + (size_t)rows * AO_D + (size_t)row * 2) = make_float2(m, l);
}

// all rows of a block without the tensor cores: a warp each, four dims a lane, key by key
__device__ __noinline__ void as_multiply_out(const AoParams& p, const AsSeg& s, bool prompt, int rows, const int* lim_s) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    auto four = [](const uint2& v, float (&f)[4]) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
        f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
    };
    for (int row = warp; row < rows; row += warps) {
        int token, head;
        if (!as_row(p, s, prompt, row, &token, &head)) continue;
        float q[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
        four(*reinterpret_cast<const uint2*>(p.q + (size_t)token * p.q_pitch + (size_t)head * AO_D + lane * 4), q);
        const int end = min(lim_s[row], s.tb * AS_KEYS);
        for (int key = s.ta * AS_KEYS; key < end; ++key) {
            const int page = ao_page(p, s.slot, key >> p.c.page_shift);
            float k[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (page >= 0) {
                const size_t at = (((size_t)page * p.c.n_kv + s.kvh) * p.c.page + (key & (p.c.page - 1))) * AO_D + lane * 4;
                four(*reinterpret_cast<const uint2*>(p.k + at), k);
                four(*reinterpret_cast<const uint2*>(p.v + at), v);
            }
            float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
            for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            x *= p.sl2;
            const float top = fmaxf(m, x), base = top == -INFINITY ? 0.0f : top;
            const float corr = m == -INFINITY ? 0.0f : ao_exp2(m - base), e = ao_exp2(x - base);
            m = top;
            l = l * corr + e;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = o[i] * corr + e * v[i];
        }
        if (s.place >= 0) {
            as_store(p, s.place, rows, row, lane, make_float4(o[0], o[1], o[2], o[3]));
            if (lane == 0) as_store_ml(p, s.place, rows, row, m, l);
        } else {
            const float inv = 1.0f / l;
            const bool on = l > 0.0f || l != l;
            const __half2 a = __floats2half2_rn(on ? o[0] * inv : 0.0f, on ? o[1] * inv : 0.0f), b = __floats2half2_rn(on ? o[2] * inv : 0.0f, on ? o[3] * inv : 0.0f);
            *reinterpret_cast<uint2*>(p.out + ((size_t)token * p.n_heads + head) * AO_D + lane * 4) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
    }
}

template <int NT, bool PROMPT>
__global__ void __launch_bounds__(AsShape<NT>::THREADS, NT == 1 ? 2 : 1)
    attention_shared_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const AoParams p, int nsplit) {
    using W = AsShape<NT>;
    constexpr int ST = W::STAGES, ROWS = W::ROWS;
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t* k_full = reinterpret_cast<uint64_t*>(smem);        // [ST] a tile of K is in shared memory
    uint64_t* v_full = k_full + ST;                              // [ST] of V
    uint64_t* k_empty = v_full + ST;                             // [ST] the scores of all rows are formed
    uint64_t* v_empty = k_empty + ST;                            // [ST] the products of all rows are
    uint64_t* s_full = v_empty + ST;                             // [NT][2] scores are there
    uint64_t* p_full = s_full + 2 * NT;                          // [NT][2] weights are stored
    uint64_t* o_done = p_full + 2 * NT;                          // [NT][2] O has a tile's products
    uint64_t* drained = o_done + 2 * NT;                         // after a time-out
    uint64_t* landed = drained + 1;                              // a tile of V that is looked through before it is given out
    volatile int* dead_s = reinterpret_cast<volatile int*>(smem + 384);
    uint32_t* tmem_s = reinterpret_cast<uint32_t*>(smem + 388);
    volatile int* odd_s = reinterpret_cast<volatile int*>(smem + 392);
    int* most_s = reinterpret_cast<int*>(smem + 396);            // keys that any row attends to, that every row (with keys) does, rows
    int* least_s = most_s + 1;
    int* lim_s = reinterpret_cast<int*>(smem + 512);             // [ROWS]
    const uint32_t q_s = smem_u32(smem) + AS_HDR, k_s = q_s + NT * 2 * AS_QBOX, v_s = k_s + ST * AS_TILE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(k_full + i, 1), mbar_init(v_full + i, 1);
            mbar_init(k_empty + i, 1), mbar_init(v_empty + i, 1);
        }
        for (int i = 0; i < 2 * NT; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 4);
            mbar_init(o_done + i, 1);
        }
        mbar_init(drained, 1), mbar_init(landed, 1);
        *dead_s = 0, *odd_s = 0;
        fence_mbar_init();
    }
    pdl_wait();
    if (warp == W::IWARP) {
        // (only when the kernel in front has ended, and the kernel behind may start only when this one has it: neither can wait for
        // columns that the other holds while the other waits for it to end)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_s)), "r"(W::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        pdl_launch_dependents();                                 // (one warp's says it for the CTA)
        aq_fence_before();
    }
    __syncthreads();
    aq_fence_after();
    const uint32_t tbase = *tmem_s;
    bool ok = true;
    long long x = 0, x_end = 0, total = 0;                       // this CTA's tiles of the list
    int shares = 1;
    if (!PROMPT) {
        ao_find(p, 0, -1, &total);
        shares = ao_shares(p, total);
        if ((int)blockIdx.x < shares) x = ao_first(total, shares, blockIdx.x), x_end = ao_first(total, shares, blockIdx.x + 1);
    } else {
        x_end = 1;
    }
    int looked = 0;                                              // tiles of V that were looked through
    int n0 = 0;                                                  // tiles that went through the rings so far
    int m0[NT];                                                  // ... that a set of 128 rows has seen
#pragma unroll
    for (int i = 0; i < NT; ++i) m0[i] = 0;

    while (x < x_end) {
        // ------------------------------ the next block ------------------------------
        AsSeg s;
        if (PROMPT) {
            const int nblk = (p.tps * p.R + ROWS - 1) / ROWS, part = (int)blockIdx.x % nsplit;
            int u = (int)blockIdx.x / nsplit;
            const int per = p.seqs * p.c.n_kv;
            const int blk = nblk - 1 - u / per;                  // (the last rows have the longest contexts)
            u %= per;
            s.seq0 = u / p.c.n_kv, s.seq1 = s.seq0 + 1, s.kvh = u % p.c.n_kv, s.row0 = blk * ROWS;
            s.slot = ao_slot(p, s.seq0);
            s.ta = part, s.tb = 0, s.keys = 0;
            s.place = nsplit == 1 ? -1 : ((s.seq0 * p.c.n_kv + s.kvh) * nblk + blk) * nsplit + part;
            x = x_end;
        } else {
            long long t;
            const AoFind f = ao_find(p, x, -1, &t);
            const int in = (int)(x - f.tile0), seg = in / f.group.tiles;
            s.ta = in - seg * f.group.tiles;
            s.tb = (int)min((long long)f.group.tiles, s.ta + (x_end - x));
            s.kvh = seg / f.group.blocks;
            s.seq0 = f.group.s0 + (seg % f.group.blocks) * p.per_block, s.seq1 = min(f.group.s1, s.seq0 + p.per_block), s.row0 = 0;
            s.slot = ao_slot(p, f.group.s0), s.keys = f.group.keys;
            s.place = f.seg0 + seg + (int)blockIdx.x;
            x += s.tb - s.ta;
        }
        if (threadIdx.x == 0) *most_s = 0, *least_s = 0x7fffffff, *odd_s = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < ROWS; i += W::THREADS) {
            int token, head, lim = -1;                           // -1: no row
            if (as_row(p, s, PROMPT, i, &token, &head)) {
                lim = ao_limit(p, __ldg(p.positions + token));
                if (!PROMPT) lim = min(lim, s.keys);
            }
            lim_s[i] = lim;
            const int hi = __reduce_max_sync(0xffffffffu, lim), lo = __reduce_min_sync(0xffffffffu, lim > 0 ? lim : 0x7fffffff);
            if (lane == 0) atomicMax(most_s, hi), atomicMin(least_s, lo);
        }
        for (int c = threadIdx.x; c < ROWS * 16; c += W::THREADS) {
            const int row = c >> 4, ch = c & 15;
            int token, head;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (as_row(p, s, PROMPT, row, &token, &head)) v = *reinterpret_cast<const uint4*>(p.q + (size_t)token * p.q_pitch + (size_t)head * AO_D + ch * 8);
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(q_s + (row >> 7) * 2 * AS_QBOX + (ch >> 3) * AS_QBOX + (row & 127) * 128 +
                                                                       (((ch & 7) ^ (row & 7)) << 4)),
                         "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                         : "memory");
        }
        fence_proxy_async();                                     // the MMAs read through the asynchronous proxy
        __syncthreads();
        const int P = PROMPT ? max(*most_s, 0) : s.keys, pmin = *least_s;
        if (PROMPT) {
            const int tiles = (P + AS_KEYS - 1) / AS_KEYS, per = max((tiles + nsplit - 1) / nsplit, nsplit > 1 ? AS_LEAST : 1);
            const int part = s.ta;
            s.ta = min(tiles, part * per), s.tb = min(tiles, s.ta + per);
        }
        const int cnt = s.tb - s.ta;
        const int sets = NT == 1 || lim_s[NT == 1 ? 0 : 128] < 0 ? 1 : 2;      // sets of 128 rows that hold any

        if (*dead_s) {                                           // (a wait ran out before: the rest without the tensor cores)
        } else if (warp == W::KWARP || warp == W::VWARP) {
            // ------------------------------ K, V ------------------------------
            const bool is_k = warp == W::KWARP;
            uint64_t* empty = is_k ? k_empty : v_empty;
            uint64_t* full = is_k ? k_full : v_full;
            const int sh = p.c.page_shift, boxes = sh < 6 ? 64 >> sh : 1, nowhere = p.c.pages * p.c.n_kv * p.c.page;
            const uint32_t box_bytes = AS_KBOX / boxes;
            auto entry = [&](int t) {                            // row of the map where this lane's box of tile t begins
                const int key = t * AS_KEYS + (lane << sh);
                if (lane >= boxes || t >= s.tb || key >= P) return nowhere;
                const int page = ao_page(p, s.slot, key >> sh);
                if (page < 0) {
                    atomicOr(p.c.status, SBVR_PAGES_NO_ENTRY);
                    return nowhere;
                }
                return (page * p.c.n_kv + s.kvh) * p.c.page + (key & (p.c.page - 1));
            };
            int y = entry(s.ta);
            for (int i = 0; i < cnt; ++i) {
                const int n = n0 + i, b = n % ST, next = entry(s.ta + i + 1);
                if (n >= ST && (*dead_s || !mbar_wait_async(empty + b, (uint32_t)(n / ST - 1) & 1u))) ok = false;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                unsigned char* dst = smem + AS_HDR + NT * 2 * AS_QBOX + ((is_k ? 0 : ST) + b) * AS_TILE;
                // Keys that not every row attends to: a weight of zero hides finite values only.  Behind the last key zeros take the place of
                // whatever lies there; in front of it the CTA leaves the tensor cores where a value is not finite.
                const bool look = !is_k && (s.ta + i + 1) * AS_KEYS > pmin;
                uint64_t* bar = look ? landed : full + b;
                if (lane == 0) mbar_arrive_expect_tx(bar, AS_TILE);
                __syncwarp();
                if (lane < boxes) {
                    ts_tma_2d(dst + lane * box_bytes, is_k ? &kmap : &vmap, 0, y, bar);
                    ts_tma_2d(dst + AS_KBOX + lane * box_bytes, is_k ? &kmap : &vmap, 64, y, bar);
                }
                __syncwarp();
                if (look) {
                    uint32_t any = 0;
                    const bool there = mbar_wait_async(landed, (uint32_t)looked & 1u);
                    ++looked;
                    ok = __all_sync(0xffffffffu, there);
                    if (!ok) break;
                    const int last = P - (s.ta + i) * AS_KEYS;   // rows of the tile from here on: nobody's
#pragma unroll 4
                    for (int e = lane; e < (int)AS_TILE / 16; e += 32) {
                        const uint32_t at = v_s + b * AS_TILE + e * 16;
                        if (((e >> 3) & (AS_KEYS - 1)) >= last) {
                            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(at), "r"(0u) : "memory");
                            continue;
                        }
                        uint32_t v[4];
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
#pragma unroll
                        for (int j = 0; j < 4; ++j) any |= (v[j] & 0x7c007c00u) + 0x04000400u;     // (an exponent of all ones: bit 15)
                    }
                    if (any & 0x80008000u) *odd_s = 1;
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + b);
                }
                y = next;
            }
            if (!ok) *dead_s = 1;
        } else if (warp == W::IWARP) {
            // ------------------------------ MMA issuer ------------------------------
            if (elect_one()) {
                constexpr uint32_t QK = (1u << 4) | ((AS_KEYS >> 3) << 17) | ((128 >> 4) << 24);
                constexpr uint32_t PV = (1u << 4) | (1u << 16) | ((AO_D >> 3) << 17) | ((128 >> 4) << 24);     // (bit 16: B is V as it lies)
                const uint32_t qd = (q_s >> 4) | (1u << 16), kd = (k_s >> 4) | (1u << 16), vd = (v_s >> 4) | ((AS_KBOX >> 4) << 16);
                auto scores = [&](int i) {
                    const int n = n0 + i, b = n % ST;
                    if (*dead_s || !mbar_wait_async(k_full + b, (uint32_t)(n / ST) & 1u)) return false;
                    aq_fence_after();
#pragma unroll
                    for (int r = 0; r < NT; ++r) {
                        if (r >= sets) break;
                        const int sb = (m0[r] + i) & 1;
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            aq_mma_ss(tbase + r * 256 + sb * 64, qd + r * (2 * AS_QBOX >> 4) + (k >> 2) * (AS_QBOX >> 4) + (k & 3) * 2,
                                      kd + b * (AS_TILE >> 4) + (k >> 2) * (AS_KBOX >> 4) + (k & 3) * 2, QK, k ? 1u : 0u);
                        aq_commit(s_full + 2 * r + sb);
                    }
                    aq_commit(k_empty + b);
                    return true;
                };
                if (cnt) ok = scores(0);
                for (int i = 0; i < cnt && ok; ++i) {
                    const int n = n0 + i, b = n % ST;
                    // (S of the tile after the next lies over the weights of this one: their MMAs are in front of it)
                    if (i + 1 < cnt && !scores(i + 1)) ok = false;
                    if (ok && !mbar_wait_async(v_full + b, (uint32_t)(n / ST) & 1u)) ok = false;
#pragma unroll
                    for (int r = 0; r < NT; ++r) {
                        if (r >= sets || !ok) break;
                        const int m = m0[r] + i, sb = m & 1;
                        if (!mbar_wait_async(p_full + 2 * r + sb, (uint32_t)(m >> 1) & 1u)) ok = false;
                        if (!ok) break;
                        aq_fence_after();
#pragma unroll
                        for (int k = 0; k < 4; ++k)              // sixteen keys: 2 KB of V, eight columns of weights
                            aq_mma_ts(tbase + r * 256 + 128, tbase + r * 256 + sb * 64 + k * 8, vd + b * (AS_TILE >> 4) + k * 128, PV, (i | k) ? 1u : 0u);
                        aq_commit(o_done + 2 * r + sb);
                    }
                    if (ok) aq_commit(v_empty + b);
                }
                if (!ok) {                                       // MMAs that were issued end before the CTA goes on
                    *dead_s = 1;
                    const long long c0 = clock64();
                    aq_commit(drained);
                    while (!mbar_test(drained, 0u) && clock64() - c0 < 200000000LL) {}
                }
            }
            __syncwarp();
        } else if ((warp >> 2) < sets) {
            // ------------------------------ weights ------------------------------
            const int r = warp >> 2, row = warp * 32 + lane;     // (row of the block: 128 r + 32 (warp % 4) + lane)
            const int lim = lim_s[row];
            const int wmin = __reduce_min_sync(0xffffffffu, lim < 0 ? 0x7fffffff : lim);        // (no rows: anything finite)
            const bool idle = !__any_sync(0xffffffffu, lim > 0);
            const uint32_t mine = tbase + r * 256 + ((uint32_t)((warp & 3) * 32) << 16);
            int mr = 0;
#pragma unroll
            for (int i = 0; i < NT; ++i)
                if (i == r) mr = m0[i];
            const float sl2 = p.sl2;
            float ref = -INFINITY, sum = 0.0f;
            for (int i = 0; i < cnt; ++i) {
                const int m = mr + i, b = m & 1;
                if (*dead_s || !mbar_wait_async(s_full + 2 * r + b, (uint32_t)(m >> 1) & 1u)) ok = false;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                aq_fence_after();
                if (!idle) {
                    uint32_t u[64];
                    aq_ld32(mine + b * 64, u);
                    aq_ld32(mine + b * 64 + 32, u + 32);
                    aq_ld_wait(u);
                    aq_ld_wait(u + 32);
                    const int key0 = (s.ta + i) * AS_KEYS;
                    if (key0 + AS_KEYS > wmin) {                 // some row's keys end inside or before this tile
#pragma unroll
                        for (int e = 0; e < 64; ++e)
                            if (key0 + e >= lim) u[e] = 0xff800000u;
                    }
                    float m4[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) m4[e] = __uint_as_float(u[e]);
#pragma unroll
                    for (int e = 4; e < 64; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(u[e]));
                    const float top = fmaxf(ref, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
                    if (__any_sync(0xffffffffu, (top - ref) * sl2 > 5.0f)) {
                        const float corr = ref == -INFINITY ? 0.0f : ao_exp2((ref - top) * sl2);
                        ref = top;
                        sum *= corr;
                        if (i > 0) {
                            if (!mbar_wait_async(o_done + 2 * r + (b ^ 1), (uint32_t)((m - 1) >> 1) & 1u)) ok = false;
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            aq_fence_after();
#pragma unroll 1
                            for (int c = 0; c < 4; ++c) {
                                uint32_t o[32];
                                aq_ld32(mine + 128 + c * 32, o);
                                aq_ld_wait(o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                aq_st32(mine + 128 + c * 32, o);
                            }
                        }
                    }
                    const float base = (ref == -INFINITY ? 0.0f : ref * sl2) - AO_LIFT;        // a row without any key so far
                    float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    uint32_t w[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float a = ao_exp2(fmaf(__uint_as_float(u[2 * e]), sl2, -base)), c = ao_exp2(fmaf(__uint_as_float(u[2 * e + 1]), sl2, -base));
                        s4[(2 * e) & 3] += a, s4[(2 * e + 1) & 3] += c;
                        const __half2 h = __floats2half2_rn(a, c);
                        w[e] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
                    aq_st32(mine + b * 64, w);
                    aq_st_wait();
                }
                aq_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 2 * r + b);
            }
            if (ok && cnt && !mbar_wait_async(o_done + 2 * r + ((mr + cnt - 1) & 1), (uint32_t)((mr + cnt - 1) >> 1) & 1u)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) *dead_s = 1;
            aq_fence_after();
            const bool direct = s.place < 0;
            const float inv = 1.0f / sum;
            const bool on = sum > 0.0f || sum != sum;
            int token = 0, head = 0;
            const bool here = as_row(p, s, PROMPT, row, &token, &head);
            __half* dst = p.out + ((size_t)token * p.n_heads + head) * AO_D;
#pragma unroll 1
            for (int c = 0; c < 4 && ok; ++c) {
                uint32_t o[32];
                aq_ld32(mine + 128 + c * 32, o);
                aq_ld_wait(o);
                if (!cnt || (direct && !on)) {                   // no key at all
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                if (!direct) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (here) as_store(p, s.place, ROWS, row, c * 8 + e, make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3])));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t h[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float f = on ? inv : 0.0f;
                            const __half2 v = __floats2half2_rn(__uint_as_float(o[8 * e + 2 * j]) * f, __uint_as_float(o[8 * e + 2 * j + 1]) * f);
                            h[j] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        if (here) *reinterpret_cast<uint4*>(dst + c * 32 + e * 8) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                }
                __syncwarp();
            }
            if (ok && !direct && here) as_store_ml(p, s.place, ROWS, row, ref == -INFINITY ? ref : ref * sl2 - AO_LIFT, sum);
            aq_fence_before();
        }
        __syncthreads();
        aq_fence_after();
        n0 += cnt;
#pragma unroll
        for (int i = 0; i < NT; ++i)
            if (i < sets) m0[i] += cnt;
        if (*dead_s) {                                           // copies that were issued land before the CTA goes on
            const long long c0 = clock64();
            while (clock64() - c0 < (1LL << 22)) {}
        }
        if (*odd_s || *dead_s) as_multiply_out(p, s, PROMPT, ROWS, lim_s);
        __syncthreads();
    }
    if (warp == W::IWARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tbase), "r"(W::COLS) : "memory");
}

template <int NT, bool PROMPT>
static int launch_shape(const AoParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap, int nsplit, int grid, cudaStream_t st) {
    static SmemOnce once;
    const int rc = set_max_smem_once(once, attention_shared_kernel<NT, PROMPT>, AsShape<NT>::SMEM);
    if (rc) return rc;
    SBVR_CUDA_TRY(launch_pdl(attention_shared_kernel<NT, PROMPT>, dim3((unsigned)grid), dim3(AsShape<NT>::THREADS), (size_t)AsShape<NT>::SMEM, st, kmap, vmap, p, nsplit));
    return SBVR_OK;
}

int launch_attention_shared(const AoParams& p, bool prompt, int nsplit, int grid, cudaStream_t st) {
    CUtensorMap kmap, vmap;
    const size_t map_rows = (size_t)p.c.pages * p.c.n_kv * p.c.page;
    const int box = p.c.page < AS_KEYS ? p.c.page : AS_KEYS;
    int rc = ts_map_2d(&kmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, p.k, map_rows, AO_D, AO_D * 2, box, 64);
    if (!rc) rc = ts_map_2d(&vmap, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, p.v, map_rows, AO_D, AO_D * 2, box, 64);
    if (rc) return rc;
    if (p.rows == 128) return prompt ? launch_shape<1, true>(p, kmap, vmap, nsplit, grid, st) : launch_shape<1, false>(p, kmap, vmap, nsplit, grid, st);
    return prompt ? launch_shape<2, true>(p, kmap, vmap, nsplit, grid, st) : launch_shape<2, false>(p, kmap, vmap, nsplit, grid, st);
}

}  // namespace sbvr
