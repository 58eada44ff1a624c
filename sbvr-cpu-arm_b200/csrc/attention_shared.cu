// Attention of blocks of 128 or 256 rows over a paged cache on the fifth-generation tensor cores: keys that a group's sequences share, for the rows of
// all of them, or a prompt's rows over all keys they attend to.  Leaves parts (attention_pages.cuh), or the output where a CTA has all of a block's keys.
//
// A tile is 64 keys:
//   scores   S[128 rows, 64 keys] = q . k, both from shared memory (128-byte swizzle), fp32 in tensor memory
//   weights  a thread per row: 2^(s - reference + 10) in fp32, rounded to fp16 once, stored over S
//   output   O[128 rows, 128 dims] += weights . V, weights from tensor memory, V as it lies in the cache
// The reference of a row is the largest score it has met, but follows it only when the weights of half a tile, 2^10 each for a score like the reference, add up
// to more than 2^15: then its sums are scaled.  Every weight that is kept is at most that, which fp16 holds.
//
// A reference of 2^22 and more has no room for fractions beside it: such a piece is multiplied out without the tensor cores, weights in fp32.
//
// Shared keys: every block's tiles are cut into pieces, one per CTA where that fits (attention_pages.cuh).  Prompts: a CTA per block, or per part of its
// tiles where blocks are few, longest blocks first.
//
// Warps: four per 128 rows form weights; one issues the MMAs (one lane); two bring K and V, boxes of a page by TMA (places past the last page: a box
// behind the end, which TMA fills with zeros).  The roles run through the pieces of a CTA by mbarriers alone.  Blocks of 128 rows: two CTAs per SM.  256 rows
// (two sets of S and O in tensor memory, a tile of K and V for both): one; it is taken where a group has more than 128 rows on average, to read its keys
// half as often: 128 sequences of 4 heads on 65536 keys, calls back to back for a second, 220 us, in blocks of 128 225.  Prompts take 128 rows throughout:
// uneven lengths leave less idle (8 x 300 tokens on 4001: 137 us; an earlier form 151, with 256 rows 164).  Every wait is bounded; a CTA in which one runs out, or among whose keys values are not finite that only
// some rows attend to, multiplies its rows out without the tensor cores.
//
// What bounds it.  Few rows: bytes behind a prologue (pieces, queries, the first keys) and sums: 64 sequences of 4 heads, 16 on 8000 keys each, 132 MB, 36 us
// alone and cold where the bytes need 20.  Many rows: the chain from scores to weights to outputs of a tile, 2260 cycles for 256 rows (128 sequences of 4 heads
// on 65536 keys: 250 000 active cycles of an SM, 110.7 tiles), in which the tensor pipe counts 1024 as active (45 %) and the units for exponentials 1070 (47 %).
// Without exponentials a launch takes as long, with an eighth of the MMAs a tenth less.  Tried without gain: a polynomial for some exponentials, two warps per
// 32 rows, a warp each for the MMAs of S and of O.
#include <cuda.h>

#include <climits>

#include "attention_pages.cuh"
#include "attention_tc.cuh"
#include "tc_stream.cuh"

namespace sbvr {

constexpr uint32_t AS_QBOX = 128 * 128, AS_KBOX = AS_KEYS * 128, AS_TILE = 2 * AS_KBOX;        // boxes of 64 dims, a tile of K or V
constexpr int AS_HDR = 1024;

template <int NT>
struct AsShape {
    static constexpr int ROWS = 128 * NT, STAGES = NT == 1 ? 2 : 5;
    static constexpr int IWARP = 4 * NT, KWARP = IWARP + 1, VWARP = IWARP + 2, THREADS = (4 * NT + 3) * 32;
    static constexpr int SMEM = AS_HDR + NT * 2 * (int)AS_QBOX + STAGES * 2 * (int)AS_TILE;
    static constexpr uint32_t COLS = 256 * NT;
};

__device__ __forceinline__ float as_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 as_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 as_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// the largest of 32 scores
__device__ __forceinline__ float as_top32(const uint32_t* u) {
    float m[4] = {__uint_as_float(u[0]), __uint_as_float(u[1]), __uint_as_float(u[2]), __uint_as_float(u[3])};
#pragma unroll
    for (int e = 4; e < 32; e += 2) m[(e >> 1) & 3] = as_max3(m[(e >> 1) & 3], __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
    return as_max3(fmaxf(m[0], m[1]), m[2], m[3]);
}
// weights 2^(s sl2 - base) of 32 scores as fp16, their sums added to `sum`
__device__ __forceinline__ void as_weights32(const uint32_t* u, float sl2, float base, uint32_t* w, float2 (&sum)[2]) {
    const float2 a = make_float2(sl2, sl2), c = make_float2(-base, -base);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float2 x = as_fma2(make_float2(__uint_as_float(u[2 * e]), __uint_as_float(u[2 * e + 1])), a, c);
        x.x = ao_exp2(x.x), x.y = ao_exp2(x.y);
        sum[e & 1] = as_add2(sum[e & 1], x);
        const __half2 h = __floats2half2_rn(x.x, x.y);
        w[e] = *reinterpret_cast<const uint32_t*>(&h);
    }
}

// One box of a 2-D tensor map, global -> shared, with a policy for L2
__device__ __forceinline__ void as_tma_2d(void* dst_smem, const CUtensorMap* tmap, int c0, int c1, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;"
        ::"r"(smem_u32(dst_smem)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

struct AsSeg {                                     // a piece: what a CTA works on at a time
    int tok0, ntok;                                // tokens whose rows it has
    int row0, rows;                                // its first row among those of the first token, rows
    int kvh, slot;                                 // slot whose table is read
    int ta, tb;                                    // tiles
    int keys;                                      // keys that any row attends to
    int least;                                     // ... that all rows do (which attend to any)
    int place;                                     // of its part, -1: the output
    bool once;                                     // no other piece reads these keys
};

// row i of a piece -> token, query head
__device__ __forceinline__ void as_row(const AoParams& p, const AsSeg& s, int i, int* token, int* head) {
    const int r = s.row0 + i, t = r / p.R;
    *token = s.tok0 + t, *head = s.kvh * p.R + (r - t * p.R);
}
// keys that row i attends to, -1 where there is no such row
template <bool PROMPT>
__device__ __forceinline__ int as_limit(const AoParams& p, const AsSeg& s, int i) {
    if (i >= s.rows) return -1;
    const int lim = ao_limit(p, __ldg(p.positions + s.tok0 + (s.row0 + i) / p.R));
    return PROMPT ? lim : min(lim, s.keys);
}

// piece number `j` of this CTA; false: there are no more.  Every warp finds out by itself.
template <int ROWS, bool PROMPT>
__device__ __forceinline__ bool as_piece(const AoParams& p, float density, int nsplit, int j, AsSeg& s) {
    const int lane = threadIdx.x & 31;
    if (PROMPT) {
        if (j) return false;
        const int rps = p.tps * p.R, nblk = (rps + ROWS - 1) / ROWS, per = p.seqs * p.c.n_kv, u = (int)blockIdx.x / nsplit;
        const int blk = nblk - 1 - u / per, seq = u % per / p.c.n_kv;          // (the last rows have the longest contexts: first)
        s.kvh = u % per % p.c.n_kv;
        s.tok0 = seq * p.tps, s.row0 = blk * ROWS, s.rows = min(ROWS, rps - s.row0);
        const int t0 = s.row0 / p.R;
        s.tok0 += t0, s.row0 -= t0 * p.R;
        s.slot = ao_slot(p, seq);
        s.place = nsplit == 1 ? -1 : ((seq * p.c.n_kv + s.kvh) * nblk + blk) * nsplit + (int)blockIdx.x % nsplit;
        s.keys = INT_MAX, s.once = nblk == 1;
    } else {
        const int piece = (int)blockIdx.x + j * (int)gridDim.x;
        if (piece >= p.places) return false;                     // (only where groups overlap)
        const AoPiece f = ao_find(p, density, piece, -1);
        if (f.g < 0) return false;
        const int in = piece - f.piece0, seg = in / f.n, i = in - seg * f.n, each = f.group.tiles / f.n, more = f.group.tiles - each * f.n;
        s.ta = each * i + min(i, more), s.tb = s.ta + each + (i < more ? 1 : 0);
        s.kvh = seg / f.group.blocks;
        const int seq = f.group.s0 + (seg - s.kvh * f.group.blocks) * p.per_block;
        s.tok0 = seq * p.tps, s.row0 = 0, s.rows = min(p.per_block, f.group.s1 - seq) * p.tps * p.R;
        s.slot = ao_slot(p, f.group.s0), s.keys = f.group.keys;
        s.place = piece, s.once = f.group.blocks == 1;
    }
    s.ntok = (s.row0 + s.rows + p.R - 1) / p.R;
    int hi = 0, lo = INT_MAX;
    for (int t = lane; t < s.ntok; t += 32) {
        const int lim = min(s.keys, ao_limit(p, __ldg(p.positions + s.tok0 + t)));
        hi = max(hi, lim);
        if (lim > 0) lo = min(lo, lim);
    }
    s.least = __reduce_min_sync(0xffffffffu, lo);
    if (PROMPT) {
        s.keys = __reduce_max_sync(0xffffffffu, hi);
        const int tiles = (s.keys + AS_KEYS - 1) / AS_KEYS, per = max((tiles + nsplit - 1) / nsplit, nsplit > 1 ? AS_LEAST : 1);
        s.ta = min(tiles, (int)blockIdx.x % nsplit * per), s.tb = min(tiles, s.ta + per);
    }
    return true;
}

__device__ __forceinline__ void as_store(const AoParams& p, int place, int rows, int row, int dim4, const float4& v) {
    *reinterpret_cast<float4*>(p.part + (size_t)place * ao_place_floats(rows) + ((size_t)dim4 * rows + row) * 4) = v;
}
__device__ __forceinline__ void as_store_ml(const AoParams& p, int place, int rows, int row, float m, float l) {
    *reinterpret_cast<float2*>(p.part + (size_t)place * ao_place_floats(rows) + (size_t)rows * AO_D + (size_t)row * 2) = make_float2(m, l);
}

// all rows of a piece without the tensor cores: a warp each, four dims a lane, key by key
template <bool PROMPT>
__device__ __noinline__ void as_multiply_out(const AoParams& p, const AsSeg& s, int rows) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    auto four = [](const uint2& v, float (&f)[4]) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
        f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
    };
    for (int row = warp; row < s.rows; row += warps) {
        int token, head;
        as_row(p, s, row, &token, &head);
        float q[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
        four(*reinterpret_cast<const uint2*>(p.q + (size_t)token * p.q_pitch + (size_t)head * AO_D + lane * 4), q);
        const int end = min(as_limit<PROMPT>(p, s, row), s.tb * AS_KEYS);
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
            as_store(p, s.place, rows, row, lane, make_float4(o[0] * AO_LIFTED, o[1] * AO_LIFTED, o[2] * AO_LIFTED, o[3] * AO_LIFTED));
            if (lane == 0) as_store_ml(p, s.place, rows, row, m, l * AO_LIFTED);
        } else {
            const float inv = 1.0f / l;
            const bool on = end > 0;                             // (a prompt's rows: all of their keys are this piece's)
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
    uint64_t* q_full = landed + 1;                               // [NT] the queries of a piece are in shared memory
    volatile int* dead_s = reinterpret_cast<volatile int*>(smem + 384);
    uint32_t* tmem_s = reinterpret_cast<uint32_t*>(smem + 388);
    volatile int* odd_s = reinterpret_cast<volatile int*>(smem + 392);          // bit j % 32: piece j has to be multiplied out
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
        for (int i = 0; i < NT; ++i) mbar_init(q_full + i, 4);
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
    const float density = PROMPT ? 0.0f : ao_density(p);
    bool ok = true;
    int n0 = 0;                                                  // tiles that went through the rings so far
    AsSeg s;

    if (warp == W::KWARP || warp == W::VWARP) {
            // ------------------------------ K, V ------------------------------
            const bool is_k = warp == W::KWARP;
            uint64_t* empty = is_k ? k_empty : v_empty;
            uint64_t* full = is_k ? k_full : v_full;
            const int sh = p.c.page_shift, boxes = sh < 6 ? 64 >> sh : 1, nowhere = p.c.pages * p.c.n_kv * p.c.page;
            const uint32_t box_bytes = AS_KBOX / boxes;
            auto entry = [&](int t) {                            // row of the map where this lane's box of tile t begins
                const int key = t * AS_KEYS + (lane << sh);
                if (lane >= boxes || t >= s.tb || key >= s.keys) return nowhere;
                const int page = ao_page(p, s.slot, key >> sh);
                if (page < 0) {
                    atomicOr(p.c.status, SBVR_PAGES_NO_ENTRY);
                    return nowhere;
                }
                return (page * p.c.n_kv + s.kvh) * p.c.page + (key & (p.c.page - 1));
            };
            int looked = 0;                                      // tiles of V that were looked through
            for (int j = 0; ok && as_piece<ROWS, PROMPT>(p, density, nsplit, j, s); ++j) {
              int y = entry(s.ta);
              const uint64_t policy = s.once ? ao_read_once() : ao_read_again();
              for (int t = s.ta; t < s.tb; ++t, ++n0) {
                const int b = n0 % ST, next = entry(t + 1);
                if (n0 >= ST && (*dead_s || !mbar_wait_async(empty + b, (uint32_t)(n0 / ST - 1) & 1u))) ok = false;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                unsigned char* dst = smem + AS_HDR + NT * 2 * AS_QBOX + ((is_k ? 0 : ST) + b) * AS_TILE;
                // Keys that not every row attends to: a weight of zero hides finite values only.  Behind the last key zeros take the place of
                // whatever lies there; in front of it the CTA leaves the tensor cores where a value is not finite.
                const bool look = !is_k && (t + 1) * AS_KEYS > s.least;
                uint64_t* bar = look ? landed : full + b;
                if (lane == 0) mbar_arrive_expect_tx(bar, AS_TILE);
                __syncwarp();
                if (lane < boxes) {
                    as_tma_2d(dst + lane * box_bytes, is_k ? &kmap : &vmap, 0, y, bar, policy);
                    as_tma_2d(dst + AS_KBOX + lane * box_bytes, is_k ? &kmap : &vmap, 64, y, bar, policy);
                }
                __syncwarp();
                if (look) {
                    uint32_t any = 0;
                    const bool there = mbar_wait_async(landed, (uint32_t)looked & 1u);
                    ++looked;
                    ok = __all_sync(0xffffffffu, there);
                    if (!ok) break;
                    const int last = s.keys - t * AS_KEYS;   // rows of the tile from here on: nobody's
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
                        for (int e4 = 0; e4 < 4; ++e4) any |= (v[e4] & 0x7c007c00u) + 0x04000400u;     // (an exponent of all ones: bit 15)
                    }
                    if (any & 0x80008000u) atomicOr(const_cast<int*>(odd_s), 1 << (j & 31));
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + b);
                }
                y = next;
              }
            }
            if (!ok) *dead_s = 1;
        } else if (warp == W::IWARP) {
            // ------------------------------ MMA issuer ------------------------------
            int m0[NT], j0[NT];                                  // tiles and pieces that a set of 128 rows has seen
#pragma unroll
            for (int r = 0; r < NT; ++r) m0[r] = j0[r] = 0;
            for (int j = 0; ok && as_piece<ROWS, PROMPT>(p, density, nsplit, j, s); ++j) {
              const int cnt = s.tb - s.ta, sets = NT == 2 && s.rows > 128 ? 2 : 1;
              if (elect_one()) {
                constexpr uint32_t QK = (1u << 4) | ((AS_KEYS >> 3) << 17) | ((128 >> 4) << 24);
                constexpr uint32_t PV = (1u << 4) | (1u << 16) | ((AO_D >> 3) << 17) | ((128 >> 4) << 24);     // (bit 16: B is V as it lies)
                const uint32_t qd = (q_s >> 4) | (1u << 16), kd = (k_s >> 4) | (1u << 16), vd = (v_s >> 4) | ((AS_KBOX >> 4) << 16);
                auto scores = [&](int r, int i) {                // S of a set of rows: two tiles ahead of its weights
                    const int n = n0 + i, b = n % ST, sb = (m0[r] + i) & 1;
                    if (r == 0 && (*dead_s || !mbar_wait_async(k_full + b, (uint32_t)(n / ST) & 1u))) return false;
                    aq_fence_after();
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        aq_mma_ss(tbase + r * 256 + sb * 64, qd + r * (2 * AS_QBOX >> 4) + (k >> 2) * (AS_QBOX >> 4) + (k & 3) * 2,
                                  kd + b * (AS_TILE >> 4) + (k >> 2) * (AS_KBOX >> 4) + (k & 3) * 2, QK, k ? 1u : 0u);
                    aq_commit(s_full + 2 * r + sb);
                    if (r == sets - 1) aq_commit(k_empty + b);
                    return true;
                };
#pragma unroll
                for (int r = 0; r < NT; ++r)
                    if (r < sets && ok && (*dead_s || !mbar_wait_async(q_full + r, (uint32_t)j0[r] & 1u))) ok = false;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < NT; ++r)
                        if (r < sets && i < cnt && ok) ok = scores(r, i);
                for (int i = 0; i < cnt && ok; ++i) {
                    const int n = n0 + i, b = n % ST;
                    if (!mbar_wait_async(v_full + b, (uint32_t)(n / ST) & 1u)) ok = false;
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
                        if (r == sets - 1) aq_commit(v_empty + b);
                        if (i + 2 < cnt) ok = scores(r, i + 2);  // (over the weights of this tile: their MMAs are in front of it)
                    }
                }
                if (!ok) {                                       // MMAs that were issued end before the CTA goes on
                    *dead_s = 1;
                    const long long c0 = clock64();
                    aq_commit(drained);
                    while (!mbar_test(drained, 0u) && clock64() - c0 < 200000000LL) {}
                }
              }
              ok = __all_sync(0xffffffffu, ok);
              n0 += cnt;
#pragma unroll
              for (int r = 0; r < NT; ++r)
                  if (r < sets) m0[r] += cnt, ++j0[r];
            }
        } else {
            // ------------------------------ weights ------------------------------
            const int r = warp >> 2, row = warp * 32 + lane;     // (row of the block: 128 r + 32 (warp % 4) + lane)
            const uint32_t mine = tbase + r * 256 + ((uint32_t)((warp & 3) * 32) << 16);
            int mr = 0;                                          // tiles that these 128 rows have seen
            for (int j = 0; as_piece<ROWS, PROMPT>(p, density, nsplit, j, s); ++j) {
            const int cnt = s.tb - s.ta;
            if (r && s.rows <= 128) continue;                    // (a piece without rows for this set)
            // The queries of the warp's rows (the scores of the piece before are formed: its output was waited for).
            int token = 0, head = 0;
            const bool here = row < s.rows;
            if (here) as_row(p, s, row, &token, &head);
            {
                const long long from = here ? (long long)token * p.q_pitch + (long long)head * AO_D : -1;
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const int q = 2 * c + (lane >> 4), ch = lane & 15;
                    const long long at = __shfl_sync(0xffffffffu, from, q);
                    const uint32_t dst = q_s + r * 2 * AS_QBOX + (ch >> 3) * AS_QBOX + ((warp & 3) * 32 + q) * 128 + (((ch & 7) ^ (q & 7)) << 4);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p.q + (at < 0 ? 0 : at) + ch * 8), "r"(at < 0 ? 0u : 16u) : "memory");
                }
            }
            const int lim = as_limit<PROMPT>(p, s, row);
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_proxy_async();                                 // the MMAs read through the asynchronous proxy
            aq_fence_before();                                   // (and what was read of the piece before has been)
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + r);
            const int wmin = __reduce_min_sync(0xffffffffu, lim < 0 ? 0x7fffffff : lim);        // (no rows: anything finite)
            const bool idle = !__any_sync(0xffffffffu, lim > 0);
            const float sl2 = p.sl2;
            // Half a tile at a time, the next half on its way.  Weights are formed with the reference there is, and once more, from scores that still stand in
            // tensor memory, where a half's sum turns out too large for it: nothing waits for the largest score.  What a wait or a vote takes is
            // asked for before the work that hides it.  References are whole numbers (of scores times sl2): what was summed up with the last one is
            // scaled by a power of two.
            float ref = -INFINITY, sum = 0.0f;
            uint32_t u[2][32], w[32];
            bool ahead = false;                                  // the first half is on its way
            for (int i = 0; i < cnt; ++i) {
                const int m = mr + i, b = m & 1, key0 = (s.ta + i) * AS_KEYS;
                if (!ahead) {
                    if (*dead_s || !mbar_wait_async(s_full + 2 * r + b, (uint32_t)(m >> 1) & 1u)) ok = false;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    aq_fence_after();
                    if (!idle) aq_ld32(mine + b * 64, u[0]);
                }
                ahead = false;
                if (!idle) {
                    const bool ends = key0 + AS_KEYS > wmin;     // some row's keys end inside or before this tile
                    auto hide = [&](int h) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (key0 + 32 * h + e >= lim) u[h][e] = 0xff800000u;
                    };
                    aq_ld_wait(u[0]);
                    aq_ld32(mine + b * 64 + 32, u[1]);
                    const bool soon = i + 1 < cnt && mbar_test(s_full + 2 * r + (b ^ 1), (uint32_t)((m + 1) >> 1) & 1u);
                    if (ends) hide(0);
                    float2 p0[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}}, p1[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
                    const float base = (ref == -INFINITY ? 0.0f : ref) - AO_LIFT;
                    as_weights32(u[0], sl2, base, w, p0);
                    aq_ld_wait(u[1]);
                    ahead = __all_sync(0xffffffffu, soon);
                    if (ahead) {
                        aq_fence_after();
                        aq_ld32(mine + (b ^ 1) * 64, u[0]);
                    }
                    if (ends) hide(1);
                    as_weights32(u[1], sl2, base, w + 16, p1);
                    float a0 = (p0[0].x + p0[1].x) + (p0[0].y + p0[1].y), a1 = (p1[0].x + p1[1].x) + (p1[0].y + p1[1].y);
                    if (__any_sync(0xffffffffu, fmaxf(a0, a1) > 32768.0f || (ref == -INFINITY && key0 < lim))) {
                        aq_ld_wait(u[0]);                        // (the next tile's first half is asked for again)
                        ahead = false;
                        aq_ld32(mine + b * 64, u[0]);
                        aq_ld_wait(u[0]);
                        if (ends) hide(0);
                        const float now = fmaxf(ref, ceilf(fmaxf(as_top32(u[0]), as_top32(u[1])) * sl2)), corr = ref == -INFINITY ? 0.0f : ao_exp2(ref - now);
                        ref = now;
                        if (fabsf(ref) >= 4194304.0f && fabsf(ref) < INFINITY) atomicOr(const_cast<int*>(odd_s), 1 << (j & 31));
                        sum *= corr;
                        if (i > 0) {
                            if (!mbar_wait_async(o_done + 2 * r + (b ^ 1), (uint32_t)((m - 1) >> 1) & 1u)) ok = false;
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            aq_fence_after();
#pragma unroll 1
                            for (int c = 0; c < 8; ++c) {
                                uint32_t lo[8], hi[8];
                                ts_ld16_issue(mine + 128 + c * 16, lo, hi);
                                ts_wait_ld(lo), ts_wait_ld(hi);
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    lo[e] = __float_as_uint(__uint_as_float(lo[e]) * corr), hi[e] = __float_as_uint(__uint_as_float(hi[e]) * corr);
                                ts_st8(mine + 128 + c * 16, lo[0], lo[1], lo[2], lo[3], lo[4], lo[5], lo[6], lo[7]);
                                ts_st8(mine + 128 + c * 16 + 8, hi[0], hi[1], hi[2], hi[3], hi[4], hi[5], hi[6], hi[7]);
                            }
                        }
                        p0[0] = p0[1] = make_float2(0.0f, 0.0f);
                        const float moved = (ref == -INFINITY ? 0.0f : ref) - AO_LIFT;
                        as_weights32(u[0], sl2, moved, w, p0);
                        as_weights32(u[1], sl2, moved, w + 16, p0);
                        a0 = (p0[0].x + p0[1].x) + (p0[0].y + p0[1].y), a1 = 0.0f;
                    }
                    sum += a0 + a1;
                    aq_st32(mine + b * 64, w);                   // (over scores that are in registers)
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
            const bool on = lim > 0;                             // (scores that are all -inf: zero over zero)
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
            if (ok && !direct && here) as_store_ml(p, s.place, ROWS, row, ref, sum);
            mr += cnt;
            if (!ok) break;
            }
            aq_fence_before();
        }
    // ------------------------------ teardown ------------------------------
    __syncthreads();
    aq_fence_after();
    if (*dead_s) {                                               // copies that were issued land before the CTA leaves
        const long long c0 = clock64();
        while (clock64() - c0 < (1LL << 22)) {}
    }
    if (*dead_s || *odd_s)
        for (int j = 0; as_piece<ROWS, PROMPT>(p, density, nsplit, j, s); ++j)
            if (*dead_s || (*odd_s >> (j & 31)) & 1) as_multiply_out<PROMPT>(p, s, ROWS);
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
    if (prompt) return launch_shape<1, true>(p, kmap, vmap, nsplit, grid, st);
    return p.rows == 128 ? launch_shape<1, false>(p, kmap, vmap, nsplit, grid, st) : launch_shape<2, false>(p, kmap, vmap, nsplit, grid, st);
}

}  // namespace sbvr
