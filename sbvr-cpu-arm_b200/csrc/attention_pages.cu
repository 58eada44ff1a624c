// Attention over a KV cache in pages (pages.cu), head_dim 128, any number of query heads per KV head.
//
// Few rows per sequence (tokens x query heads of a KV head, fewer than 64): two kernels.
//   attention_shared_kernel    the pages that the sequences of a group share, once for the rows of all of them: blocks of 128 rows on the
//                              tensor cores (tcgen05), the keys of all blocks cut into equal shares, one per CTA; leaves unnormalised sums
//   attention_own_kernel       every sequence's own keys (all of them where nothing is shared), joined with those sums
// Many rows per sequence (prompts): the first kernel takes the rows of one sequence as its blocks and all keys they attend to.
//
// A part of a softmax is (m, l, o): o = sum of 2^(s - m + 10) v, l = sum of 2^(s - m + 10) over its keys, s the scores times scale * log2(e), all fp32.
// Parts join as M = max m, l = sum l 2^(m - M), o = sum o 2^(m - M); a part without keys has m = -inf, l = 0.
#include <algorithm>
#include <climits>

#include "attention_pages.cuh"

namespace sbvr {

// ---------------------------------------------------------------------------------------------
// A sequence's own keys.  A cluster of `nsplit` CTAs per (sequence, KV head, 16 rows); every warp takes sixteen keys at a time, a running maximum
// and sums of its own: no barrier until the end, when the warps' and the CTAs' parts are joined through (distributed) shared memory.  mma.sync: sixteen rows
// at most share a key, so bytes and latencies bound it, not the products.  Two stages of sixteen keys per warp, 64 KB, three CTAs per SM: 16
// sequences of up to 4000 keys, 8 KV heads (3393 on average, 222 MB) 39.5 us = 5.6 TB/s, 64 of up to 300 (154, 40 MB) 13.5 us = 3.0 TB/s, in a graph of
// calls.  In a loop of calls 44 and 13, with three stages 40 and 15, with two warps per CTA 79 and 16.
// ---------------------------------------------------------------------------------------------
constexpr int AO_STAGES = 2, AO_KEYS = 16, AO_WARPS = 4, AO_PITCH = AO_D + 4;
constexpr int AO_HALF_STAGE = AO_KEYS * AO_D * 2;                            // bytes of K or V of sixteen keys
constexpr int AO_SMEM = AO_WARPS * AO_STAGES * 2 * AO_HALF_STAGE;            // 64 KB; later the warps' sums

__device__ __forceinline__ void ao_ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ao_ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ao_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t ao_map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void ao_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ao_ld_cluster4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float2 ao_ld_cluster2(uint32_t a) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

struct AoJoin {                                    // four dims of a row: parts joined as they come
    float top = -INFINITY, l = 0.0f;
    float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    // N parts whose values are in registers (no keys: m = -inf, l = 0; m = -inf and l = NaN: all scores are)
    template <int N>
    __device__ __forceinline__ void add(const float2 (&ml)[N], const float4 (&v)[N]) {
        float now = top;
#pragma unroll
        for (int i = 0; i < N; ++i) now = fmaxf(now, ml[i].x);
        const float c = top == -INFINITY ? (l != l ? 1.0f : 0.0f) : ao_exp2(top - now);
        top = now;
        o.x *= c, o.y *= c, o.z *= c, o.w *= c, l *= c;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float f = ml[i].x == -INFINITY ? (ml[i].y != ml[i].y ? 1.0f : 0.0f) : ao_exp2(ml[i].x - top);
            if (f == 0.0f) continue;               // (what lies there may be anything)
            o.x += f * v[i].x, o.y += f * v[i].y, o.z += f * v[i].z, o.w += f * v[i].w;
            l += f * ml[i].y;
        }
    }
};
__device__ __forceinline__ float2 ao_part_ml(const float* part, int rows, int row) {
    return *reinterpret_cast<const float2*>(part + (size_t)rows * AO_D + (size_t)row * 2);
}
__device__ __forceinline__ float4 ao_part_o(const float* part, int rows, int row, int d4) {
    return *reinterpret_cast<const float4*>(part + ((size_t)d4 * rows + row) * 4);
}
// n parts of a row, eight at a time on their way
__device__ __forceinline__ void ao_join_parts(AoJoin& j, const float* part, int n, int rows, int row, int d4) {
    for (int c0 = 0; c0 < n; c0 += 8) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float* at = part + (size_t)min(c0 + c, n - 1) * ao_place_floats(rows);
            ml[c] = ao_part_ml(at, rows, row);
            v[c] = ao_part_o(at, rows, row, d4);
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c0 + c >= n) ml[c] = make_float2(-INFINITY, 0.0f);
        j.add(ml, v);
    }
}
// `on`: the row attends to a key (else: zeros).  Scores that are all -inf leave l = 0 and o = 0: NaN, as zero over zero is.
__device__ __forceinline__ void ao_put(const AoParams& p, int token, int head, int d4, const AoJoin& j, bool on) {
    const float inv = 1.0f / j.l;
    const __half2 a = __floats2half2_rn(on ? j.o.x * inv : 0.0f, on ? j.o.y * inv : 0.0f), b = __floats2half2_rn(on ? j.o.z * inv : 0.0f, on ? j.o.w * inv : 0.0f);
    *reinterpret_cast<uint2*>(p.out + ((size_t)token * p.n_heads + head) * AO_D + d4 * 4) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

__global__ void __launch_bounds__(AO_WARPS * 32) attention_own_kernel(const AoParams p, int nsplit) {
    extern __shared__ __align__(128) unsigned char ao_smem[];
    __shared__ float2 ml_s[AO_WARPS][16];          // a warp's m, l
    __shared__ __align__(16) float2 ml_c[16];      // the CTA's
    __shared__ bool on_s[16];                      // rows that attend to a key
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int rps = p.tps * p.R, nrb = (rps + 15) / 16;
    const int unit = (int)blockIdx.x / nsplit, rank = (int)blockIdx.x - unit * nsplit;
    const int rb = unit % nrb, kvh = (unit / nrb) % p.c.n_kv, seq = unit / (nrb * p.c.n_kv);
    const int row0 = rb * 16, nrows = min(16, rps - row0);
    // Behind the first kernel this one starts when that one's CTAs have all begun, which they do when everything in front of them has ended: only
    // the parts are waited for, and last.
    pdl_launch_dependents();
    const bool behind = p.starts != nullptr;
    if (!behind) pdl_wait();
    const int slot = ao_slot(p, seq);
    int lim[2];
    const __half* qrow[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = min(g + 8 * h, nrows - 1) + row0, tok = r / p.R;
        lim[h] = g + 8 * h < nrows ? ao_limit(p, __ldg(p.positions + (size_t)seq * p.tps + tok)) : 0;
        qrow[h] = p.q + ((size_t)seq * p.tps + tok) * p.q_pitch + ((size_t)kvh * p.R + (r - tok * p.R)) * AO_D;
    }
    if (tid < 32 && t4 == 0) on_s[g] = lim[0] > 0, on_s[g + 8] = lim[1] > 0;
    const int most = __reduce_max_sync(0xffffffffu, max(lim[0], lim[1]));
    const int least = __reduce_min_sync(0xffffffffu, min(g < nrows ? lim[0] : INT_MAX, g + 8 < nrows ? lim[1] : INT_MAX));
    const int seen = __reduce_min_sync(0xffffffffu, min(lim[0] > 0 ? lim[0] : INT_MAX, lim[1] > 0 ? lim[1] : INT_MAX));      // (rows without keys come out as zeros)
    uint32_t q[8][4];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        q[k][0] = *reinterpret_cast<const uint32_t*>(qrow[0] + k * 16 + 2 * t4), q[k][1] = *reinterpret_cast<const uint32_t*>(qrow[1] + k * 16 + 2 * t4);
        q[k][2] = *reinterpret_cast<const uint32_t*>(qrow[0] + k * 16 + 8 + 2 * t4), q[k][3] = *reinterpret_cast<const uint32_t*>(qrow[1] + k * 16 + 8 + 2 * t4);
    }
    AoPiece f = {};
    f.g = -1;
    if (behind) f = ao_find(p, ao_density(p), -1, seq);
    const int blk = f.g < 0 ? 0 : (seq - f.group.s0) / p.per_block, place = f.piece0 + (kvh * f.group.blocks + blk) * f.n;
    const int from = f.g < 0 || place + f.n > p.places ? 0 : f.group.keys;     // tokens that the first kernel takes
    const int step = nsplit * AO_WARPS, chunks = (most + AO_KEYS - 1) / AO_KEYS;
    const uint32_t ring = smem_u32(ao_smem) + warp * (AO_STAGES * 2 * AO_HALF_STAGE);
    const uint64_t policy = nrb == 1 ? ao_read_once() : ao_read_again();
    auto fetch = [&](int ch, int stage) {          // sixteen keys lie in one page
        if (ch < chunks) {
            const int key0 = ch * AO_KEYS, page = ao_page(p, slot, key0 >> p.c.page_shift);
            if (page < 0 && lane == 0) atomicOr(p.c.status, SBVR_PAGES_NO_ENTRY);
            const size_t at = (((size_t)max(page, 0) * p.c.n_kv + kvh) * p.c.page + (key0 & (p.c.page - 1))) * AO_D + (lane & 15) * 8;
            const uint32_t dst = ring + stage * 2 * AO_HALF_STAGE;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = 2 * i + (lane >> 4);
                const uint32_t d = dst + row * 256 + (((lane & 15) ^ (row & 7)) << 4);
                const uint32_t n = page >= 0 && key0 + row < most ? 16u : 0u;      // (behind the last key: zeros)
                asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(d), "l"(p.k + at + (size_t)row * AO_D), "r"(n), "l"(policy) : "memory");
                asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(d + AO_HALF_STAGE), "l"(p.v + at + (size_t)row * AO_D), "r"(n), "l"(policy) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[16][4];
#pragma unroll
    for (int n = 0; n < 16; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    int ch = from / AO_KEYS + rank * AO_WARPS + warp, stage = 0;
#pragma unroll
    for (int s = 0; s < AO_STAGES - 1; ++s) fetch(ch + s * step, s);
    for (; ch < chunks; ch += step) {
        fetch(ch + (AO_STAGES - 1) * step, stage == 0 ? AO_STAGES - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(AO_STAGES - 1) : "memory");
        __syncwarp();
        const uint32_t ks = ring + stage * 2 * AO_HALF_STAGE, vs = ks + AO_HALF_STAGE;
        float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        {
            const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                uint32_t b[4];
                ao_ldsm4(ks + row * 256 + (((2 * k + ((lane >> 3) & 1)) ^ (row & 7)) << 4), b);
                ao_mma(s[0], q[k], b[0], b[1]);
                ao_mma(s[1], q[k], b[2], b[3]);
            }
        }
        const int key0 = ch * AO_KEYS;
        uint32_t w[4];
        float f[2][4];                             // weights of rows g and g + 8: keys 2 t4, + 1, + 8, + 9
        float corr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x[4] = {__fmul_rn(s[0][2 * h], p.sl2), __fmul_rn(s[0][2 * h + 1], p.sl2), __fmul_rn(s[1][2 * h], p.sl2), __fmul_rn(s[1][2 * h + 1], p.sl2)};
            if (key0 + AO_KEYS > least) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key0 + 2 * t4 + (e & 1) + 8 * (e >> 1) >= lim[h]) x[e] = -INFINITY;
            }
            float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            top = fmaxf(top, m[h]);
            const float base = top == -INFINITY ? 0.0f : top;
            corr[h] = m[h] == -INFINITY ? 0.0f : ao_exp2(m[h] - top);
            m[h] = top;
            l[h] *= corr[h];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[h][e] = ao_exp2((x[e] - base) + AO_LIFT), l[h] += f[h][e];
            const __half2 a = __floats2half2_rn(f[h][0], f[h][1]), b = __floats2half2_rn(f[h][2], f[h][3]);
            w[h] = *reinterpret_cast<const uint32_t*>(&a), w[2 + h] = *reinterpret_cast<const uint32_t*>(&b);
        }
#pragma unroll
        for (int n = 0; n < 16; ++n) o[n][0] *= corr[0], o[n][1] *= corr[0], o[n][2] *= corr[1], o[n][3] *= corr[1];
        bool plain = true;
        if (key0 + AO_KEYS > seen && seen < most) {              // a weight of zero hides finite values only
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t v[4];
                asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(vs + (i * 32 + lane) * 16) : "memory");
#pragma unroll
                for (int e = 0; e < 4; ++e) any |= (v[e] & 0x7c007c00u) + 0x04000400u;     // (an exponent of all ones: bit 15)
            }
            plain = !__any_sync(0xffffffffu, any & 0x80008000u);
        }
        if (plain) {
            const int row = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                uint32_t b[4];
                ao_ldsm4t(vs + row * 256 + (((2 * n + (lane >> 4)) ^ (row & 7)) << 4), b);
                ao_mma(o[2 * n], w, b[0], b[1]);
                ao_mma(o[2 * n + 1], w, b[2], b[3]);
            }
        } else {
#pragma unroll 1
            for (int key = 0; key < AO_KEYS; ++key) {
                float wt[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float mine = (key & 8) ? ((key & 1) ? f[h][3] : f[h][2]) : ((key & 1) ? f[h][1] : f[h][0]);
                    wt[h] = __shfl_sync(0xffffffffu, mine, (lane & 28) | ((key & 7) >> 1));
                }
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    uint32_t v;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(vs + key * 256 + ((n ^ (key & 7)) << 4) + t4 * 4) : "memory");
                    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&v));
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (key0 + key < lim[h]) o[n][2 * h] += wt[h] * x.x, o[n][2 * h + 1] += wt[h] * x.y;
                }
            }
        }
        __syncwarp();                              // read before the next copy writes there
        stage = stage + 1 == AO_STAGES ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // ------------------------------ the parts of the warps ------------------------------
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    __syncthreads();                               // every warp is done with its ring
    float* o_s = reinterpret_cast<float*>(ao_smem);                // [warp][16][AO_PITCH]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (t4 == 0) ml_s[warp][g + 8 * h] = make_float2(m[h], l[h]);
        if (g + 8 * h < nrows) {
#pragma unroll
            for (int n = 0; n < 16; ++n)
                *reinterpret_cast<float2*>(o_s + ((warp * 16 + g + 8 * h) * AO_PITCH + n * 8 + 2 * t4)) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        }
    }
    __syncthreads();
    for (int it = tid; it < nrows * 32; it += AO_WARPS * 32) {     // four dims of a row
        const int r = it / 32, d = (it & 31) * 4;
        AoJoin j;
        float2 ml[AO_WARPS];
        float4 v[AO_WARPS];
#pragma unroll
        for (int w = 0; w < AO_WARPS; ++w) ml[w] = ml_s[w][r], v[w] = *reinterpret_cast<const float4*>(o_s + (w * 16 + r) * AO_PITCH + d);
        j.add(ml, v);
        *reinterpret_cast<float4*>(o_s + r * AO_PITCH + d) = j.o;  // (warp 0's place, read by this thread)
        if (d == 0) ml_c[r] = make_float2(j.top, j.l);
    }
    if (nsplit > 1) ao_cluster_sync();
    else __syncthreads();
    // ------------------------------ the parts of the CTAs and of the first kernel ------------------------------
    if (behind) pdl_wait();
    const int prow = (seq - f.group.s0 - blk * p.per_block) * rps + row0;
    const float* part = p.part + (size_t)place * ao_place_floats(p.rows);
    const uint32_t ob = smem_u32(o_s), mb = smem_u32(ml_c);
    for (int it = rank * AO_WARPS * 32 + tid; it < nrows * 32; it += nsplit * AO_WARPS * 32) {
        const int r = it % nrows, d4 = it / nrows;
        AoJoin j;
        for (int w0 = 0; w0 < nsplit; w0 += 4) {
            float2 ml[4];
            float4 v[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int c = min(w0 + w, nsplit - 1);
                ml[w] = ao_ld_cluster2(ao_map_rank(mb + r * 8, c)), v[w] = ao_ld_cluster4(ao_map_rank(ob + (r * AO_PITCH + d4 * 4) * 4, c));
                if (w0 + w >= nsplit) ml[w] = make_float2(-INFINITY, 0.0f);
            }
            j.add(ml, v);
        }
        if (from > 0) ao_join_parts(j, part, f.n, p.rows, prow + r, d4);
        const int row = row0 + r, tok = row / p.R;
        ao_put(p, seq * p.tps + tok, kvh * p.R + (row - tok * p.R), d4, j, on_s[r]);
    }
    if (nsplit > 1) ao_cluster_sync();             // nobody leaves while its sums are read
}

// ---------------------------------------------------------------------------------------------
// The parts of a prompt's blocks, where several CTAs share a block's keys: 32 rows and four dims a warp.
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) attention_join_kernel(const AoParams p, int nsplit) {
    pdl_launch_dependents();
    pdl_wait();
    const int groups = p.rows / 32, block = (int)blockIdx.x / groups, row = ((int)blockIdx.x % groups) * 32 + (threadIdx.x & 31);
    const int nblk = (p.tps * p.R + p.rows - 1) / p.rows, blk = block % nblk, u = block / nblk;
    const int at_row = blk * p.rows + row, tok = at_row / p.R;
    if (tok >= p.tps) return;
    const int kvh = u % p.c.n_kv, seq = u / p.c.n_kv;
    const float* part = p.part + (size_t)block * nsplit * ao_place_floats(p.rows);
    const bool on = ao_limit(p, __ldg(p.positions + (size_t)seq * p.tps + tok)) > 0;
    for (int d4 = threadIdx.x >> 5; d4 < 32; d4 += 8) {
        AoJoin j;
        ao_join_parts(j, part, nsplit, p.rows, row, d4);
        ao_put(p, seq * p.tps + tok, kvh * p.R + (at_row - tok * p.R), d4, j, on);
    }
}

}  // namespace sbvr

using namespace sbvr;

// How a call is carried out.
struct AoPlan {
    bool prompt, shared;                           // rows of a sequence in blocks of their own; the first kernel runs
    int rows, per_block, blocks, nsplit, ctas;     // blocks: of all sequences (prompt), at most (shared)
    size_t places;                                 // of parts
};
static AoPlan ao_plan(const PgCache& c, int seqs, int tps, int n_heads, int groups, int sm_count) {
    AoPlan r = {};
    const long long rps = (long long)tps * (n_heads / c.n_kv);
    // Rows of a block that share their keys, or a sequence's own 16 at a time?  8 KV heads of 4 query heads, 8, 12, 16, 20, 24 tokens each (32 to 96 rows),
    // us as prompts / as few rows.  64 sequences, up to 2000 keys, none shared: 63, 68, 70, 72, 73 / 82, 110, 140, 171, 200.  8 such: 25, 26, 27, 28, 28 /
    // 26, 39, 41, 43, 44.  One on 8000: 35, 37, 38, 39, 39 / 20, 26, 28, 43, 43.  64 on 8000 shared: 232, 267, 281, 294, 296 / 131, 202, 233, 339, 415.
    // The lines lie between 32 and 80 rows.
    r.prompt = rps >= 64;
    if (r.prompt) {
        r.rows = 128;
        r.blocks = (int)(seqs * c.n_kv * ((rps + r.rows - 1) / r.rows));
        r.ctas = 2 * sm_count;
        r.nsplit = std::max(1, std::min(64, r.ctas / r.blocks));
        r.places = r.nsplit > 1 ? (size_t)r.blocks * r.nsplit : 0;
    } else {
        // What sharing can save at most: reading what the slots can hold once per group instead of once per sequence (what they do hold, the device knows).
        // The first kernel costs 9 us, in which the second reads the same keys again, most of them from L2.  With it and without, 8 KV heads, one token:
        // 8 sequences on 1024 tokens (29 MB) 16.6 and 10.4 us, 16 on 1024 (64) 17.1, 15.6, 4 on 8192 (97) 27.4, 25.8, 16 on 2048 (124) 18.8, 24.9, 64 on
        // 1024 (268) 25.4, 36.2; 2 KV heads, 4 on 32 768 (96) 37.4, 42.3; 8 tokens each, 16 on 1024 28.5, 28.5, on 2048 31.1, 47.4.  On the wrong side of
        // the line: 128 on 256 (159) 31.5, 23.7; and few tokens in slots that could hold many, 4 of 2 KV heads on 256 15.0, 5.4.
        r.shared = groups > 0 && (long long)(seqs - groups) * c.max_pages * c.page * c.n_kv * (4 * AO_D) > (100 << 20);
        if (r.shared) {
            r.rows = seqs * rps > 128LL * groups ? 256 : 128;
            r.per_block = r.rows / (int)rps;
            r.ctas = r.rows == 128 ? 2 * sm_count : sm_count;
            r.blocks = c.n_kv * (std::min(groups, seqs / 2) + seqs / r.per_block);     // (groups of two and more)
            r.places = (size_t)r.blocks + AS_ROUNDS * r.ctas;  // (ao_density)
        }
        const long long units = (long long)seqs * c.n_kv * ((rps + 15) / 16);
        r.nsplit = 1;                              // CTAs on a sequence's own keys: as many as make about two per SM, at most 16 (a cluster)
        while (r.nsplit < 16 && units * r.nsplit * 2 <= 2 * sm_count) r.nsplit *= 2;
    }
    return r;
}

extern "C" {

int sbvr_pages_attention_scratch_bytes(const sbvr_pages_t* cache, int seqs, int tokens_per_seq, int n_heads, int groups, size_t* bytes) {
    PgCache c;
    int rc = pg_cache(cache, &c);
    if (rc) return rc;
    if (!bytes || seqs < 1 || tokens_per_seq < 1 || n_heads < 1 || groups < 0 || n_heads % c.n_kv) return SBVR_ERR_BAD_ARG;
    if ((long long)seqs * tokens_per_seq > INT_MAX / 4 / n_heads) return SBVR_ERR_UNSUPPORTED;
    DeviceInfo di;
    int dev = 0;
    SBVR_CUDA_TRY(cudaGetDevice(&dev));
    rc = device_info(dev, &di);
    if (rc) return rc;
    const AoPlan r = ao_plan(c, seqs, tokens_per_seq, n_heads, groups, di.sm_count);
    *bytes = r.places * ao_place_floats(r.rows) * sizeof(float);
    return SBVR_OK;
}

int sbvr_pages_attention_f16(const sbvr_pages_t* cache, int layer, const void* q, long long q_pitch, const int* slots, const int* positions,
                             const int* group_starts, const int* shared, int groups, void* out, void* scratch, size_t scratch_bytes, int seqs,
                             int tokens_per_seq, int n_heads, float scale, sbvr_stream_t stream) {
    AoParams p = {};
    int rc = pg_cache(cache, &p.c);
    if (rc) return rc;
    const PgCache& c = p.c;
    if (!q || !positions || !out || layer < 0 || layer >= c.layers || seqs < 1 || tokens_per_seq < 1 || n_heads < 1 || n_heads % c.n_kv || groups < 0 ||
        groups > seqs || (groups && (!group_starts || !shared)) || q_pitch < (long long)n_heads * AO_D || !(scale > 0.0f) || scale > 1e30f)
        return SBVR_ERR_BAD_ARG;
    if (!slots && seqs > c.max_seqs) return SBVR_ERR_BAD_ARG;
    if ((long long)seqs * tokens_per_seq > INT_MAX / 4 / n_heads) return SBVR_ERR_UNSUPPORTED;
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scratch)) & 15) || q_pitch % 8) return SBVR_ERR_ALIGN;
    const size_t tokens = (size_t)seqs * tokens_per_seq;         // other CTAs still read q while out is written
    if (pg_overlap(q, ((tokens - 1) * q_pitch + (size_t)n_heads * AO_D) * 2, out, tokens * n_heads * AO_D * 2)) return SBVR_ERR_BAD_ARG;
    DeviceInfo di;
    int dev = 0;
    SBVR_CUDA_TRY(cudaGetDevice(&dev));
    rc = device_info(dev, &di);
    if (rc) return rc;
    const AoPlan r = ao_plan(c, seqs, tokens_per_seq, n_heads, groups, di.sm_count);
    if (r.places && (!scratch || scratch_bytes < r.places * ao_place_floats(r.rows) * sizeof(float))) return SBVR_ERR_WORKSPACE;
    p.k = c.pool + (size_t)layer * 2 * pg_plane(c), p.v = p.k + pg_plane(c);
    p.q = static_cast<const __half*>(q), p.slots = slots, p.positions = positions, p.starts = r.shared ? group_starts : nullptr, p.shared = shared;
    p.out = static_cast<__half*>(out), p.part = static_cast<float*>(scratch), p.q_pitch = q_pitch;
    p.seqs = seqs, p.tps = tokens_per_seq, p.n_heads = n_heads, p.R = n_heads / c.n_kv, p.groups = r.shared ? groups : 0;
    p.sl2 = scale * 1.4426950408889634f;
    p.rows = r.rows, p.per_block = r.per_block, p.ctas = r.ctas, p.places = (int)std::min<size_t>(r.places, INT_MAX);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (r.prompt || r.shared) {
        rc = launch_attention_shared(p, r.prompt, r.nsplit, r.prompt ? r.blocks * r.nsplit : r.ctas, st);
        if (rc) return rc;
    }
    if (r.prompt) {
        if (r.nsplit > 1) SBVR_CUDA_TRY(launch_pdl(attention_join_kernel, dim3((unsigned)(r.blocks * (r.rows / 32))), dim3(256), 0, st, p, r.nsplit));
        return SBVR_OK;
    }
    static SmemOnce once, once_cluster;
    rc = set_max_smem_once(once, attention_own_kernel, AO_SMEM);
    if (!rc) rc = set_attribute_once(once_cluster, attention_own_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);      // (clusters of 16)
    if (rc) return rc;
    const int units = seqs * c.n_kv * ((p.tps * p.R + 15) / 16);
    SBVR_CUDA_TRY(launch_pdl_cluster(attention_own_kernel, dim3((unsigned)(units * r.nsplit)), dim3(AO_WARPS * 32), r.nsplit, (size_t)AO_SMEM, st, p, r.nsplit));
    return SBVR_OK;
}

}  // extern "C"
