// Attention over a KV cache in pages (pages.cu), head_dim 128, any number of query heads per KV head.
//
// Few rows per sequence (tokens x query heads of a KV head, fewer than 64): two kernels.
//   attention_shared_kernel    the pages that the sequences of a group share, once for the rows of all of them: blocks of 128 rows on the
//                              tensor cores (tcgen05), the keys of all blocks cut into equal shares, one per CTA; leaves unnormalised sums
//   attention_own_kernel       every sequence's own keys (all of them where nothing is shared), joined with those sums
// Many rows per sequence (prompts): the first kernel takes the rows of one sequence as its blocks and all keys they attend to.
//
// A part of a softmax is (m, l, o): o = sum of 2^(s - m) v, l = sum of 2^(s - m) over its keys, s the scores times scale * log2(e), all fp32.
// Parts join as M = max m, l = sum l 2^(m - M), o = sum o 2^(m - M); a part without keys has m = -inf, l = 0.
#include <cuda.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "pages.cuh"
#include "tc_stream.cuh"

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
    int per_block;                                 // sequences whose rows share a block
    int ctas;                                      // shares of the first kernel
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

// ---------------------------------------------------------------------------------------------
// A sequence's own keys.  A cluster of `nsplit` CTAs per (sequence, KV head, 16 rows); every warp takes sixteen keys at a time, a running maximum
// and sums of its own: no barrier until the end, when the warps' and the CTAs' parts are joined through (distributed) shared memory.
// ---------------------------------------------------------------------------------------------
constexpr int AO_STAGES = 3, AO_KEYS = 16, AO_WARPS = 4;
constexpr int AO_HALF_STAGE = AO_KEYS * AO_D * 2;                            // bytes of K or V of sixteen keys
constexpr int AO_SMEM = AO_WARPS * AO_STAGES * 2 * AO_HALF_STAGE;            // 96 KB; later the warps' sums

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

__global__ void __launch_bounds__(AO_WARPS * 32) attention_own_kernel(const AoParams p, int nsplit) {
    extern __shared__ __align__(128) unsigned char ao_smem[];
    __shared__ float2 ml_s[AO_WARPS][16];          // a warp's m, l
    __shared__ __align__(16) float2 ml_c[16];      // the CTA's
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int rps = p.tps * p.R, nrb = (rps + 15) / 16;
    const int unit = (int)blockIdx.x / nsplit, rank = (int)blockIdx.x - unit * nsplit;
    const int rb = unit % nrb, kvh = (unit / nrb) % p.c.n_kv, seq = unit / (nrb * p.c.n_kv);
    const int row0 = rb * 16, nrows = min(16, rps - row0);
    pdl_launch_dependents();
    pdl_wait();
    const int slot = ao_slot(p, seq);
    int lim[2];
    const __half* qrow[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = min(g + 8 * h, nrows - 1) + row0, tok = r / p.R;
        lim[h] = g + 8 * h < nrows ? ao_limit(p, __ldg(p.positions + (size_t)seq * p.tps + tok)) : 0;
        qrow[h] = p.q + ((size_t)seq * p.tps + tok) * p.q_pitch + ((size_t)kvh * p.R + (r - tok * p.R)) * AO_D;
    }
    const int most = __reduce_max_sync(0xffffffffu, max(lim[0], lim[1]));
    const int least = __reduce_min_sync(0xffffffffu, min(g < nrows ? lim[0] : INT_MAX, g + 8 < nrows ? lim[1] : INT_MAX));
    uint32_t q[8][4];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        q[k][0] = *reinterpret_cast<const uint32_t*>(qrow[0] + k * 16 + 2 * t4), q[k][1] = *reinterpret_cast<const uint32_t*>(qrow[1] + k * 16 + 2 * t4);
        q[k][2] = *reinterpret_cast<const uint32_t*>(qrow[0] + k * 16 + 8 + 2 * t4), q[k][3] = *reinterpret_cast<const uint32_t*>(qrow[1] + k * 16 + 8 + 2 * t4);
    }
    const int step = nsplit * AO_WARPS, chunks = (most + AO_KEYS - 1) / AO_KEYS;
    const uint32_t ring = smem_u32(ao_smem) + warp * (AO_STAGES * 2 * AO_HALF_STAGE);
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
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(p.k + at + (size_t)row * AO_D), "r"(n) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + AO_HALF_STAGE), "l"(p.v + at + (size_t)row * AO_D), "r"(n) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[16][4];
#pragma unroll
    for (int n = 0; n < 16; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    int ch = rank * AO_WARPS + warp, stage = 0;
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
            float x[4] = {s[0][2 * h] * p.sl2, s[0][2 * h + 1] * p.sl2, s[1][2 * h] * p.sl2, s[1][2 * h + 1] * p.sl2};
            if (key0 + AO_KEYS > least) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key0 + 2 * t4 + (e & 1) + 8 * (e >> 1) >= lim[h]) x[e] = -INFINITY;
            }
            float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            top = fmaxf(top, m[h]);
            const float base = (top == -INFINITY ? 0.0f : top) - AO_LIFT;
            corr[h] = m[h] == -INFINITY ? 0.0f : ao_exp2(m[h] - top);
            m[h] = top;
            l[h] *= corr[h];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[h][e] = ao_exp2(x[e] - base), l[h] += f[h][e];
            const __half2 a = __floats2half2_rn(f[h][0], f[h][1]), b = __floats2half2_rn(f[h][2], f[h][3]);
            w[h] = *reinterpret_cast<const uint32_t*>(&a), w[2 + h] = *reinterpret_cast<const uint32_t*>(&b);
        }
#pragma unroll
        for (int n = 0; n < 16; ++n) o[n][0] *= corr[0], o[n][1] *= corr[0], o[n][2] *= corr[1], o[n][3] *= corr[1];
        bool plain = true;
        if (key0 + AO_KEYS > least && least < most) {              // a weight of zero hides finite values only
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
    float* o_s = reinterpret_cast<float*>(ao_smem);                // [warp][16][128]
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (t4 == 0) ml_s[warp][g + 8 * h] = make_float2(m[h] == -INFINITY ? m[h] : m[h] - AO_LIFT, l[h]);
        if (g + 8 * h < nrows) {
#pragma unroll
            for (int n = 0; n < 16; ++n)
                *reinterpret_cast<float2*>(o_s + ((warp * 16 + g + 8 * h) * AO_D + n * 8 + 2 * t4)) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        }
    }
    __syncthreads();
    auto put = [&](int r, int d, const float4& v, float sum) {
        const int row = row0 + r, tok = row / p.R;
        const float inv = 1.0f / sum;
        const bool on = sum > 0.0f || sum != sum;  // (a row without keys: zeros)
        const __half2 a = __floats2half2_rn(on ? v.x * inv : 0.0f, on ? v.y * inv : 0.0f), b = __floats2half2_rn(on ? v.z * inv : 0.0f, on ? v.w * inv : 0.0f);
        *reinterpret_cast<uint2*>(p.out + (((size_t)seq * p.tps + tok) * p.n_heads + (size_t)kvh * p.R + (row - tok * p.R)) * AO_D + d) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    };
    for (int it = tid; it < nrows * 32; it += AO_WARPS * 32) {     // four dims of a row
        const int r = it >> 5, d = (it & 31) * 4;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < AO_WARPS; ++w) top = fmaxf(top, ml_s[w][r].x);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (top != -INFINITY) {
#pragma unroll
            for (int w = 0; w < AO_WARPS; ++w) {
                const float2 ml = ml_s[w][r];
                const float f = ml.x == -INFINITY ? 0.0f : ao_exp2(ml.x - top);
                if (f == 0.0f) continue;
                const float4 v = *reinterpret_cast<const float4*>(o_s + (w * 16 + r) * AO_D + d);
                acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
                sum += f * ml.y;
            }
        } else {
#pragma unroll
            for (int w = 0; w < AO_WARPS; ++w) sum += ml_s[w][r].y;                // (zero, or NaN where all scores are)
            if (sum != sum) acc = make_float4(sum, sum, sum, sum);
        }
        if (nsplit == 1) {
            put(r, d, acc, sum);
        } else {
            *reinterpret_cast<float4*>(o_s + r * AO_D + d) = acc;  // (warp 0's place, read by this thread)
            if (d == 0) ml_c[r] = make_float2(top, sum);
        }
    }
    if (nsplit == 1) return;
    ao_cluster_sync();
    const uint32_t ob = smem_u32(o_s), mb = smem_u32(ml_c);
    for (int it = rank * AO_WARPS * 32 + tid; it < nrows * 32; it += nsplit * AO_WARPS * 32) {
        const int r = it >> 5, d = (it & 31) * 4;
        float top = -INFINITY, sum = 0.0f;
        for (int w = 0; w < nsplit; ++w) top = fmaxf(top, ao_ld_cluster2(ao_map_rank(mb + r * 8, w)).x);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < nsplit; ++w) {
            const float2 ml = ao_ld_cluster2(ao_map_rank(mb + r * 8, w));
            const float f = ml.x == -INFINITY ? (ml.y != ml.y ? 1.0f : 0.0f) : ao_exp2(ml.x - top);
            if (f == 0.0f) continue;
            const float4 v = ao_ld_cluster4(ao_map_rank(ob + (r * AO_D + d) * 4, w));
            acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
            sum += f * ml.y;
        }
        put(r, d, acc, sum);
    }
    ao_cluster_sync();                             // nobody leaves while its sums are read
}

}  // namespace sbvr

using namespace sbvr;

// CTAs that share the keys of a (sequence, KV head, 16 rows): as many as make about two per SM, at most 8
static int own_split(int units, int sm_count) {
    int n = 1;
    while (n < 8 && units * n * 2 <= 2 * sm_count) n *= 2;
    return n;
}

extern "C" {

int sbvr_pages_attention_scratch_bytes(const sbvr_pages_t* cache, int seqs, int tokens_per_seq, int n_heads, int groups, size_t* bytes) {
    PgCache c;
    const int rc = pg_cache(cache, &c);
    if (rc) return rc;
    if (!bytes || seqs < 1 || tokens_per_seq < 1 || n_heads < 1 || groups < 0 || n_heads % c.n_kv) return SBVR_ERR_BAD_ARG;
    *bytes = 0;
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
    if ((long long)seqs * tokens_per_seq * n_heads > INT_MAX / 4) return SBVR_ERR_UNSUPPORTED;
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) || q_pitch % 8) return SBVR_ERR_ALIGN;
    DeviceInfo di;
    int dev = 0;
    SBVR_CUDA_TRY(cudaGetDevice(&dev));
    rc = device_info(dev, &di);
    if (rc) return rc;
    p.k = c.pool + (size_t)layer * 2 * pg_plane(c), p.v = p.k + pg_plane(c);
    p.q = static_cast<const __half*>(q), p.slots = slots, p.positions = positions, p.starts = groups ? group_starts : nullptr, p.shared = shared;
    p.out = static_cast<__half*>(out), p.part = static_cast<float*>(scratch), p.q_pitch = q_pitch;
    p.seqs = seqs, p.tps = tokens_per_seq, p.n_heads = n_heads, p.R = n_heads / c.n_kv, p.groups = groups;
    p.sl2 = scale * 1.4426950408889634f;
    (void)scratch_bytes;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    static SmemOnce once, once_cluster;
    rc = set_max_smem_once(once, attention_own_kernel, AO_SMEM);
    if (!rc) rc = set_attribute_once(once_cluster, attention_own_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (rc) return rc;
    const int units = seqs * c.n_kv * ((p.tps * p.R + 15) / 16), nsplit = own_split(units, di.sm_count);
    SBVR_CUDA_TRY(launch_pdl_cluster(attention_own_kernel, dim3((unsigned)(units * nsplit)), dim3(AO_WARPS * 32), nsplit, (size_t)AO_SMEM, st, p, nsplit));
    return SBVR_OK;
}

}  // extern "C"
