// A KV cache in pages (sbvr_pages_t): who holds which page (reserve, free, fork, compact), the copies that follow from it, and the rotary
// embedding that appends a layer's new tokens to their pages.
//
// Bookkeeping.  table[slot][k] is the page of a slot's tokens k * page ..; refs[p] counts the slots that hold page p.  Pages are handed out
// lowest index first, slots in the order they are named: prefix sums over the slots' needs and over the free pages give every page its place, so
// results do not depend on the order in which threads run.  A call that cannot be carried out (too few pages, a slot named twice) changes
// nothing and leaves a bit in the status word.  These kernels are chains of latencies: their data (refs, a few rows of the table) is a few
// hundred KB at most.
#include <algorithm>
#include <climits>

#include "common.cuh"
#include "pages.cuh"

namespace sbvr {

constexpr int PG_THREADS = 1024;
constexpr int PG_PER = 16;                         // pages a thread looks at in one step of a search

struct PgScan {                                    // exclusive prefix sums over the block's threads
    int warp[PG_THREADS / 32];
};
__device__ __forceinline__ int pg_scan(PgScan& s, int v, int* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                               // (s may still be read from the scan before)
    if (lane == 31) s.warp[w] = x;
    __syncthreads();
    if (w == 0) {
        int y = s.warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        s.warp[lane] = y;
    }
    __syncthreads();
    *total = s.warp[PG_THREADS / 32 - 1];
    return x - v + (w ? s.warp[w - 1] : 0);
}

struct PgMove {                                    // `rows` token rows of page src to page dst
    int src, dst, rows;
};

__device__ __forceinline__ int pg_slot(const int* slots, int i) { return slots ? __ldg(slots + i) : i; }
__device__ __forceinline__ int pg_pages_of(const PgCache& c, int tokens) { return min((max(tokens, 0) + c.page - 1) >> c.page_shift, c.max_pages); }

// Whether every slot is one of the cache's and none is named twice.  `seen`: a bit per slot in shared memory.
__device__ bool pg_slots_ok(const PgCache& c, const int* slots, int n, uint32_t* seen) {
    for (int i = threadIdx.x; i < (c.max_seqs + 31) / 32; i += blockDim.x) seen[i] = 0u;
    __syncthreads();
    bool ok = true;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int s = pg_slot(slots, i);
        if (s < 0 || s >= c.max_seqs) {
            ok = false;
        } else {
            const uint32_t bit = 1u << (s & 31);
            if (atomicOr(seen + (s >> 5), bit) & bit) ok = false;
        }
    }
    return __syncthreads_and(ok);
}

// The first `want` pages that nobody holds, ascending, into list; how many there were (at most `want`).
__device__ int pg_find_free(const PgCache& c, int want, int* list, PgScan& sc) {
    int found = 0;
    for (int base = 0; base < c.pages && found < want; base += PG_THREADS * PG_PER) {
        const int p0 = base + threadIdx.x * PG_PER;
        uint32_t free_bits = 0;
#pragma unroll
        for (int q = 0; q < PG_PER / 4; ++q) {     // (refs has room up to a multiple of four)
            if (p0 + 4 * q >= c.pages) break;
            const int4 v = __ldcg(reinterpret_cast<const int4*>(c.refs + p0 + 4 * q));
            const int r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (p0 + 4 * q + e < c.pages && r[e] == 0) free_bits |= 1u << (4 * q + e);
        }
        int total;
        int at = found + pg_scan(sc, __popc(free_bits), &total);
        while (free_bits && at < want) {
            list[at++] = p0 + __ffs(free_bits) - 1;
            free_bits &= free_bits - 1;
        }
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

// ---------------------------------------------------------------------------------------------
// free: a block per slot
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(128) pages_free_kernel(const PgCache c, const int* slots, int n) {
    extern __shared__ uint32_t seen[];
    pdl_launch_dependents();
    pdl_wait();
    if (!pg_slots_ok(c, slots, n, seen)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(c.status, SBVR_PAGES_BAD_SLOT);
        return;
    }
    const int slot = pg_slot(slots, blockIdx.x), have = pg_pages_of(c, c.lengths[slot]);
    int* row = c.table + (size_t)slot * c.max_pages;
    for (int k = threadIdx.x; k < have; k += blockDim.x) {
        const int p = row[k];
        if (p >= 0 && p < c.pages) atomicSub(c.refs + p, 1);
        row[k] = -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) c.lengths[slot] = 0;
}

// ---------------------------------------------------------------------------------------------
// reserve: one block.  scratch: [4: verdict][two words per slot][free pages].  More than PG_POSITIONS positions are written by a launch of their own behind
// it (64 slots x 4000 by the one block: 60 us).
// ---------------------------------------------------------------------------------------------
constexpr int PG_POSITIONS = 8192, PG_SHARED = 2048;

__global__ void __launch_bounds__(256) pages_positions_kernel(const PgCache c, const int* slots, const int* tokens, int each, int* positions, int tps) {
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.x, t = tokens ? tokens[s] : each;
    const bool done = c.scratch[0] == 0;
    const int first = done ? c.lengths[pg_slot(slots, s)] - t : 0, end = done ? t : 0;
    for (int j = blockIdx.y * 256 + threadIdx.x; j < tps; j += gridDim.y * 256) positions[(size_t)s * tps + j] = j < end ? first + j : -1;
}

__global__ void __launch_bounds__(PG_THREADS) pages_reserve_kernel(const PgCache c, const int* slots, const int* tokens, int each, int n,
                                                                   int* positions, int tps) {
    extern __shared__ uint32_t seen[];
    __shared__ PgScan sc;
    pdl_launch_dependents();
    pdl_wait();
    int fault = pg_slots_ok(c, slots, n, seen) ? 0 : SBVR_PAGES_BAD_SLOT;
    // what every slot needs, summed up [n + 1], and the table's entry of its first new page [n]: in shared memory for up to PG_SHARED slots
    int* first = n <= PG_SHARED ? reinterpret_cast<int*>(seen + (c.max_seqs + 31) / 32) : c.scratch + 4;
    int* entry = n <= PG_SHARED ? first + n + 1 : c.scratch + 4 + c.max_seqs + 4;
    int* list = c.scratch + 4 + 2 * (c.max_seqs + 4);
    int sum = 0;
    for (int base = 0; base < n; base += PG_THREADS) {
        const int i = base + threadIdx.x;
        int need = 0, bad = 0;
        if (i < n && !fault) {
            const int slot = pg_slot(slots, i), len = c.lengths[slot], t = tokens ? tokens[i] : each;
            if (t < 0) bad = SBVR_PAGES_BAD_SLOT;
            else if (len > c.max_pages * c.page - t) bad = SBVR_PAGES_TOO_LONG;
            else need = pg_pages_of(c, len + t) - pg_pages_of(c, len);
        }
        int total;
        const int at = sum + pg_scan(sc, need, &total);
        if (i < n) {
            first[i] = at;
            if (!fault) entry[i] = pg_slot(slots, i) * c.max_pages + pg_pages_of(c, c.lengths[pg_slot(slots, i)]);
        }
        // (needs are bounded by n * max_pages, which the host keeps below 2^31)
        sum += total;
        fault |= __syncthreads_or(bad & SBVR_PAGES_BAD_SLOT) ? SBVR_PAGES_BAD_SLOT : 0;
        fault |= __syncthreads_or(bad & SBVR_PAGES_TOO_LONG) ? SBVR_PAGES_TOO_LONG : 0;
    }
    if (threadIdx.x == 0) first[n] = sum;
    if (!fault && sum > c.pages) fault = SBVR_PAGES_NO_PAGE;
    if (!fault && pg_find_free(c, sum, list, sc) < sum) fault = SBVR_PAGES_NO_PAGE;
    __syncthreads();
    if (threadIdx.x == 0) c.scratch[0] = fault;
    if (fault) {
        if (threadIdx.x == 0) atomicOr(c.status, fault);
        if (positions)
            for (int i = threadIdx.x; i < n * tps; i += PG_THREADS) positions[i] = -1;
        return;
    }
    for (int j = threadIdx.x; j < sum; j += PG_THREADS) {
        int lo = 0, hi = n;                        // the last i with first[i] <= j: the slot that page j of the list goes to
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= j) lo = mid;
            else hi = mid;
        }
        const int p = list[j];
        c.table[entry[lo] + (j - first[lo])] = p;
        c.refs[p] = 1;
    }
    if (positions) {
        for (int i = threadIdx.x; i < n * tps; i += PG_THREADS) {
            const int s = i / tps, j = i - s * tps;
            positions[i] = j < (tokens ? tokens[s] : each) ? c.lengths[pg_slot(slots, s)] + j : -1;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PG_THREADS) c.lengths[pg_slot(slots, i)] += tokens ? tokens[i] : each;
}

// ---------------------------------------------------------------------------------------------
// fork / copy: one block, then the copies.  scratch: [4: number of copies][free pages][copies: src, dst, rows]
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(PG_THREADS) pages_fork_kernel(const PgCache c, const int* src, const int* dst, int n, int share) {
    extern __shared__ uint32_t seen[];
    __shared__ PgScan sc;
    pdl_launch_dependents();
    pdl_wait();
    // pairs in shared memory: slots, the parent's and the child's tokens, first page of the child's own
    int* src_s = reinterpret_cast<int*>(seen + (c.max_seqs + 31) / 32);
    int *dst_s = src_s + n, *slen = dst_s + n, *dlen = slen + n, *first = dlen + n;
    int* list = c.scratch + 4;
    PgMove* moves = reinterpret_cast<PgMove*>(list + ((c.pages + 3) & ~3));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, me = threadIdx.x;
    bool ok = pg_slots_ok(c, dst, n, seen);
    int need = 0;
    if (me < n) {                                  // (n <= 1024)
        const int s = src[me], d = dst[me];
        src_s[me] = s, dst_s[me] = d;
        if (s < 0 || s >= c.max_seqs) {
            ok = false;
        } else if (ok) {
            const int len = max(c.lengths[s], 0);
            slen[me] = len, dlen[me] = c.lengths[d];
            if (s != d) need = pg_pages_of(c, len) - (share ? min(len >> c.page_shift, c.max_pages) : 0);
        }
    }
    int fault = __syncthreads_and(ok) ? 0 : SBVR_PAGES_BAD_SLOT, sum;
    {
        const int at = pg_scan(sc, fault ? 0 : need, &sum);
        if (me < n) first[me] = at;
        if (me == 0) first[n] = sum;
    }
    if (!fault && sum > c.pages) fault = SBVR_PAGES_NO_PAGE;
    __syncthreads();
    auto counts = [&](int sign) {                  // what the children give up and what they take part in; pages that are read are held
        for (int i = warp; i < n; i += PG_THREADS / 32) {
            if (src_s[i] == dst_s[i]) continue;
            const int* rs = c.table + (size_t)src_s[i] * c.max_pages;
            const int* rd = c.table + (size_t)dst_s[i] * c.max_pages;
            const int have = pg_pages_of(c, dlen[i]), need = pg_pages_of(c, slen[i]);
            for (int k = lane; k < max(have, need); k += 32) {
                const int o = k < have ? rd[k] : -1, s = k < need ? rs[k] : -1;
                if (o == s) continue;
                if (o >= 0 && o < c.pages) atomicSub(c.refs + o, sign);
                if (s >= 0 && s < c.pages) atomicAdd(c.refs + s, sign);
            }
        }
        __threadfence();
        __syncthreads();
    };
    if (!fault) {
        counts(1);
        if (pg_find_free(c, sum, list, sc) < sum) {
            counts(-1);
            fault = SBVR_PAGES_NO_PAGE;
        }
    }
    if (threadIdx.x == 0) c.scratch[0] = fault ? 0 : sum;
    if (fault) {
        if (threadIdx.x == 0) atomicOr(c.status, fault);
        return;
    }
    for (int i = warp; i < n; i += PG_THREADS / 32) {          // pages of their own
        if (src_s[i] == dst_s[i]) continue;
        const int need = pg_pages_of(c, slen[i]), own = first[i + 1] - first[i], full = need - own;
        for (int j = lane; j < own; j += 32) {
            const int s = c.table[(size_t)src_s[i] * c.max_pages + full + j], p = list[first[i] + j];
            const bool on = s >= 0 && s < c.pages;
            c.refs[p] = 1;
            if (on) atomicSub(c.refs + s, 1);      // (no longer held)
            moves[first[i] + j] = PgMove{on ? s : p, p, on ? min(c.page, slen[i] - ((full + j) << c.page_shift)) : 0};
        }
    }
    __syncthreads();
    // Rows of the table, some columns of all children at a time: what is a child in one pair may be the parent in another.
    constexpr int PER = 8;
    const int cols = PG_THREADS * PER / n;         // (n <= 1024)
    int most = 0;
    for (int i = threadIdx.x; i < n; i += PG_THREADS)
        if (src_s[i] != dst_s[i]) most = max(most, max(pg_pages_of(c, slen[i]), pg_pages_of(c, dlen[i])));
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) sc.warp[warp] = most;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, sc.warp[lane]);
    for (int k0 = 0; k0 < most; k0 += cols) {
        int v[PER];
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int e = q * PG_THREADS + threadIdx.x, i = e / cols, k = k0 + e % cols;
            v[q] = -2;
            if (i >= n || k >= c.max_pages || src_s[i] == dst_s[i]) continue;
            const int need = pg_pages_of(c, slen[i]), full = need - (first[i + 1] - first[i]);
            if (k < full) v[q] = c.table[(size_t)src_s[i] * c.max_pages + k];
            else if (k < need) v[q] = list[first[i] + k - full];
            else if (k < pg_pages_of(c, dlen[i])) v[q] = -1;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int e = q * PG_THREADS + threadIdx.x;
            if (v[q] != -2) c.table[(size_t)dst_s[e / cols] * c.max_pages + k0 + e % cols] = v[q];
        }
        __syncthreads();
    }
    if (me < n) c.lengths[dst_s[me]] = slen[me];
}

// ---------------------------------------------------------------------------------------------
// compact: one block pairs the pages in use at or behind U, their number, with the free ones in front of it, both ascending.
// scratch: [4: number of copies, U][free pages][new place of a page][copies]
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(PG_THREADS) pages_compact_kernel(const PgCache c) {
    __shared__ PgScan sc;
    pdl_launch_dependents();
    pdl_wait();
    int* head = c.scratch;
    int* holes = c.scratch + 4;
    const int pages4 = (c.pages + 3) & ~3;
    int* place = holes + pages4;
    PgMove* moves = reinterpret_cast<PgMove*>(place + pages4);
    auto used_bits = [&](int p0) {
        uint32_t bits = 0;
#pragma unroll
        for (int q = 0; q < PG_PER / 4; ++q) {
            if (p0 + 4 * q >= c.pages) break;
            const int4 v = *reinterpret_cast<const int4*>(c.refs + p0 + 4 * q);
            const int r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (p0 + 4 * q + e < c.pages && r[e] > 0) bits |= 1u << (4 * q + e);
        }
        return bits;
    };
    int mine = 0, used;
    for (int base = 0; base < c.pages; base += PG_THREADS * PG_PER) mine += __popc(used_bits(base + threadIdx.x * PG_PER));
    pg_scan(sc, mine, &used);
    int nh = 0, nm = 0;
    for (int base = 0; base < c.pages; base += PG_THREADS * PG_PER) {
        const int p0 = base + threadIdx.x * PG_PER;
        const uint32_t bits = used_bits(p0);
        const int in_front = max(0, min(PG_PER, used - p0)), here = max(0, min(PG_PER, c.pages - p0));      // pages before U, pages there are
        const uint32_t lo = in_front >= 32 ? ~0u : (1u << in_front) - 1u;
        uint32_t hole = ~bits & lo & ((1u << here) - 1u), move = bits & ~lo;
        int total;
        int at = nh + pg_scan(sc, __popc(hole), &total);
        nh += total;
        for (; hole; hole &= hole - 1) holes[at++] = p0 + __ffs(hole) - 1;
        at = nm + pg_scan(sc, __popc(move), &total);
        nm += total;
        for (; move; move &= move - 1) moves[at++].src = p0 + __ffs(move) - 1;
    }
    __syncthreads();
    // (as many holes as pages to move: U pages are in use, those in front of U and nm behind)
    for (int i = threadIdx.x; i < nm; i += PG_THREADS) {
        const int s = moves[i].src, d = holes[i];
        moves[i].dst = d, moves[i].rows = c.page;
        place[s] = d;
        c.refs[d] = c.refs[s];
        c.refs[s] = 0;
    }
    if (threadIdx.x == 0) head[0] = nm, head[1] = used;
}

// ---------------------------------------------------------------------------------------------
// The copies of a fork (rows of a page, all layers and heads) or of a compaction (then also the table's entries).
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) pages_move_kernel(const PgCache c, int list_at, int place_at) {
    pdl_launch_dependents();
    pdl_wait();
    const int count = c.scratch[0];
    const PgMove* moves = reinterpret_cast<const PgMove*>(c.scratch + list_at);
    if (place_at) {
        const int used = c.scratch[1];
        const int* place = c.scratch + place_at;
        for (int s = blockIdx.x; s < c.max_seqs; s += gridDim.x) {
            const int have = pg_pages_of(c, c.lengths[s]);
            for (int k = threadIdx.x; k < have; k += blockDim.x) {
                int* e = c.table + (size_t)s * c.max_pages + k;
                if (*e >= used && *e < c.pages) *e = place[*e];
            }
        }
    }
    const int planes = 2 * c.layers;
    // A unit: one head of one plane of one page, or all heads, where planes make half the grid.  A fork's us by heads / by all, 8 heads: 64 planes of 250
    // tokens 15.6 / 23.6, 256 of 120 21.7 / 25.0, 400 of 60 28.3 / 30.0; 448 of 15 19.5 / 12.7, 448 of 40 19.9 / 17.5, 960 of 40 30.8 / 23.9, 4032 of
    // 40 96 / 74.  On the wrong side of the line: 512 of 120 36.0 / 39.8.
    const int parts = (long long)count * planes * 2 >= (int)gridDim.x ? 1 : c.n_kv;
    const int heads = c.n_kv / parts;
    const long long units = (long long)count * planes * parts;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int part = (int)(u % parts);
        const long long r = u / parts;
        const int plane = (int)(r % planes);
        const PgMove m = moves[r / planes];
        const size_t base = (size_t)plane * pg_plane(c) + (size_t)part * heads * c.page * PG_D;
        const uint4* from = reinterpret_cast<const uint4*>(c.pool + base + (size_t)m.src * c.n_kv * c.page * PG_D);
        uint4* to = reinterpret_cast<uint4*>(c.pool + base + (size_t)m.dst * c.n_kv * c.page * PG_D);
        const int per = m.rows * (PG_D / 8), pitch = c.page * (PG_D / 8);      // 16-byte pieces of a head: to be copied, there are
        int h = 0, v = threadIdx.x;
        while (v >= per && h < heads) v -= per, ++h;
        while (h < heads) {
            uint4 x[8];
            int at[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                at[q] = h < heads ? h * pitch + v : -1;
                if (at[q] >= 0) x[q] = from[at[q]];
                v += 256;
                while (v >= per && h < heads) v -= per, ++h;
            }
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (at[q] >= 0) to[at[q]] = x[q];
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Tokens that all sequences of a group hold in the same pages: whole pages in front.  A block per group.
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) pages_common_kernel(const PgCache c, const int* slots, const int* starts, int n, int* out) {
    __shared__ int same;
    pdl_launch_dependents();
    pdl_wait();
    const int s0 = max(0, min(starts[blockIdx.x], n)), s1 = max(s0, min(starts[blockIdx.x + 1], n));
    if (threadIdx.x == 0) same = s1 - s0 < 2 ? 0 : c.max_pages;
    __syncthreads();
    const int lead = s0 < n ? pg_slot(slots, s0) : -1;
    for (int s = s0; s < s1; ++s) {
        const int slot = pg_slot(slots, s);
        if (slot < 0 || slot >= c.max_seqs || lead < 0 || lead >= c.max_seqs) {
            if (threadIdx.x == 0) atomicOr(c.status, SBVR_PAGES_BAD_SLOT), atomicMin(&same, 0);
            continue;
        }
        const int whole = min(max(c.lengths[slot], 0) >> c.page_shift, c.max_pages);
        if (threadIdx.x == 0) atomicMin(&same, whole);
        for (int k = threadIdx.x; k < whole; k += blockDim.x)
            if (c.table[(size_t)slot * c.max_pages + k] != c.table[(size_t)lead * c.max_pages + k]) {
                atomicMin(&same, k);
                break;
            }
    }
    __syncthreads();
    if (threadIdx.x == 0) out[blockIdx.x] = same << c.page_shift;
}

// ---------------------------------------------------------------------------------------------
// rotary embedding of q and k; q to its own rows, k and v to the tokens' pages.  A block per token.
// The angle pos * inv_freq is formed and reduced to half a turn in 64 bits: in 32 it is off by 2^-24 of itself, 4e-3 radians at position 65536.
// The rotation is computed in 32 bits and rounded once.
// ---------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) pages_rope_append_kernel(const PgCache c, int layer, const __half* __restrict__ qkv, const int* __restrict__ positions,
                                                                const float* __restrict__ inv_freq, float attn_scaling, const int* __restrict__ slots,
                                                                int tps, int n_heads, __half* __restrict__ q_out) {
    __shared__ __align__(16) float cs_s[2][PG_D / 2];
    __shared__ long long row_s;                    // element of the page's first head where this token's rows go, -1: nowhere
    pdl_launch_dependents();
    pdl_wait();
    constexpr int CH = PG_D / 16;                  // pieces of 8 elements in half a head
    const int t = blockIdx.x, rot = (n_heads + c.n_kv) * CH, all = rot + c.n_kv * CH;
    const __half* row = qkv + (size_t)t * (n_heads + 2 * c.n_kv) * PG_D;
    auto load = [&](int it, uint4 (&x)[2]) {
        if (it >= all) return;
        const __half* p = row + (size_t)(it / CH) * PG_D + (it % CH) * 8;
        x[0] = *reinterpret_cast<const uint4*>(p), x[1] = *reinterpret_cast<const uint4*>(p + PG_D / 2);
    };
    uint4 x[2][2];
    int pos = -1;
    if (tps > 1) {                                 // places without a token read nothing (half of a batch of uneven prompts)
        pos = positions[t];
        if (pos < 0) {
            for (int it = threadIdx.x; it < n_heads * (PG_D / 8); it += 256)
                *reinterpret_cast<uint4*>(q_out + (size_t)t * n_heads * PG_D + it * 8) = make_uint4(0u, 0u, 0u, 0u);
            return;
        }
    }
    load(threadIdx.x, x[0]);
    load(threadIdx.x + 256, x[1]);
    if (tps == 1) pos = positions[t];
    if (threadIdx.x < PG_D / 2) {
        const double turn = (double)pos * (double)inv_freq[threadIdx.x];
        const float a = (float)fma(-rint(turn * 0.15915494309189535), 6.283185307179586, turn);
        float s, co;
        sincosf(a, &s, &co);
        cs_s[0][threadIdx.x] = co * attn_scaling, cs_s[1][threadIdx.x] = s * attn_scaling;
    }
    if (threadIdx.x == 64) {
        const int slot = pg_slot(slots, t / tps), k = pos >> c.page_shift;
        long long at = -1;
        if (pos >= 0) {
            const int p = slot >= 0 && slot < c.max_seqs && k < c.max_pages ? c.table[(size_t)slot * c.max_pages + k] : -1;
            if (p >= 0 && p < c.pages) at = ((long long)p * c.n_kv * c.page + (pos & (c.page - 1))) * PG_D;
            else atomicOr(c.status, SBVR_PAGES_NO_ENTRY);
        }
        row_s = at;
    }
    __syncthreads();
    const long long at = row_s;
    __half* kp = c.pool + (size_t)layer * 2 * pg_plane(c);
    auto finish = [&](int it, uint4 (&v)[2]) {
        if (it >= all) return;
        const int head = it / CH, i = (it % CH) * 8;
        if (it < rot) {
            __half2 *a = reinterpret_cast<__half2*>(&v[0]), *b = reinterpret_cast<__half2*>(&v[1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = __half22float2(a[e]), g = __half22float2(b[e]);
                const float2 cc = *reinterpret_cast<const float2*>(&cs_s[0][i + 2 * e]), ss = *reinterpret_cast<const float2*>(&cs_s[1][i + 2 * e]);
                a[e] = __floats2half2_rn(f.x * cc.x - g.x * ss.x, f.y * cc.y - g.y * ss.y);
                b[e] = __floats2half2_rn(g.x * cc.x + f.x * ss.x, g.y * cc.y + f.y * ss.y);
            }
        }
        __half* p;
        if (head < n_heads) {
            p = q_out + ((size_t)t * n_heads + head) * PG_D + i;
            if (pos < 0) v[0] = v[1] = make_uint4(0u, 0u, 0u, 0u);
        } else {
            if (at < 0) return;
            const int kv = it < rot ? head - n_heads : head - n_heads - c.n_kv;
            p = kp + (it < rot ? 0 : pg_plane(c)) + at + (size_t)kv * c.page * PG_D + i;
        }
        *reinterpret_cast<uint4*>(p) = v[0], *reinterpret_cast<uint4*>(p + PG_D / 2) = v[1];
    };
    finish(threadIdx.x, x[0]);
    finish(threadIdx.x + 256, x[1]);
    for (int it = threadIdx.x + 512; it < all; it += 256) {
        load(it, x[0]);
        finish(it, x[0]);
    }
}

int pg_cache(const sbvr_pages_t* c, PgCache* o) {
    if (!c || !c->pool || !c->table || !c->lengths || !c->refs || !c->status || !c->scratch) return SBVR_ERR_BAD_ARG;
    if (c->layers < 1 || c->pages < 1 || c->n_kv < 1 || c->max_seqs < 1 || c->max_pages < 1) return SBVR_ERR_BAD_ARG;
    if (c->head_dim != PG_D || c->page < 16 || c->page > 256 || (c->page & (c->page - 1)) || c->max_seqs > 65536) return SBVR_ERR_UNSUPPORTED;
    // rows of a plane, tokens of a slot and entries of the table are counted in 32 bits
    if ((long long)c->pages * c->n_kv * c->page > INT_MAX / 2 || (long long)c->max_pages * c->page > INT_MAX / 2 ||
        (long long)c->max_pages * c->max_seqs > INT_MAX / 2)
        return SBVR_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(c->pool) | reinterpret_cast<uintptr_t>(c->refs) | reinterpret_cast<uintptr_t>(c->scratch)) & 15) return SBVR_ERR_ALIGN;
    if ((reinterpret_cast<uintptr_t>(c->table) | reinterpret_cast<uintptr_t>(c->lengths) | reinterpret_cast<uintptr_t>(c->status)) & 3) return SBVR_ERR_ALIGN;
    *o = PgCache{static_cast<__half*>(c->pool), c->table, c->lengths, c->refs, c->status, c->scratch, c->layers, c->pages, c->page, 0, c->n_kv,
                 c->max_seqs, c->max_pages};
    while ((1 << o->page_shift) < c->page) ++o->page_shift;
    return SBVR_OK;
}

}  // namespace sbvr

using namespace sbvr;

static size_t seen_bytes(const PgCache& c) { return (size_t)(c.max_seqs + 31) / 32 * 4; }
// where the copies stand in the scratch of a fork, and of a compaction
static int fork_moves_at(const PgCache& c) { return 4 + ((c.pages + 3) & ~3); }
static int compact_moves_at(const PgCache& c) { return 4 + 2 * ((c.pages + 3) & ~3); }

static int launch_moves(const PgCache& c, int list_at, int place_at, cudaStream_t st) {
    DeviceInfo di;
    int dev = 0;
    SBVR_CUDA_TRY(cudaGetDevice(&dev));
    const int rc = device_info(dev, &di);
    if (rc) return rc;
    // (six CTAs per SM: 63 children of a 32-layer page 81 us, 346 pages of 2 MB 125; four 87 and 129, eight 91 and 123)
    SBVR_CUDA_TRY(launch_pdl(pages_move_kernel, dim3((unsigned)(6 * di.sm_count)), dim3(256), 0, st, c, list_at, place_at));
    return SBVR_OK;
}

extern "C" {

int sbvr_pages_scratch_bytes(const sbvr_pages_t* cache, size_t* bytes) {
    if (!cache || !bytes || cache->pages < 1 || cache->max_seqs < 1) return SBVR_ERR_BAD_ARG;
    const size_t pages4 = ((size_t)cache->pages + 3) & ~(size_t)3;
    *bytes = 4 * (16 + 2 * ((size_t)cache->max_seqs + 4) + 2 * pages4 + 3 * (size_t)cache->pages);
    return SBVR_OK;
}

int sbvr_pages_free(const sbvr_pages_t* cache, const int* slots, int n, sbvr_stream_t stream) {
    PgCache c;
    const int rc = pg_cache(cache, &c);
    if (rc) return rc;
    if (n < 1 || n > c.max_seqs) return SBVR_ERR_BAD_ARG;
    SBVR_CUDA_TRY(launch_pdl(pages_free_kernel, dim3((unsigned)n), dim3(128), seen_bytes(c), reinterpret_cast<cudaStream_t>(stream), c, slots, n));
    return SBVR_OK;
}

int sbvr_pages_reserve(const sbvr_pages_t* cache, const int* slots, const int* tokens, int tokens_each, int n, int* positions, int tokens_per_seq,
                       sbvr_stream_t stream) {
    PgCache c;
    const int rc = pg_cache(cache, &c);
    if (rc) return rc;
    if (n < 1 || n > c.max_seqs || (!tokens && tokens_each < 0) || (positions && tokens_per_seq < 1)) return SBVR_ERR_BAD_ARG;
    if (positions && (long long)n * tokens_per_seq > INT_MAX / 2) return SBVR_ERR_UNSUPPORTED;
    const bool many = positions && (long long)n * tokens_per_seq > PG_POSITIONS;
    SBVR_CUDA_TRY(launch_pdl(pages_reserve_kernel, dim3(1), dim3(PG_THREADS), seen_bytes(c) + (n <= PG_SHARED ? (2 * (size_t)n + 1) * 4 : 0), reinterpret_cast<cudaStream_t>(stream), c, slots, tokens,
                             tokens_each, n, many ? nullptr : positions, tokens_per_seq));
    if (many)
        SBVR_CUDA_TRY(launch_pdl(pages_positions_kernel, dim3((unsigned)n, (unsigned)std::min((tokens_per_seq + 1023) / 1024, 64)), dim3(256), 0,
                                 reinterpret_cast<cudaStream_t>(stream), c, slots, tokens, tokens_each, positions, tokens_per_seq));
    return SBVR_OK;
}

int sbvr_pages_fork(const sbvr_pages_t* cache, const int* src, const int* dst, int n, int share, sbvr_stream_t stream) {
    PgCache c;
    const int rc = pg_cache(cache, &c);
    if (rc) return rc;
    if (!src || !dst || n < 1 || n > c.max_seqs) return SBVR_ERR_BAD_ARG;
    if (n > PG_THREADS) return SBVR_ERR_UNSUPPORTED;
    SBVR_CUDA_TRY(launch_pdl(pages_fork_kernel, dim3(1), dim3(PG_THREADS), seen_bytes(c) + (5 * (size_t)n + 1) * 4, reinterpret_cast<cudaStream_t>(stream), c, src, dst, n, share ? 1 : 0));
    return launch_moves(c, fork_moves_at(c), 0, reinterpret_cast<cudaStream_t>(stream));
}

int sbvr_pages_compact(const sbvr_pages_t* cache, sbvr_stream_t stream) {
    PgCache c;
    const int rc = pg_cache(cache, &c);
    if (rc) return rc;
    SBVR_CUDA_TRY(launch_pdl(pages_compact_kernel, dim3(1), dim3(PG_THREADS), 0, reinterpret_cast<cudaStream_t>(stream), c));
    return launch_moves(c, compact_moves_at(c), 4 + ((c.pages + 3) & ~3), reinterpret_cast<cudaStream_t>(stream));
}

int sbvr_pages_common(const sbvr_pages_t* cache, const int* slots, int n, const int* group_starts, int groups, int* shared, sbvr_stream_t stream) {
    PgCache c;
    const int rc = pg_cache(cache, &c);
    if (rc) return rc;
    if (!group_starts || !shared || n < 1 || groups < 1) return SBVR_ERR_BAD_ARG;
    SBVR_CUDA_TRY(launch_pdl(pages_common_kernel, dim3((unsigned)groups), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), c, slots, group_starts, n, shared));
    return SBVR_OK;
}

int sbvr_pages_rope_append_f16(const sbvr_pages_t* cache, int layer, const void* qkv, const int* positions, const float* inv_freq, float attn_scaling,
                               const int* slots, int seqs, int tokens_per_seq, int n_heads, void* q_out, sbvr_stream_t stream) {
    PgCache c;
    const int rc = pg_cache(cache, &c);
    if (rc) return rc;
    if (!qkv || !positions || !inv_freq || !q_out || layer < 0 || layer >= c.layers || seqs < 1 || tokens_per_seq < 1 || n_heads < 1) return SBVR_ERR_BAD_ARG;
    if (!slots && seqs > c.max_seqs) return SBVR_ERR_BAD_ARG;
    if ((long long)seqs * tokens_per_seq > INT_MAX / 2 || (long long)n_heads + 2 * c.n_kv > INT_MAX / 16) return SBVR_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 15) return SBVR_ERR_ALIGN;
    const size_t tokens = (size_t)seqs * tokens_per_seq;
    if (pg_overlap(qkv, tokens * (n_heads + 2 * c.n_kv) * PG_D * 2, q_out, tokens * n_heads * PG_D * 2)) return SBVR_ERR_BAD_ARG;
    SBVR_CUDA_TRY(launch_pdl(pages_rope_append_kernel, dim3((unsigned)(seqs * tokens_per_seq)), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), c, layer,
                             static_cast<const __half*>(qkv), positions, inv_freq, attn_scaling, slots, tokens_per_seq, n_heads, static_cast<__half*>(q_out)));
    return SBVR_OK;
}

}  // extern "C"
