// gs_cache.hip -- the pages of the cache of keys and values: rows grow, are
// forked, freed and lose tokens (include/gs_cache.h).
//
// The bookkeeping is whole numbers in a fixed order, so a call's result does
// not depend on timing: pages are counted over the rows by a scan, taken from
// the free ones in ascending order, and reference counts change by atomic
// additions, whose order does not matter.  A call that takes pages does that
// in one workgroup (the order makes it one chain), and the data moves in a
// second launch over all CUs, which reads the list the first one left in ws.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/gs_cache.h"
#include "gs_cache.hpp"

namespace gs {

constexpr int kBook = 1024;             // threads of the bookkeeping workgroup
constexpr int kScan = 16;               // reference counts per thread and step of the search
constexpr uint32_t kOwners = 8192;      // rows whose marks fit in LDS

// One row of a fork or a drop, in ws.
struct Move {
    uint32_t row, from;         // fork: dst, src (GS_KV_NONE: none); drop: the row, its first token that leaves
    uint32_t len, left;         // tokens before and after
    uint32_t old_len;           // fork: tokens of dst before
    uint32_t base;              // its first new page in the list
    uint32_t ok;                // 0: leave the row as it is
    uint32_t in_place;          // drop: a written page keeps its place
};

struct Cache {
    char *k, *v;
    uint32_t n_layers, n_pages, n_kv, d, rows, ld;
    int shift;                  // log2 of the page size
    uint32_t *table, *len, *ref;
    uint32_t *list;             // [n_pages] the pages taken by the call
    uint32_t *owner;            // [rows] the first i that names a row
    Move *moves;                // [rows]
    uint32_t *stage;            // [rows][ld]
};

__device__ __forceinline__ uint32_t pages_of(const Cache &c, uint32_t len) { return (uint32_t)(((uint64_t)len + (1u << c.shift) - 1) >> c.shift); }

// Tokens of a row, held to what its table has room for.
__device__ __forceinline__ uint32_t row_len(const Cache &c, uint32_t row) { return min(c.len[row], c.ld << c.shift); }

// Exclusive sum over the workgroup's kBook threads; `total` to all.
__device__ __forceinline__ uint32_t scan(uint32_t x, uint32_t &total)
{
    __shared__ uint32_t wave[kBook / 64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t s = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(s, o);
        if (lane >= o) s += y;
    }
    __syncthreads();            // (the last call's readers are done)
    if (lane == 63) wave[w] = s;
    __syncthreads();
    uint32_t before = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < kBook / 64; i++) {
        const uint32_t y = wave[i];
        before += i < w ? y : 0;
        sum += y;
    }
    total = sum;
    return before + s - x;
}

// The free pages from `page` on, ascending, to list[found ..] until it has
// `want`; both run on from call to call of one kernel.  A wave reads 64 counts
// that lie together, kScan times 1024 apart, and the free ones of each such
// read are counted by a ballot; the 256 counts are summed in order by wave 0.
__device__ __forceinline__ void take(const Cache &c, uint32_t want, uint32_t &page, uint32_t &found)
{
    __shared__ uint32_t s_cnt[kScan * kBook / 64 + 1];
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    while (found < want && page < c.n_pages) {
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < kScan; i++) {
            const uint32_t p = page + i * kBook + threadIdx.x;
            if (p < c.n_pages) mask |= (uint32_t)(c.ref[p] == 0) << i;
        }
        uint64_t free[kScan];
#pragma unroll
        for (int i = 0; i < kScan; i++) {
            free[i] = __ballot(mask >> i & 1);
            if (lane == 0) s_cnt[i * (kBook / 64) + w] = __popcll(free[i]);
        }
        __syncthreads();
        if (w == 0) {
            constexpr int kEach = kScan * kBook / 64 / 64;
            uint32_t x[kEach], sum = 0;
#pragma unroll
            for (int i = 0; i < kEach; i++) { x[i] = s_cnt[lane * kEach + i]; sum += x[i]; }
            uint32_t at = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(at, o);
                if ((int)lane >= o) at += y;
            }
            if (lane == 63) s_cnt[kScan * kBook / 64] = at;
            at -= sum;
#pragma unroll
            for (int i = 0; i < kEach; i++) { s_cnt[lane * kEach + i] = at; at += x[i]; }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kScan; i++)
            if (mask >> i & 1)          // (at most n_pages in all)
                c.list[found + s_cnt[i * (kBook / 64) + w] + __popcll(free[i] & ((1ull << lane) - 1))] = page + i * kBook + threadIdx.x;
        found += s_cnt[kScan * kBook / 64];
        page += kBook * kScan;
        __syncthreads();
    }
}

__global__ void reset_kernel(const Cache c)
{
    const size_t n = (size_t)c.rows * c.ld, step = (size_t)gridDim.x * blockDim.x;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
        c.table[i] = GS_KV_NONE;
        if (i < c.rows) c.len[i] = 0;
    }
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < c.n_pages; i += step) c.ref[i] = 0;
}

// The rows' needs are summed 1024 at a time; then each thread writes pages of
// the 1024, whose row it finds in the sums, so one row's many pages (a prompt)
// take no longer than many rows' few.  What bounds it is its chain (lengths,
// reference counts, the scan): 256 rows, 2.5 us of kernel (one that reads a
// word and ends: 1.3).
__global__ void __launch_bounds__(kBook) extend_kernel(const Cache c, const uint32_t *rows, uint32_t n, const uint32_t *add,
                                                       uint32_t add_all, int32_t *status)
{
    __shared__ uint32_t s_first[kBook], s_row[kBook], s_was[kBook];
    uint32_t page = 0, found = 0, given = 0;    // given: needed by the rows before
    for (uint32_t i0 = 0; i0 < n; i0 += kBook) {
        const uint32_t i = i0 + threadIdx.x;
        uint32_t row = 0, len = 0, more = 0, need = 0, was = 0;
        int32_t rc = GS_OK;
        if (i < n) {
            row = rows ? rows[i] : i;
            more = add ? add[i] : add_all;
            if (row >= c.rows) rc = GS_ERR_INVALID;
            else {
                len = row_len(c, row);
                if ((uint64_t)len + more > (uint64_t)c.ld << c.shift) rc = GS_ERR_UNSUPPORTED;
                else { was = pages_of(c, len); need = pages_of(c, len + more) - was; }
            }
        }
        uint32_t total;
        const uint32_t first = scan(need, total);       // (below 2^31: rows * ld fits the table's words)
        take(c, (uint32_t)min((uint64_t)given + total, (uint64_t)c.n_pages), page, found);
        const uint32_t have = found > given ? found - given : 0;
        if (rc == GS_OK && need && (uint64_t)first + need > have) { rc = GS_ERR_NOMEM; }
        s_first[threadIdx.x] = first;
        s_row[threadIdx.x] = rc == GS_OK ? row : GS_KV_NONE;
        s_was[threadIdx.x] = was;
        __syncthreads();
        for (uint32_t p = threadIdx.x; p < min(total, have); p += kBook) {
            uint32_t lo = 0, hi = kBook - 1;            // the last thread whose pages begin at or before p
            while (lo < hi) {
                const uint32_t mid = (lo + hi + 1) >> 1;
                if (s_first[mid] <= p) lo = mid;
                else hi = mid - 1;
            }
            if (s_row[lo] == GS_KV_NONE) continue;
            const uint32_t id = c.list[given + p];
            c.table[(size_t)s_row[lo] * c.ld + s_was[lo] + (p - s_first[lo])] = id;
            c.ref[id] = 1;
        }
        if (i < n) {
            if (rc == GS_OK) c.len[row] = len + more;
            if (status) status[i] = rc;
        }
        given = (uint32_t)min((uint64_t)given + total, 0xffffffffull);
        __syncthreads();
    }
}

// Marks, for each row named, the first i that names it: in LDS, or for caches
// of more than kOwners rows in ws.  (Device-scope accesses there: the marks
// are in L2.)
__device__ __forceinline__ void claim(const Cache &c, uint32_t *owner, const uint32_t *rows, uint32_t n)
{
    const bool local = c.rows <= kOwners;
    for (uint32_t i = threadIdx.x; i < n; i += kBook) {
        const uint32_t r = rows[i];
        if (r >= c.rows) continue;
        if (local) owner[r] = GS_KV_NONE;
        else __hip_atomic_store(&c.owner[r], GS_KV_NONE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!local) __threadfence();
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kBook) {
        const uint32_t r = rows[i];
        if (r < c.rows) atomicMin(local ? &owner[r] : &c.owner[r], i);
    }
    if (!local) __threadfence();
    __syncthreads();
}

__device__ __forceinline__ bool claimed(const Cache &c, const uint32_t *owner, uint32_t row, uint32_t i)
{
    return (c.rows <= kOwners ? owner[row] : __hip_atomic_load(&c.owner[row], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == i;
}

// Fork, 1 of 3: which pairs go ahead, and the page for each partial last page.
// A chain again (marks, lengths, counts): 8 to 256 pairs, 4.8 us.
__global__ void __launch_bounds__(kBook) fork_plan_kernel(const Cache c, const uint32_t *src, const uint32_t *dst, uint32_t n,
                                                          int32_t *status)
{
    __shared__ uint32_t s_owner[kOwners];
    claim(c, s_owner, dst, n);
    uint32_t page = 0, found = 0, given = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += kBook) {
        const uint32_t i = i0 + threadIdx.x;
        Move m = {};
        uint32_t need = 0;
        int32_t rc = GS_OK;
        if (i < n) {
            m.row = dst[i];
            m.from = src[i];
            if (m.row >= c.rows || (m.from >= c.rows && m.from != GS_KV_NONE) || !claimed(c, s_owner, m.row, i)) rc = GS_ERR_INVALID;
            else if (m.from != m.row) {
                m.ok = 1;
                m.old_len = row_len(c, m.row);
                m.len = m.from == GS_KV_NONE ? 0 : row_len(c, m.from);
                need = (m.len & ((1u << c.shift) - 1)) != 0;
            }
        }
        uint32_t total;
        const uint32_t first = scan(need, total);
        take(c, min(given + total, c.n_pages), page, found);
        if (need) {
            if (given + first >= found) { rc = GS_ERR_NOMEM; m.ok = 0; }
            else {
                m.base = c.list[given + first];
                c.ref[m.base] = 1;
            }
        }
        if (i < n) {
            c.moves[i] = m;
            if (status) status[i] = rc;
        }
        given += total;
        __syncthreads();
    }
}

// Fork, 2 of 3: pair blockIdx.x.  The new table to `stage` (rows of the call
// may be each other's sources), the shared pages counted, and the partial
// page's tokens copied: a wave moves one (k or v, layer, head) piece, which is
// contiguous; blockIdx.y shares the pieces out.  What bounds it is the write:
// 16 rows forked to 256, 340 MB: 93 us, 3.6 TB/s (the 16 sources stay in the
// caches); one row to 8, 11 MB: 4.4 us.
template <bool PAST> __global__ void __launch_bounds__(256) fork_copy_kernel(const Cache c)
{
    const Move m = c.moves[blockIdx.x];
    if (!m.ok || m.from == GS_KV_NONE) return;
    const uint32_t full = m.len >> c.shift, rest = m.len & ((1u << c.shift) - 1);
    const uint32_t *from = c.table + (size_t)m.from * c.ld;
    for (uint32_t j = blockIdx.y * 256 + threadIdx.x; j < full; j += gridDim.y * 256) {
        const uint32_t p = from[j];
        c.stage[(size_t)blockIdx.x * c.ld + j] = p;
        if (p < c.n_pages) atomicAdd(&c.ref[p], 1u);
    }
    if (!rest) return;
    const uint32_t old = from[full];
    if (old >= c.n_pages) return;
    const size_t slot = (size_t)c.d * 2, head = slot << c.shift, plane = (size_t)c.n_pages * c.n_kv * head;
    const uint32_t lane = threadIdx.x & 63, pieces = 2 * c.n_layers * c.n_kv;
    const size_t bytes = rest * slot;
    for (uint32_t q = blockIdx.y * 4 + (threadIdx.x >> 6); q < pieces; q += gridDim.y * 4) {
        const uint32_t h = q % c.n_kv, l = q / c.n_kv >> 1;
        char *base = (q / c.n_kv & 1 ? c.v : c.k) + l * plane;
        const char *a = base + ((size_t)old * c.n_kv + h) * head;
        char *b = base + ((size_t)m.base * c.n_kv + h) * head;
        for (size_t o = lane * 16; o < bytes; o += 64 * 16) store<PAST>((u4v *)(b + o), *(const u4v *)(a + o));
    }
}

// Fork, 3 of 3: pair blockIdx.x's old pages released, the new table written.
// (8 pairs 2.4 us, 256 4.8: words only.)
__global__ void __launch_bounds__(256) fork_write_kernel(const Cache c)
{
    const Move m = c.moves[blockIdx.x];
    if (!m.ok) return;
    uint32_t *table = c.table + (size_t)m.row * c.ld;
    const uint32_t full = m.len >> c.shift, now = pages_of(c, m.len), was = pages_of(c, m.old_len);
    for (uint32_t j = threadIdx.x; j < max(now, was); j += 256) {
        if (j < was && table[j] < c.n_pages) atomicSub(&c.ref[table[j]], 1u);
        table[j] = j < full ? c.stage[(size_t)blockIdx.x * c.ld + j] : j < now ? m.base : GS_KV_NONE;
    }
    if (threadIdx.x == 0) c.len[m.row] = m.len;
}

// Row rows[blockIdx.x] emptied.  Its length is taken by an exchange: a row
// named twice is released once.  (Waits for three reads in a row: 3 to 5 us for
// 8 to 256 rows.)
__global__ void __launch_bounds__(256) free_kernel(const Cache c, const uint32_t *rows)
{
    __shared__ uint32_t held;
    const uint32_t row = rows[blockIdx.x];
    if (row >= c.rows) return;
    if (threadIdx.x == 0) held = min(atomicExch(&c.len[row], 0u), c.ld << c.shift);
    __syncthreads();
    uint32_t *table = c.table + (size_t)row * c.ld;
    for (uint32_t j = threadIdx.x; j < pages_of(c, held); j += 256) {
        if (table[j] < c.n_pages) atomicSub(&c.ref[table[j]], 1u);
        table[j] = GS_KV_NONE;
    }
}

// Drop, 1 of 3: what leaves each row, and the new pages for its written pages
// that others hold too.  A wave counts a row's pages; stage[i][j] is the
// number of new pages before place j, with the top bit where j gets one.  (One
// row of 512 pages or 16 of up to 94: 6.7 us, a chain of reads.)
__global__ void __launch_bounds__(kBook) drop_plan_kernel(const Cache c, const uint32_t *rows, uint32_t n, const uint32_t *from,
                                                          const uint32_t *to, int32_t *status)
{
    __shared__ uint32_t s_owner[kOwners];
    claim(c, s_owner, rows, n);
    constexpr int kPlan = 8;            // reads of 64 places that a wave has under way
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t i = threadIdx.x >> 6; i < n; i += kBook / 64) {
        Move m = {};
        m.row = rows[i];
        m.ok = m.row < c.rows && claimed(c, s_owner, m.row, i);
        uint32_t need = 0, written = 0;
        if (m.ok) {
            m.len = row_len(c, m.row);
            m.from = min(from[i], m.len);
            m.left = m.len - (min(max(to[i], m.from), m.len) - m.from);
            const uint32_t first = m.from >> c.shift, now = pages_of(c, m.left);
            if (m.left < m.len) {
                const uint32_t *table = c.table + (size_t)m.row * c.ld;
                for (uint32_t j = first; j < now; j += 64 * kPlan) {
                    uint32_t p[kPlan], held[kPlan];
#pragma unroll
                    for (int e = 0; e < kPlan; e++) p[e] = j + 64 * e + lane < now ? table[j + 64 * e + lane] : GS_KV_NONE;
#pragma unroll
                    for (int e = 0; e < kPlan; e++) held[e] = p[e] < c.n_pages ? c.ref[p[e]] : 0;
#pragma unroll
                    for (int e = 0; e < kPlan; e++) {
                        const bool fresh = held[e] > 1;
                        const uint64_t b = __ballot(fresh);
                        if (j + 64 * e + lane < now)
                            c.stage[(size_t)i * c.ld + j + 64 * e + lane] =
                                (need + __popcll(b & ((1ull << lane) - 1))) | (fresh ? 0x80000000u : 0u);
                        need += __popcll(b);
                    }
                }
                written = now > first ? now - first : 0;
            }
        }
        m.in_place = need < written;
        m.base = need;                  // (for the moment)
        if (lane == 0) c.moves[i] = m;
    }
    __threadfence_block();
    __syncthreads();
    uint32_t page = 0, found = 0, given = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += kBook) {
        const uint32_t i = i0 + threadIdx.x;
        Move m = {};
        uint32_t total;
        if (i < n) m = c.moves[i];
        const uint32_t need = m.base, first = scan(need, total);
        take(c, (uint32_t)min((uint64_t)given + total, (uint64_t)c.n_pages), page, found);
        if (i < n) {
            int32_t rc = m.ok ? GS_OK : GS_ERR_INVALID;
            if (need && (uint64_t)given + first + need > found) { m.ok = 0; rc = GS_ERR_NOMEM; }
            m.base = given + first;
            m.ok = m.ok && m.left < m.len;
            c.moves[i] = m;
            if (status) status[i] = rc;
        }
        given = (uint32_t)min((uint64_t)given + total, 0xffffffffull);
        __syncthreads();
    }
}

// The page that place j of row i of a drop has after it.
__device__ __forceinline__ uint32_t new_page(const Cache &c, const Move &m, uint32_t i, uint32_t j)
{
    if (j >= m.from >> c.shift) {
        const uint32_t s = c.stage[(size_t)i * c.ld + j];
        if (s >> 31) return c.list[m.base + (s & 0x7fffffffu)];
    }
    return c.table[(size_t)m.row * c.ld + j];
}

// How a stream's values move: as they are or turned within vectors of 8 (the
// interleaved layout); turned in pairs of vectors (the half layout); or value
// by value, where the turned part is no whole number of such vectors.
enum { kMoveVector, kMovePairs, kMoveValues };

// The tokens of one stream (k or v, layer, head: `base`) of row i, kStep
// rounds of 256 items at a time, where an item is a vector, two or a pair of
// values of a token.  All of a step's reads come before its writes, and the
// pages' numbers of the next step are read before both: the reads are what a
// step waits for.  Both go past the caches (2048 of 8192 tokens, 681 MB moved:
// 185 -> 178 us).
template <class T, int MODE>
__device__ __forceinline__ void move_stream(const Cache &c, const Move &m, uint32_t i, T *base, uint32_t h, int rot, bool interleaved,
                                            const float2 *cs, uint32_t t0, uint32_t slice, uint32_t slices)
{
    constexpr int kStep = MODE == kMoveVector ? 8 : 4, kW = MODE == kMoveValues ? 1 : 8;
    typedef T vec __attribute__((ext_vector_type(kW)));
    const uint32_t pairs = rot >> 1, size = 1u << c.shift, gone = m.len - m.left;
    const uint32_t nturn = MODE == kMoveVector ? rot / 8 : MODE == kMovePairs ? rot / 16 : pairs;
    const uint32_t per = nturn + (MODE == kMoveValues ? (c.d - rot) / 2 : (c.d - rot) / 8);     // items of a token, at most 128
    const uint32_t each = 256 / per, tl = threadIdx.x / per, item = threadIdx.x - tl * per;      // tokens of a round; this thread's
    const bool works = tl < each, turned = item < nturn;
    uint32_t p, q;
    if (MODE == kMoveVector) p = q = 8 * item;
    else if (MODE == kMovePairs) { p = turned ? 8 * item : rot + 8 * (item - nturn); q = turned ? p + pairs : p; }
    else { p = turned && !interleaved ? item : 2 * item; q = turned && !interleaved ? item + pairs : p + 1; }
    const uint32_t *table = c.table + (size_t)m.row * c.ld;
    const size_t head = (size_t)c.d << c.shift;

    uint32_t to[kStep], from[kStep];            // pages
    auto pages = [&](uint32_t t) {
#pragma unroll
        for (int s = 0; s < kStep; s++) {
            const uint32_t x = t + s * each + tl;
            to[s] = from[s] = GS_KV_NONE;
            if (!works || x >= m.left) continue;
            to[s] = new_page(c, m, i, x >> c.shift);
            from[s] = table[(x >= m.from ? x + gone : x) >> c.shift];
        }
    };
    const uint32_t step = slices * each * kStep;
    pages(t0 + slice * each * kStep);
    for (uint32_t t = t0 + slice * each * kStep; t < m.left; t += step) {
        vec a[kStep], b[kStep];
        T *at[kStep];
#pragma unroll
        for (int s = 0; s < kStep; s++) {
            const uint32_t x = t + s * each + tl, y = x >= m.from ? x + gone : x;
            at[s] = nullptr;
            if (to[s] >= c.n_pages || from[s] >= c.n_pages) continue;
            const T *f = base + ((size_t)from[s] * c.n_kv + h) * head + (y & (size - 1)) * c.d;
            at[s] = base + ((size_t)to[s] * c.n_kv + h) * head + (x & (size - 1)) * c.d;
            a[s] = __builtin_nontemporal_load((const vec *)(f + p));
            if (MODE == kMoveValues || (MODE == kMovePairs && turned)) b[s] = __builtin_nontemporal_load((const vec *)(f + q));
        }
        pages(t + step);
#pragma unroll
        for (int s = 0; s < kStep; s++) {
            if (!at[s] || !turned || t + s * each + tl < m.from) continue;
            if constexpr (MODE == kMoveVector) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float u = (float)a[s][2 * e], w = (float)a[s][2 * e + 1];
                    turn_pair(u, w, cs[4 * item + e]);
                    a[s][2 * e] = (T)u; a[s][2 * e + 1] = (T)w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < kW; e++) {
                    float u = (float)a[s][e], w = (float)b[s][e];
                    turn_pair(u, w, cs[kW * item + e]);
                    a[s][e] = (T)u; b[s][e] = (T)w;
                }
            }
        }
        if (m.in_place) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // every read of the step is done
            __syncthreads();
        }
#pragma unroll
        for (int s = 0; s < kStep; s++) {
            if (!at[s]) continue;
            __builtin_nontemporal_store(a[s], (vec *)(at[s] + p));
            if (MODE == kMoveValues || (MODE == kMovePairs && turned)) __builtin_nontemporal_store(b[s], (vec *)(at[s] + q));
        }
    }
}

// Drop, 2 of 3: the tokens move.  blockIdx.x: a stream of row blockIdx.z.
// Tokens go down in ascending order and a step's reads are all done before its
// writes, so a workgroup that has the stream alone may write over what it has
// read.  Rows all of whose written pages are new are read from other pages
// than they are written to, and their steps are shared by gridDim.y
// workgroups.  What bounds it is memory: 2048 of 8192 tokens of 28 x 4 streams
// of keys and as many of values, 681 MB, shared pages: 136 to 152 us, 4.5 to 5.0
// TB/s (a copy: 5.15); in place, by one workgroup per stream, 3.5 TB/s with 224
// streams and 4.6 with 2048.
// MODE: of keys that are turned.
template <class T, int MODE>
__global__ void __launch_bounds__(256) drop_move_kernel(const Cache c, const uint64_t *turns, int rot, int interleaved)
{
    __shared__ float2 cs[128];
    const uint32_t i = blockIdx.z, stream = blockIdx.x;
    const Move m = c.moves[i];
    if (!m.ok || (m.in_place && blockIdx.y)) return;
    const uint32_t slice = blockIdx.y, slices = m.in_place ? 1 : gridDim.y;
    const uint32_t h = stream % c.n_kv, l = stream / c.n_kv >> 1;
    const bool keys = !(stream / c.n_kv & 1);
    // tokens before `from` move only where their page is a new one
    const uint32_t first = m.from >> c.shift;
    const bool fresh = first < pages_of(c, m.left) && (c.stage[(size_t)i * c.ld + first] >> 31);
    const uint32_t t0 = fresh ? first << c.shift : m.from;
    T *base = (T *)(keys ? c.k : c.v) + (size_t)l * c.n_pages * c.n_kv * ((size_t)c.d << c.shift);
    if (!keys || rot == 0) {
        move_stream<T, kMoveVector>(c, m, i, base, h, 0, true, cs, t0, slice, slices);
        return;
    }
    for (uint32_t e = threadIdx.x; e < (uint32_t)rot >> 1; e += 256) cs[e] = turn_of(turns[e], (int64_t)m.left - m.len, 1.0f);
    __syncthreads();
    move_stream<T, MODE>(c, m, i, base, h, rot, interleaved, cs, t0, slice, slices);
}

// Drop, 3 of 3: row blockIdx.x's table, its released pages, its length.  (4.7
// us: words only.)
__global__ void __launch_bounds__(256) drop_write_kernel(const Cache c)
{
    const uint32_t i = blockIdx.x;
    const Move m = c.moves[i];
    if (!m.ok) return;
    uint32_t *table = c.table + (size_t)m.row * c.ld;
    const uint32_t now = pages_of(c, m.left), was = pages_of(c, m.len);
    for (uint32_t j = (m.from >> c.shift) + threadIdx.x; j < was; j += 256) {
        const uint32_t old = table[j], p = j < now ? new_page(c, m, i, j) : GS_KV_NONE;
        if (p == old) continue;
        if (old < c.n_pages) atomicSub(&c.ref[old], 1u);
        if (p != GS_KV_NONE) c.ref[p] = 1;
        table[j] = p;
    }
    if (threadIdx.x == 0) c.len[m.row] = m.left;
}

} // namespace gs

namespace {

size_t up4(size_t x) { return (x + 3) & ~(size_t)3; }

gs::Cache device_cache(const gs_kv_cache *c)
{
    gs::Cache d = {};
    d.k = (char *)c->k; d.v = (char *)c->v;
    d.n_layers = c->n_layers; d.n_pages = c->n_pages; d.n_kv = c->n_kv; d.d = c->d; d.rows = c->rows; d.ld = c->ld_table;
    d.shift = log2_of(c->page_size);
    d.table = c->table; d.len = c->len; d.ref = c->ref;
    uint32_t *w = c->ws;
    d.list = w; w += up4(c->n_pages);
    d.owner = w; w += up4(c->rows);
    d.moves = (gs::Move *)w; w += (size_t)c->rows * (sizeof(gs::Move) / 4);
    d.stage = w;
    return d;
}

int check_call(const gs_kv_cache *c, size_t n)
{
    if (int rc = check_cache(c)) return rc;
    if (!c->ws || ((uintptr_t)c->ws & 15u)) return GS_ERR_INVALID;
    return n <= c->rows && n <= 65535 ? GS_OK : GS_ERR_INVALID;     // (a grid's second and third sizes)
}

int launched() { return hipGetLastError() == hipSuccess ? GS_OK : GS_ERR_HIP; }

// Workgroups that share each of n pieces of data, up to `most`, so that there
// are `all`.
unsigned shares(size_t n, size_t all, size_t most)
{
    size_t s = (all + n - 1) / n;
    if (s > most) s = most;
    return (unsigned)(s ? s : 1);
}

} // namespace

extern "C" {

size_t gs_kv_workspace(const gs_kv_cache *c)
{
    if (check_cache(c)) return 0;
    return up4(c->n_pages) + up4(c->rows) + (size_t)c->rows * (sizeof(gs::Move) / 4) + (size_t)c->rows * c->ld_table;
}

int gs_kv_reset(const gs_kv_cache *c, void *stream)
{
    if (int rc = check_call(c, 0)) return rc;
    hipLaunchKernelGGL(gs::reset_kernel, dim3(1024), dim3(256), 0, (hipStream_t)stream, device_cache(c));
    return launched();
}

int gs_kv_extend(const gs_kv_cache *c, const uint32_t *rows, size_t n, const uint32_t *add, uint32_t add_all,
                 int32_t *status, void *stream)
{
    if (int rc = check_call(c, 0)) return rc;
    if (n > c->rows) return GS_ERR_INVALID;         // (one workgroup: any number of rows)
    if (n == 0) return GS_OK;
    hipLaunchKernelGGL(gs::extend_kernel, dim3(1), dim3(gs::kBook), 0, (hipStream_t)stream, device_cache(c), rows, (uint32_t)n,
                       add, add_all, status);
    return launched();
}

int gs_kv_fork(const gs_kv_cache *c, const uint32_t *src, const uint32_t *dst, size_t n, int32_t *status, void *stream)
{
    if (int rc = check_call(c, n)) return rc;
    if (n == 0) return GS_OK;
    if (!src || !dst) return GS_ERR_INVALID;
    const gs::Cache d = device_cache(c);
    hipStream_t st = (hipStream_t)stream;
    const unsigned y = shares(n, 2048, (2 * (size_t)c->n_layers * c->n_kv + 3) / 4);
    hipLaunchKernelGGL(gs::fork_plan_kernel, dim3(1), dim3(gs::kBook), 0, st, d, src, dst, (uint32_t)n, status);
    // (at most a page of every layer for each pair; half of it on average)
    const bool past = n * c->n_layers * c->n_kv * c->page_size * c->d * 2 > kPastCaches;
    if (past) hipLaunchKernelGGL(gs::fork_copy_kernel<true>, dim3((unsigned)n, y), dim3(256), 0, st, d);
    else hipLaunchKernelGGL(gs::fork_copy_kernel<false>, dim3((unsigned)n, y), dim3(256), 0, st, d);
    hipLaunchKernelGGL(gs::fork_write_kernel, dim3((unsigned)n), dim3(256), 0, st, d);
    return launched();
}

int gs_kv_free(const gs_kv_cache *c, const uint32_t *rows, size_t n, void *stream)
{
    if (int rc = check_call(c, n)) return rc;
    if (n == 0) return GS_OK;
    if (!rows) return GS_ERR_INVALID;
    hipLaunchKernelGGL(gs::free_kernel, dim3((unsigned)n), dim3(256), 0, (hipStream_t)stream, device_cache(c), rows);
    return launched();
}

int gs_kv_drop(const gs_kv_cache *c, const uint32_t *rows, size_t n, const uint32_t *from, const uint32_t *to,
               const gs_rope *rope, int32_t *status, void *stream)
{
    if (int rc = check_call(c, n)) return rc;
    if (rope && (rope->d != c->d || !is_here(rope))) return GS_ERR_INVALID;
    if (n == 0) return GS_OK;
    if (!rows || !from || !to) return GS_ERR_INVALID;
    const gs::Cache d = device_cache(c);
    hipStream_t st = (hipStream_t)stream;
    const size_t streams = 2 * (size_t)c->n_layers * c->n_kv;
    if (streams * 256 > 0xffffffffull) return GS_ERR_UNSUPPORTED;       // (a grid's threads side by side)
    const int rot = rope ? (int)rope->rot : 0;
    const bool inter = rope && rope->layout == GS_ROPE_INTERLEAVED;
    const uint64_t *turns = rope ? rope->turns : nullptr;
    // Several times as many workgroups as run at a time even out rows of unlike
    // lengths (16 rows of 2500 to 6000 tokens, us: 2048 workgroups 669, 4096
    // 611, 8192 586, 16384 567).
    const dim3 grid((unsigned)streams, shares(n * streams, 16384, 64), (unsigned)n);
    hipLaunchKernelGGL(gs::drop_plan_kernel, dim3(1), dim3(gs::kBook), 0, st, d, rows, (uint32_t)n, from, to, status);
    auto move = [&](auto t, auto mode) {
        hipLaunchKernelGGL((gs::drop_move_kernel<decltype(t), decltype(mode)::value>), grid, dim3(256), 0, st, d, turns, rot, inter);
    };
    auto typed = [&](auto mode) {
        if (c->type == GS_TYPE_F16) move(_Float16(), mode);
        else move(__bf16(), mode);
    };
    if (rot == 0 || (inter && rot % 8 == 0)) typed(std::integral_constant<int, gs::kMoveVector>());
    else if (!inter && rot % 16 == 0) typed(std::integral_constant<int, gs::kMovePairs>());
    else typed(std::integral_constant<int, gs::kMoveValues>());
    hipLaunchKernelGGL(gs::drop_write_kernel, dim3((unsigned)n), dim3(256), 0, st, d);
    return launched();
}

} // extern "C"
