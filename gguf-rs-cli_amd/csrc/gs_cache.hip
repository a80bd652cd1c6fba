// gs_cache.hip -- the pages of the cache of keys and values: rows grow, are
// forked, freed, lose tokens and are cut to a budget (include/gs_cache.h).
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
    uint32_t row, from;         // fork: dst, src (GS_KV_NONE: none); drop, eviction: the row, its first token that leaves
    uint32_t len, left;         // tokens before and after
    uint32_t old_len;           // fork: tokens of dst before
    uint32_t base;              // its first new page in the list
    uint32_t ok;                // 0: leave the row as it is
    uint32_t in_place;          // drop, eviction: a written page keeps its place
};

// Where the tokens of an eviction were: place x of row i of the call has
// token list[i * ld + x] after it.  Ascending, and never below x.
struct Stays {
    uint32_t *list;
    size_t ld;
    float *mass;                // [rows][ld_mass] (of a drop: or null, and no list)
    size_t ld_mass;
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
// reference counts, the scan): 8 rows 2.7 us of kernel, 256 rows 6.2 (one that reads a
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

// Row rows[blockIdx.x] emptied, with its weights (mass, or null).  Its length is
// taken by an exchange: a row named twice is released once.  (Waits for three
// reads in a row: 3 to 5 us for 8 to 256 rows.)
__global__ void __launch_bounds__(256) free_kernel(const Cache c, const uint32_t *rows, float *mass, size_t ld_mass)
{
    __shared__ uint32_t held;
    const uint32_t row = rows[blockIdx.x];
    if (row >= c.rows) return;
    if (mass)
        for (uint32_t x = threadIdx.x; x < c.ld << c.shift; x += 256) mass[row * ld_mass + x] = 0.0f;
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
// EVICT: what leaves is in moves already (evict_select_kernel).
template <bool EVICT>
__global__ void __launch_bounds__(kBook) drop_plan_kernel(const Cache c, const uint32_t *rows, uint32_t n, const uint32_t *from,
                                                          const uint32_t *to, int32_t *status)
{
    __shared__ uint32_t s_owner[EVICT ? 1 : kOwners];
    if constexpr (!EVICT) claim(c, s_owner, rows, n);
    constexpr int kPlan = 8;            // reads of 64 places that a wave has under way
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t i = threadIdx.x >> 6; i < n; i += kBook / 64) {
        Move m = {};
        if constexpr (EVICT) m = c.moves[i];
        else {
            m.row = rows[i];
            m.ok = m.row < c.rows && claimed(c, s_owner, m.row, i);
        }
        uint32_t need = 0, written = 0;
        if (m.ok) {
            if constexpr (!EVICT) {
                m.len = row_len(c, m.row);
                m.from = min(from[i], m.len);
                m.left = m.len - (min(max(to[i], m.from), m.len) - m.from);
            }
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
// kMoveWhole: an eviction's vectors that are not turned.
enum { kMoveVector, kMovePairs, kMoveValues, kMoveWhole };

// cos and sin of -way positions' angle, where each pair of each token has its
// own: turn_of, in fewer instructions.  The high 32 bits of the product modulo
// 2^64 are the fraction of a turn, off by 2^-32 at most; the nearest quarter turn
// leaves an eighth either way, for which Taylor's series to the ninth and
// eighth power are off by 2e-9 and 3e-8 before their roundings.  (32 rows of 1100 to
// 2500 tokens cut to 1000, us of the move: 446 with turn_of, 384.)
__device__ __forceinline__ float2 turn_back(uint64_t turns, uint32_t way)
{
    const uint32_t part = (uint32_t)(turns >> 32) * way + __umulhi((uint32_t)turns, way);
    const uint32_t quarter = part + 0x20000000u;
    const float x = (float)(int32_t)(part - (quarter & 0xc0000000u)) * 0x1p-32f, y = x * x;
    const float s = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 42.0586939f, -76.7058597f), 81.6052493f), -41.3417022f), 6.28318531f);
    const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, 60.2446414f, -85.4568172f), 64.9393940f), -19.7392088f), 1.0f);
    const bool odd = quarter >> 30 & 1;
    const uint32_t minus_c = (quarter ^ quarter << 1) & 0x80000000u, minus_s = ~quarter & 0x80000000u;
    return make_float2(__uint_as_float(__float_as_uint(odd ? s : c) ^ minus_c), __uint_as_float(__float_as_uint(odd ? c : s) ^ minus_s));
}

// The tokens of one stream (k or v, layer, head: `base`) of row i, kStep
// rounds of 256 items at a time, where an item is a vector, two or a pair of
// values of a token.  All of a step's reads come before its writes, and the
// pages' numbers of the next step are read before both: the reads are what a
// step waits for.  Both go past the caches (2048 of 8192 tokens, 681 MB moved:
// 185 -> 178 us).  EVICT: the tokens come from where `from_list` says, and each
// is turned by its own way.
template <class T, int MODE, bool EVICT>
__device__ __forceinline__ void move_stream(const Cache &c, const Move &m, uint32_t i, T *base, uint32_t h, int rot, bool interleaved,
                                            const float2 *cs, uint32_t t0, uint32_t slice, uint32_t slices, const uint32_t *from_list,
                                            const uint64_t *turns)
{
    // (turning vectors of tokens that each have their own way, eight at a time, takes
    // registers that cost more than they bring: 32 rows of 1100 to 2500 tokens to
    // 1000, us of the call with eight and four: 413, 390)
    constexpr bool kVector = MODE == kMoveVector || MODE == kMoveWhole;
    constexpr int kStep = MODE == kMoveWhole || (MODE == kMoveVector && !EVICT) ? 8 : 4, kW = MODE == kMoveValues ? 1 : 8;
    typedef T vec __attribute__((ext_vector_type(kW)));
    const uint32_t pairs = rot >> 1, size = 1u << c.shift, gone = m.len - m.left;
    const uint32_t nturn = MODE == kMoveWhole ? 0 : MODE == kMoveVector ? rot / 8 : MODE == kMovePairs ? rot / 16 : pairs;
    const uint32_t per = nturn + (MODE == kMoveValues ? (c.d - rot) / 2 : (c.d - rot) / 8);     // items of a token, at most 128
    const uint32_t each = 256 / per, tl = threadIdx.x / per, item = threadIdx.x - tl * per;      // tokens of a round; this thread's
    const bool works = tl < each, turned = item < nturn;
    uint32_t p, q;
    if (kVector) p = q = 8 * item;
    else if (MODE == kMovePairs) { p = turned ? 8 * item : rot + 8 * (item - nturn); q = turned ? p + pairs : p; }
    else { p = turned && !interleaved ? item : 2 * item; q = turned && !interleaved ? item + pairs : p + 1; }
    const uint32_t *table = c.table + (size_t)m.row * c.ld;
    const size_t head = (size_t)c.d << c.shift;

    uint64_t by_turns[EVICT ? kW : 1];          // of this thread's pairs
    if constexpr (EVICT && MODE != kMoveWhole) {
        const int at = MODE == kMoveVector ? 4 * item : kW * item;
#pragma unroll
        for (int e = 0; e < (MODE == kMoveVector ? 4 : kW); e++) by_turns[e] = works && turned ? turns[at + e] : 0;
    }
    uint32_t to[kStep], from[kStep], was[kStep];        // pages, and tokens of the row before
    auto pages = [&](uint32_t t) {
#pragma unroll
        for (int s = 0; s < kStep; s++) {
            const uint32_t x = t + s * each + tl;
            to[s] = from[s] = GS_KV_NONE;
            was[s] = 0;
            if (!works || x >= m.left) continue;
            to[s] = new_page(c, m, i, x >> c.shift);
            was[s] = x < m.from ? x : EVICT ? from_list[x] : x + gone;
            from[s] = table[was[s] >> c.shift];
        }
    };
    if constexpr (EVICT) {                      // as many slices as end together
        const uint32_t all = m.left - min(t0, m.left), one = each * kStep;
        const uint32_t rounds = max((all + slices * one - 1) / (slices * one), 1u);
        slices = max((all + rounds * one - 1) / (rounds * one), 1u);
        if (slice >= slices) return;
    }
    const uint32_t step = slices * each * kStep, begin = t0 + slice * each * kStep;
    pages(begin);
    for (uint32_t t = begin; t < m.left; t += step) {
        vec a[kStep], b[kStep];
        T *at[kStep];
        uint32_t way[kStep];
#pragma unroll
        for (int s = 0; s < kStep; s++) {
            const uint32_t x = t + s * each + tl, y = EVICT ? was[s] : x >= m.from ? x + gone : x;
            if constexpr (EVICT) way[s] = y - x;
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
            if (MODE == kMoveWhole || !at[s] || !turned || t + s * each + tl < m.from) continue;
            auto turn = [&](int pair, int e) { return EVICT ? turn_back(by_turns[EVICT ? e : 0], way[s]) : cs[pair]; };
            if constexpr (MODE == kMoveVector) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float u = (float)a[s][2 * e], w = (float)a[s][2 * e + 1];
                    turn_pair(u, w, turn(4 * item + e, e));
                    a[s][2 * e] = (T)u; a[s][2 * e + 1] = (T)w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < kW; e++) {
                    float u = (float)a[s][e], w = (float)b[s][e];
                    turn_pair(u, w, turn(kW * item + e, e));
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
// EVICT: the same, from where the list says.  8192 tokens to 2048, 28 x 4 streams of
// keys, 235 MB: 53 us, 4.4 TB/s; 6 rows of 20000 to 32768 to 6001, 8 x 8: 5.0 TB/s.
template <class T, int MODE, bool EVICT>
__global__ void __launch_bounds__(256) drop_move_kernel(const Cache c, const uint64_t *turns, int rot, int interleaved, const Stays e)
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
    const uint32_t *list = EVICT ? e.list + i * e.ld : nullptr;
    if (!keys || rot == 0) {
        move_stream<T, EVICT ? kMoveWhole : kMoveVector, EVICT>(c, m, i, base, h, 0, true, cs, t0, slice, slices, list, turns);
        return;
    }
    if constexpr (!EVICT) {
        for (uint32_t e = threadIdx.x; e < (uint32_t)rot >> 1; e += 256) cs[e] = turn_of(turns[e], (int64_t)m.left - m.len, 1.0f);
        __syncthreads();
    }
    move_stream<T, MODE, EVICT>(c, m, i, base, h, rot, interleaved, cs, t0, slice, slices, list, turns);
}

// Drop, 3 of 3: row blockIdx.x's table, its released pages, its length, and its
// weights where there are any, kEach times kThreads at a time: they go down in
// ascending order, and all of a step are read before one is written.  (4.7 us:
// words only.)
template <bool EVICT> __global__ void __launch_bounds__(EVICT ? 1024 : 256) drop_write_kernel(const Cache c, const Stays e)
{
    constexpr uint32_t kThreads = EVICT ? 1024 : 256;
    const uint32_t i = blockIdx.x;
    const Move m = c.moves[i];
    if (!m.ok) return;
    if (EVICT || e.mass) {
        constexpr int kEach = 8;
        float *mass = e.mass + m.row * e.ld_mass;
        const uint32_t *list = EVICT ? e.list + i * e.ld : nullptr, gone = m.len - m.left;
        for (uint32_t x0 = m.from; x0 < m.left; x0 += kEach * kThreads) {
            float w[kEach];
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                const uint32_t x = x0 + k * kThreads + threadIdx.x;
                w[k] = x < m.left ? mass[EVICT ? list[x] : x + gone] : 0.0f;
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kEach; k++) {
                const uint32_t x = x0 + k * kThreads + threadIdx.x;
                if (x < m.left) mass[x] = w[k];
            }
        }
        __syncthreads();            // (the last step's reads are done)
        for (uint32_t x = m.left + threadIdx.x; x < m.len; x += kThreads) mass[x] = 0.0f;
    }
    uint32_t *table = c.table + (size_t)m.row * c.ld;
    const uint32_t now = pages_of(c, m.left), was = pages_of(c, m.len);
    for (uint32_t j = (m.from >> c.shift) + threadIdx.x; j < was; j += kThreads) {
        const uint32_t old = table[j], p = j < now ? new_page(c, m, i, j) : GS_KV_NONE;
        if (p == old) continue;
        if (old < c.n_pages) atomicSub(&c.ref[old], 1u);
        if (p != GS_KV_NONE) c.ref[p] = 1;
        table[j] = p;
    }
    if (threadIdx.x == 0) c.len[m.row] = m.left;
}

// A weight as a whole number that grows with it: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t rank_of(float x)
{
    const uint32_t u = __float_as_uint(x);
    if ((u << 1) > 0xff000000u) return 0xffffffffu;
    if ((u << 1) == 0) return 0x80000000u;
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Eviction, 1 of 4: which tokens of row rows[blockIdx.x] stay.  Of the tokens
// between the first and the newest the k of greatest weight: the rank of the
// k-th is found digit by digit, by counting the weights that share the bits
// found so far; then one pass over the row writes the tokens above it, and the
// lowest of those that have it, to the list.  The first digit has a sign, an
// exponent and four bits more, so that weights of a few powers of two do not all
// meet in the same counts, and kFar weights of a thread are under way at a time.
// (us of 32768 tokens: four digits of 8 bits and one weight at a time 129, of
// which most were atomics of a wave's lanes one after the other; like this 39.)
__global__ void __launch_bounds__(kBook) evict_select_kernel(const Cache c, const uint32_t *rows, const uint32_t *budget,
                                                             uint32_t budget_all, uint32_t first, uint32_t recent, const Stays e)
{
    constexpr int kEach = 4, kFar = 8;  // tokens of a thread in a step of the last pass; reads of the passes before
    constexpr int kBins = 1 << 13;
    __shared__ uint32_t s_count[kBins], s_bin, s_above, s_from;
    const uint32_t i = blockIdx.x, row = rows[i], lane = threadIdx.x & 63;
    bool again = row >= c.rows;         // (a row that an earlier i has counts there)
    for (uint32_t j = threadIdx.x; j < i; j += kBook) again |= rows[j] == row;
    again = __syncthreads_or(again);
    Move m = {};
    m.row = row;
    if (again) {
        if (threadIdx.x == 0) c.moves[i] = m;
        return;
    }
    m.ok = 1;
    m.len = row_len(c, row);
    m.left = min(m.len, budget ? budget[i] : budget_all);
    m.from = m.left;
    if (m.left == m.len) {
        if (threadIdx.x == 0) c.moves[i] = m;
        return;
    }
    const float *mass = e.mass + row * e.ld_mass;
    uint32_t *list = e.list + i * e.ld;
    const uint32_t tail = m.len - min(recent, m.left), head = min(first, m.left - (m.len - tail));
    uint32_t want = m.left - head - (m.len - tail);     // of head .. tail - 1, which are more
    uint32_t rank = 0, known = 0;
    auto digit = [&](auto at, auto bits) {
        constexpr int kShift = decltype(at)::value, kAll = 1 << decltype(bits)::value, kMine = kAll / kBook;    // counts of a thread
        for (uint32_t b = threadIdx.x; b < kAll; b += kBook) s_count[b] = 0;
        __syncthreads();
        for (uint32_t t = head + threadIdx.x; t < tail; t += kBook * kFar) {
            float w[kFar];
#pragma unroll
            for (int k = 0; k < kFar; k++) w[k] = mass[min(t + k * kBook, tail - 1)];
#pragma unroll
            for (int k = 0; k < kFar; k++) {
                const uint32_t r = rank_of(w[k]);
                if (t + k * kBook < tail && (r & known) == rank) atomicAdd(&s_count[r >> kShift & (kAll - 1)], 1u);
            }
        }
        __syncthreads();
        // from the greatest down, kMine counts a thread
        uint32_t x[kMine], sum = 0, total;
#pragma unroll
        for (int k = 0; k < kMine; k++) { x[k] = s_count[kAll - 1 - (kMine * threadIdx.x + k)]; sum += x[k]; }
        uint32_t above = scan(sum, total);
        // (want 0: the greatest, none of which is taken)
        if (want == 0 ? threadIdx.x == 0 : above < want && want <= above + sum) {
            int bin = 0;
#pragma unroll
            for (int k = 0; k + 1 < kMine; k++)
                if (bin == k && want && above + x[k] < want) { above += x[k]; bin++; }
            s_bin = kAll - 1 - (kMine * threadIdx.x + bin);
            s_above = above;
        }
        __syncthreads();
        rank |= s_bin << kShift;
        known |= (uint32_t)(kAll - 1) << kShift;
        want -= s_above;
        __syncthreads();                // (s_bin and the counts are read)
    };
    if (head < tail) {
        digit(std::integral_constant<int, 19>(), std::integral_constant<int, 13>());
        digit(std::integral_constant<int, 9>(), std::integral_constant<int, 10>());
        digit(std::integral_constant<int, 0>(), std::integral_constant<int, 10>());     // (a bit of the last digit again)
    }
    // those of rank `rank`: the lowest `want` stay
    if (threadIdx.x == 0) s_from = m.left;
    uint32_t sure = 0, even = 0;        // before this step's tokens: that stay, and that have that rank
    uint32_t leaves = m.left;           // the first token of the thread's that does
    for (uint32_t t0 = 0; t0 < m.len; t0 += kBook * kEach) {
        uint32_t above = 0, same = 0;   // bits
        float w[kEach];
#pragma unroll
        for (int k = 0; k < kEach; k++) w[k] = mass[min(t0 + threadIdx.x * kEach + k, m.len - 1)];
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const uint32_t t = t0 + threadIdx.x * kEach + k, r = rank_of(w[k]);
            if (t >= m.len) continue;
            const bool must = t < head || t >= tail;
            above |= (uint32_t)(must || r > rank) << k;
            same |= (uint32_t)(!must && r == rank) << k;
        }
        uint32_t total;
        const uint32_t before = scan(__popc(above) | __popc(same) << 16, total);
        uint32_t a = sure + (before & 0xffff), b = even + (before >> 16);
#pragma unroll
        for (int k = 0; k < kEach; k++) {
            const uint32_t t = t0 + threadIdx.x * kEach + k;
            const bool stays = above >> k & 1 || (same >> k & 1 && b < want);
            if (stays) list[a + min(b, want)] = t;
            else if (t < m.len) leaves = min(leaves, t);
            a += above >> k & 1;
            b += same >> k & 1;
        }
        sure += total & 0xffff;
        even += total >> 16;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) leaves = min(leaves, (uint32_t)__shfl_xor(leaves, o));
    if (lane == 0) atomicMin(&s_from, leaves);
    __syncthreads();
    m.from = s_from;
    if (threadIdx.x == 0) c.moves[i] = m;
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

// Weights of the rows' tokens, [rows][ld_mass].
int check_mass(const gs_kv_cache *c, const float *mass, size_t ld_mass)
{
    if (!mass || ((uintptr_t)mass & 3u) || ld_mass < (size_t)c->ld_table * c->page_size) return GS_ERR_INVALID;
    return ld_mass > (size_t)1 << 40 ? GS_ERR_UNSUPPORTED : GS_OK;
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

// (a grid's threads side by side are counted in 32 bits)
bool too_many_streams(const gs_kv_cache *c) { return 2 * (size_t)c->n_layers * c->n_kv * 256 > 0xffffffffull; }

// The tokens of a drop or an eviction to their places.
template <bool EVICT>
void move_tokens(const gs_kv_cache *c, const gs::Cache &d, size_t n, const gs_rope *rope, const gs::Stays &e, hipStream_t st)
{
    const size_t streams = 2 * (size_t)c->n_layers * c->n_kv;
    const int rot = rope ? (int)rope->rot : 0;
    const bool inter = rope && rope->layout == GS_ROPE_INTERLEAVED;
    const uint64_t *turns = rope ? rope->turns : nullptr;
    // Several times as many workgroups as run at a time even out rows of unlike
    // lengths (16 rows of 2500 to 6000 tokens, us: 2048 workgroups 669, 4096
    // 611, 8192 586, 16384 567).
    // An eviction's rows are known to hold no more than the list: each slice has two
    // steps at least of 8192 / d tokens, since workgroups without any cost a launch
    // too (one row of 8192 tokens to 2048, 28 layers of 4 heads: 103 us with 64
    // slices, 90 with 16).
    const size_t most = EVICT && e.ld * c->d / 16384 < 64 ? e.ld * c->d / 16384 + 1 : 64;
    const dim3 grid((unsigned)streams, shares(n * streams, 16384, most), (unsigned)n);
    auto move = [&](auto t, auto mode) {
        hipLaunchKernelGGL((gs::drop_move_kernel<decltype(t), decltype(mode)::value, EVICT>), grid, dim3(256), 0, st, d, turns, rot, inter, e);
    };
    auto typed = [&](auto mode) {
        if (c->type == GS_TYPE_F16) move(_Float16(), mode);
        else move(__bf16(), mode);
    };
    if (rot == 0 || (inter && rot % 8 == 0)) typed(std::integral_constant<int, gs::kMoveVector>());
    else if (!inter && rot % 16 == 0) typed(std::integral_constant<int, gs::kMovePairs>());
    else typed(std::integral_constant<int, gs::kMoveValues>());
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
    return gs_kv_free_mass(c, rows, n, nullptr, 0, stream);
}

int gs_kv_free_mass(const gs_kv_cache *c, const uint32_t *rows, size_t n, float *mass, size_t ld_mass, void *stream)
{
    if (int rc = check_call(c, n)) return rc;
    if (int rc = mass ? check_mass(c, mass, ld_mass) : GS_OK) return rc;
    if (n == 0) return GS_OK;
    if (!rows) return GS_ERR_INVALID;
    hipLaunchKernelGGL(gs::free_kernel, dim3((unsigned)n), dim3(256), 0, (hipStream_t)stream, device_cache(c), rows, mass, ld_mass);
    return launched();
}

int gs_kv_drop(const gs_kv_cache *c, const uint32_t *rows, size_t n, const uint32_t *from, const uint32_t *to,
               const gs_rope *rope, int32_t *status, void *stream)
{
    return gs_kv_drop_mass(c, rows, n, from, to, rope, nullptr, 0, status, stream);
}

int gs_kv_drop_mass(const gs_kv_cache *c, const uint32_t *rows, size_t n, const uint32_t *from, const uint32_t *to,
                    const gs_rope *rope, float *mass, size_t ld_mass, int32_t *status, void *stream)
{
    if (int rc = check_call(c, n)) return rc;
    if (rope && (rope->d != c->d || !is_here(rope))) return GS_ERR_INVALID;
    if (int rc = mass ? check_mass(c, mass, ld_mass) : GS_OK) return rc;
    if (n == 0) return GS_OK;
    if (!rows || !from || !to) return GS_ERR_INVALID;
    if (too_many_streams(c)) return GS_ERR_UNSUPPORTED;
    const gs::Cache d = device_cache(c);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(gs::drop_plan_kernel<false>, dim3(1), dim3(gs::kBook), 0, st, d, rows, (uint32_t)n, from, to, status);
    const gs::Stays e = {nullptr, 0, mass, ld_mass};
    move_tokens<false>(c, d, n, rope, e, st);
    hipLaunchKernelGGL(gs::drop_write_kernel<false>, dim3((unsigned)n), dim3(256), 0, st, d, e);
    return launched();
}

size_t gs_kv_evict_workspace(const gs_kv_cache *c, size_t n, uint32_t budget)
{
    if (check_cache(c) || n > c->rows || n > 65535) return 0;
    const size_t most = (size_t)c->ld_table * c->page_size;
    return ((n ? n : 1) * up4(budget && budget < most ? budget : most)) * 4;
}

int gs_kv_evict(const gs_kv_cache *c, const gs_kv_evict_args *x, void *stream)
{
    if (!x) return GS_ERR_INVALID;
    if (int rc = check_call(c, x->n)) return rc;
    if (x->rope && (x->rope->d != c->d || !is_here(x->rope))) return GS_ERR_INVALID;
    if (x->n == 0) return GS_OK;
    const size_t most = (size_t)c->ld_table * c->page_size;
    if (!x->rows) return GS_ERR_INVALID;
    if (int rc = check_mass(c, x->mass, x->ld_mass)) return rc;
    const uint32_t all = x->budget ? 0 : x->budget_all;
    if (!x->ws || ((uintptr_t)x->ws & 15u) || x->ws_bytes < gs_kv_evict_workspace(c, x->n, all)) return GS_ERR_INVALID;
    if (too_many_streams(c)) return GS_ERR_UNSUPPORTED;
    const gs::Cache d = device_cache(c);
    const gs::Stays e = {(uint32_t *)x->ws, up4(all && all < most ? all : most), x->mass, x->ld_mass};
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(gs::evict_select_kernel, dim3((unsigned)x->n), dim3(gs::kBook), 0, st, d, x->rows, x->budget, x->budget_all,
                       x->first, x->recent, e);
    hipLaunchKernelGGL(gs::drop_plan_kernel<true>, dim3(1), dim3(gs::kBook), 0, st, d, x->rows, (uint32_t)x->n,
                       (const uint32_t *)nullptr, (const uint32_t *)nullptr, x->status);
    move_tokens<true>(c, d, x->n, x->rope, e, st);
    hipLaunchKernelGGL(gs::drop_write_kernel<true>, dim3((unsigned)x->n), dim3(1024), 0, st, d, e);
    return launched();
}

} // extern "C"
