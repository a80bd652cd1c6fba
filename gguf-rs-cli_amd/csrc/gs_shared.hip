// gs_shared.hip -- attention of families of rows that begin with the same pages
// (gs_attn_shared, include/gs_attn.h).
//
// Softmax over two sets of keys is joined from each one's maximum, sum and
// weighted values, so the keys that a family's rows have in common are a job of
// their own: its query rows are those of all the family's tokens beside one
// another, which see every key of it (but for their windows), and keys and
// values are read once.  Each sequence's other keys are a second job.  Both
// kinds go through the kernels of gs_attn.hpp, and one more kernel joins each
// row's parts.  Which pages are common is read from the table, by each call.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "gs_attn.hpp"

namespace gs {

constexpr int kPlan = 1024;

// The jobs of family blockIdx.x and its sequences, and their tokens' positions.
// The common keys are whole pages that the tables of all rows with new tokens
// have alike, and that all of the family's new tokens come after.  What bounds
// it is its chain of reads (begins, rows, lengths, tables), so the tables are
// compared kTables pieces of 64 pages at a time.  (us: 4 rows over 600 tokens 5.5,
// 64 over 16000 in pages of 64 10, 32 over 30000 in pages of 32 15.)  Workgroups
// beyond the families only mark rows.
__global__ void __launch_bounds__(kPlan) shared_plan_kernel(const AttnArgs a, const uint32_t *families, uint32_t n, Job *jobs, int32_t *pos)
{
    constexpr int kTables = 16;
    __shared__ uint32_t s_pages, s_first, s_end, s_lead, s_count, s_row[kPlan];
    __shared__ int32_t s_p0, s_p1;
    const uint32_t j = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    // (tokens of no sequence are left as they are)
    const size_t rows = (size_t)a.n_tokens * a.n_kv * a.group;
    for (size_t i = (size_t)j * kPlan + threadIdx.x; i < rows; i += (size_t)gridDim.x * kPlan) a.where[rows + i] = kDone;
    if (j >= a.n_families) return;
    const uint32_t s0 = min(families[j], n), s1 = max(min(families[j + 1], n), s0);
    auto sequence = [&](uint32_t i) {
        Job x = {};
        x.first = a.start ? min(a.start[i], a.n_tokens) : i;
        const uint32_t end = a.start ? min(a.start[i + 1], a.n_tokens) : i + 1;
        x.nq = end > x.first ? end - x.first : 0;
        x.row = a.rows ? a.rows[i] : i;
        x.len = x.row < a.n_rows ? min(a.len[x.row], a.ld_table << a.shift) : 0;
        x.k1 = x.len;
        return x;
    };
    if (threadIdx.x == 0) {
        s_pages = a.ld_table;
        s_first = 0xffffffffu; s_end = 0; s_lead = 0xffffffffu; s_count = 0;
        s_p0 = 0x7fffffff; s_p1 = -1;
    }
    __syncthreads();
    // the sequences with new tokens: how many, the first of them, their positions, pages before the earliest token
    // (a wave's first, and then one atomic of each: 64 of them to one word take a microsecond)
    if (s0 + 64 * w < s1) {
        uint32_t pages = a.ld_table, first = 0xffffffffu, end = 0, before = 0xffffffffu, count = 0;
        int32_t p0 = 0x7fffffff, p1 = -1;
        for (uint32_t i = s0 + threadIdx.x; i < s1; i += kPlan) {
            const Job x = sequence(i);
            if (x.nq == 0) continue;
            pages = min(pages, x.len > x.nq ? (x.len - x.nq) >> a.shift : 0);
            p0 = min(p0, (int32_t)(x.len - x.nq));
            p1 = max(p1, (int32_t)x.len - 1);
            first = min(first, x.first);
            end = max(end, x.first + x.nq);
            before = min(before, i);
            count++;
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            pages = min(pages, (uint32_t)__shfl_xor(pages, o));
            p0 = min(p0, __shfl_xor(p0, o));
            p1 = max(p1, __shfl_xor(p1, o));
            first = min(first, (uint32_t)__shfl_xor(first, o));
            end = max(end, (uint32_t)__shfl_xor(end, o));
            before = min(before, (uint32_t)__shfl_xor(before, o));
            count += __shfl_xor(count, o);
        }
        if (lane == 0) {
            atomicMin(&s_pages, pages);
            atomicMin(&s_p0, p0);
            atomicMax(&s_p1, p1);
            atomicMin(&s_first, first);
            atomicMax(&s_end, end);
            atomicMin(&s_lead, before);
            atomicAdd(&s_count, count);
        }
    }
    __syncthreads();
    const uint32_t most = s_count > 1 ? s_pages : 0;
    uint32_t lead = 0;
    if (most) {
        // (every row with new tokens is there: it has pages before them)
        lead = a.rows ? a.rows[s_lead] : s_lead;
        const uint32_t *t0 = a.table + (size_t)lead * a.ld_table;
        const uint32_t pieces = (most + 63) / 64;
        uint32_t least = most;
        for (uint32_t i0 = s0; i0 < s1; i0 += kPlan) {          // the rows of up to kPlan sequences, `lead` for those without tokens
            const uint32_t m = min(s1 - i0, (uint32_t)kPlan);
            __syncthreads();
            if (threadIdx.x < m) {
                const Job y = sequence(i0 + threadIdx.x);
                s_row[threadIdx.x] = y.nq ? y.row : lead;
            }
            __syncthreads();
            const uint32_t all = m * pieces;                    // (below 2^30: a table has at most 2^26 places)
            for (uint32_t x0 = w; x0 < all; x0 += kPlan / 64 * kTables) {
                uint32_t p[kTables], mine[kTables], other[kTables];
#pragma unroll
                for (int e = 0; e < kTables; e++) {
                    const uint32_t x = min(x0 + kPlan / 64 * e, all - 1), i = x / pieces;
                    p[e] = min(64 * (x - i * pieces) + lane, most - 1);
                    mine[e] = t0[p[e]];
                    other[e] = a.table[(size_t)s_row[i] * a.ld_table + p[e]];
                }
#pragma unroll
                for (int e = 0; e < kTables; e++)
                    if (mine[e] != other[e]) least = min(least, p[e]);
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) least = min(least, (uint32_t)__shfl_xor(least, o));
        __syncthreads();                    // (s_pages is read)
        if (lane == 0) atomicMin(&s_pages, least);
    }
    __syncthreads();
    const uint32_t common = most ? s_pages << a.shift : 0;
    auto write = [&](uint32_t i, uint32_t k0) {         // (a wave)
        Job x = sequence(i);
        x.k0 = k0;
        if (lane == 0) jobs[a.n_families + i] = x;
        for (uint32_t t = lane; t < x.nq; t += 64) pos[x.first + t] = (int32_t)x.len - (int32_t)x.nq + (int32_t)t;
    };
    for (uint32_t i = s0 + w; i < s1; i += kPlan / 64) write(i, common);
    if (threadIdx.x == 0) {
        Job x = {};
        x.row = lead;
        x.len = kFamily;
        x.first = common ? s_first : 0;
        x.nq = common ? s_end - s_first : 0;
        x.k1 = common;
        x.p0 = s_p0;
        x.p1 = s_p1;
        jobs[j] = x;
    }
    // sequences of no family
    if (j == 0)
        for (uint32_t i = w; i < s0; i += kPlan / 64) write(i, 0);
    if (j + 1 == a.n_families)
        for (uint32_t i = s1 + w; i < n; i += kPlan / 64) write(i, 0);
}

// Where the parts of one of a row's jobs are.
struct Parts {
    const float *o, *m;         // the first one's values and maximum
    size_t more, skip;          // from the first to the second, from there on
    uint32_t n, sum;            // how many; from a maximum to its sum
    float lift;
};

// A row of a token and head, by D / 4 threads: the parts of its two jobs.
// The threads share out the parts' maximums and sums and then add the parts in
// order, kFar reads at a time: what bounds it is the chain of reads (the word that
// says where, maximums and sums, values).  (us: 64 tokens of 28 heads, some 20
// parts a row, 9.8; 16 at a time is no faster.)
// R1, R2: rows of a unit of the call's two kernels.
template <class TO, int D, int R1, int R2>
__global__ void __launch_bounds__(256) shared_join_kernel(const AttnArgs a, const float *parts2, float lift2)
{
    constexpr int kCols = D / 4, kRows = 256 / kCols, kWide = kCols < 32 ? kCols : 32, kFar = 8;
    const uint32_t heads = a.n_kv * a.group;
    const size_t rows = (size_t)a.n_tokens * heads, row = (size_t)blockIdx.x * kRows + threadIdx.x / kCols, here = min(row, rows - 1);
    const uint32_t dv = 4 * (threadIdx.x % kCols), j = threadIdx.x % kWide;
    const uint32_t own = a.where[rows + here];
    if (__all(own & kDone)) return;
    Parts part[2];
#pragma unroll
    for (int y = 0; y < 2; y++) {
        const uint32_t at = y == 0 ? own : own & kCommon ? a.where[here] : 0, run = at & 511, rr = at >> 19 & 255;
        Parts &p = part[y];
        p.n = at >> 9 & 1023;
        if (p.n == 0) {
            p.o = a.whole + ((y == 0 ? rows : 0) + here) * (D + 4);
            p.m = p.o + D;
            p.sum = 1;
            p.lift = 0.0f;
            p.more = p.skip = 0;
            p.n = 1;
        } else {
            const bool second = at & kSecond;
            const uint32_t R = second ? R2 : R1;
            const size_t size = (size_t)R * (D + 2);
            const float *u = (second ? parts2 : a.parts) + (2 * (size_t)run + 1) * size;
            p.o = u + (size_t)rr * D;
            p.m = u + (size_t)R * D + rr;
            p.sum = R;
            p.lift = second ? lift2 : a.lift;
            p.more = size;          // (part 0 is the run's second slot, the others their runs' first)
            p.skip = 2 * size;
        }
        if (y == 1 && !(own & kCommon)) p.n = 0;
        if (own & kDone) p.n = 0;
    }
    auto at = [](const Parts &p, uint32_t i) { return i ? p.more + (i - 1) * p.skip : 0; };
    float top = -INFINITY;
#pragma unroll
    for (int y = 0; y < 2; y++)
        for (uint32_t i = j; i < part[y].n; i += kWide) top = fmaxf(top, part[y].m[at(part[y], i)] - part[y].lift);
#pragma unroll
    for (int o = 1; o < kWide; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    f4 x = {0, 0, 0, 0};
#pragma unroll
    for (int y = 0; y < 2; y++) {
        const Parts &p = part[y];
        // (the threads of a wave have rows of their own: the longest leads)
        for (uint32_t i0 = 0; __any(i0 < p.n); i0 += kWide) {
            float by = 0.0f, add = 0.0f;
            if (i0 + j < p.n) {
                const float *m = p.m + at(p, i0 + j);
                by = __builtin_amdgcn_exp2f(m[0] - p.lift - ref);
                add = by * m[p.sum];
            }
            const uint32_t m = i0 < p.n ? min(p.n - i0, (uint32_t)kWide) : 0;
            for (uint32_t i = 0; __any(i < m); i += kFar) {
                f4 v[kFar];
#pragma unroll
                for (int e = 0; e < kFar; e++) {
                    v[e] = f4{0, 0, 0, 0};
                    if (i + e < m) v[e] = *(const f4 *)(p.o + at(p, i0 + i + e) + dv);
                }
#pragma unroll
                for (int e = 0; e < kFar; e++) {
                    const float b = __shfl(by, (int)((threadIdx.x & 63 & ~(kWide - 1)) + ((i + e) & (kWide - 1))));
                    if (i + e < m) x += v[e] * b;
                }
            }
#pragma unroll
            for (int o = 1; o < kWide; o <<= 1) add += __shfl_xor(add, o);
            total += add;
        }
    }
    if (row >= rows || (own & kDone)) return;
    const uint32_t tok = (uint32_t)(row / heads), h = (uint32_t)(row - (size_t)tok * heads);
    const bool none = a.pos[tok] < 0;
    if (dv == 0 && a.lse) a.lse[row] = none ? -INFINITY : (top + log2f(total)) * (float)M_LN2;
    if (dv >= a.d) return;
    x *= none ? 0.0f : 1.0f / total;
    const size_t to = (size_t)tok * a.ld_out + (size_t)h * a.d + dv;
    if constexpr (sizeof(TO) == 4) *(f4 *)((float *)a.out + to) = x;
    else {
        typedef TO v4 __attribute__((ext_vector_type(4)));
        *(v4 *)((TO *)a.out + to) = v4{(TO)x[0], (TO)x[1], (TO)x[2], (TO)x[3]};
    }
}

} // namespace gs

namespace {

size_t up16(size_t x) { return (x + 15) & ~(size_t)15; }

// The workspace: jobs, positions, where the parts are, units that one run has
// whole, the two kernels' parts.
struct Place {
    size_t jobs, pos, where, whole, parts, parts2, all;
};

Place place(const gs_kv_cache *c, uint32_t n_heads, size_t n, size_t n_families, size_t n_tokens)
{
    const int D = padded(c->d);
    const size_t rows = n_tokens * n_heads;
    Place p;
    p.jobs = 0;
    p.pos = p.jobs + up16((n + n_families) * sizeof(gs::Job));
    p.where = p.pos + up16(n_tokens * 4);
    p.whole = p.where + up16(2 * rows * 4);
    p.parts = p.whole + up16(2 * rows * (D + 4) * 4);
    p.parts2 = p.parts + up16(few_bytes(D));
    p.all = p.parts2 + parts_bytes(gs::kChunkRuns, D == 256 ? gs::Chunk<256>::kRows : gs::Chunk<128>::kRows, D);
    return p;
}

template <class T, int D, int NT, bool F32> void rows_launch(gs::AttnArgs &a, hipStream_t st)
{
    a.n_wg = kCUs * gs::rows_per_cu(D, NT);
    a.lift = gs::kLift<T>;
    if (a.d == D) hipLaunchKernelGGL((gs::attn_rows_kernel<T, D, NT, F32, true, gs::kShared>), dim3(a.n_wg), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((gs::attn_rows_kernel<T, D, NT, F32, false, gs::kShared>), dim3(a.n_wg), dim3(256), 0, st, a);
}

template <class T, int D> void chunk_launch(gs::AttnArgs &a, hipStream_t st)
{
    a.n_wg = gs::kChunkRuns;
    a.lift = gs::kChunkLift<T>;
    const dim3 grid(a.n_wg), block(gs::Chunk<D>::kThreads);
    if (a.d == D) hipLaunchKernelGGL((gs::attn_chunk_kernel<T, D, true, gs::kShared>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((gs::attn_chunk_kernel<T, D, false, gs::kShared>), grid, block, 0, st, a);
}

template <class TO, int D, int R1, int R2> void join(const gs::AttnArgs &a, const gs::AttnArgs &b, hipStream_t st)
{
    const size_t rows = (size_t)a.n_tokens * a.n_kv * a.group, each = 256 / (D / 4);
    hipLaunchKernelGGL((gs::shared_join_kernel<TO, D, R1, R2>), dim3((unsigned)((rows + each - 1) / each)), dim3(256), 0, st, a, b.parts, b.lift);
}

// `own`, `family`: the most query rows per head of keys that a sequence, or a
// family, may have.  Jobs of few rows are the first kernel's, the others the
// second's.
template <class T, int D, int NT, bool F32> void few_and_many(gs::AttnArgs &a, gs::AttnArgs &b, uint64_t family, hipStream_t st)
{
    if constexpr (!F32)
        if (family > 16 * NT) {
            b.second = gs::kSecond;
            // Few sequences' own keys do not fill a launch of their own.  (us with two
            // kernels and with the second alone, heads of 128: one family of 8 rows
            // over 1000 tokens and up to 50 of their own, 8 heads of keys, 40.4, 29.5;
            // 4 of 8 over 2000, 43.3, 38.2; one of 64 over 4000, 56.5, 54.8; 8 of 32 over
            // 2000, 4 heads of keys, 86.6, 94.4.  Heads of 256, one of 16 over 8000, 62.4,
            // 48.2; 16 of 16 over 2000 and up to 1000, 288, 319.)
            if ((uint64_t)(a.n - a.n_families) * a.n_kv > gs::kChunkRuns) {
                a.max_rows = 16 * NT;
                b.min_rows = 16 * NT + 1;
                rows_launch<T, D, NT, F32>(a, st);
            }
            chunk_launch<T, D>(b, st);
            join<T, D, 16 * NT, gs::Chunk<D>::kRows>(a, b, st);
            return;
        }
    rows_launch<T, D, NT, F32>(a, st);
    join<std::conditional_t<F32, float, T>, D, 16 * NT, 16 * NT>(a, a, st);
}

template <class T, int D, bool F32> void by_rows(gs::AttnArgs &a, gs::AttnArgs &b, uint64_t own, uint64_t family, hipStream_t st)
{
    if constexpr (D == 256) few_and_many<T, D, 1, F32>(a, b, family, st);       // (two tiles of rows spill, or go to the second kernel)
    else if ((F32 ? family : own) <= 16) few_and_many<T, D, 1, F32>(a, b, family, st);
    else few_and_many<T, D, 2, F32>(a, b, family, st);
}

template <class T, bool F32> void by_head(gs::AttnArgs &a, gs::AttnArgs &b, uint64_t own, uint64_t family, hipStream_t st)
{
    switch (padded(a.d)) {
    case 64: return by_rows<T, 64, F32>(a, b, own, family, st);
    case 128: return by_rows<T, 128, F32>(a, b, own, family, st);
    default: return by_rows<T, 256, F32>(a, b, own, family, st);
    }
}

} // namespace

extern "C" {

size_t gs_attn_shared_workspace(const gs_kv_cache *c, uint32_t n_heads, uint32_t n, uint32_t n_families, uint32_t n_tokens)
{
    if (check_cache(c) || n_heads == 0 || n_heads % c->n_kv || n_heads > 65535) return 0;
    if (n > 65536 || n_families > 65536 || (uint64_t)n_tokens * (n_heads / c->n_kv) > 0x7fffffffull) return 0;
    return place(c, n_heads, n, n_families, n_tokens).all;
}

int gs_attn_shared(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const uint32_t *families, uint32_t n_families,
                   const gs_attn_args *x, float *lse, void *stream)
{
    if (int rc = check_attn(c, layer, b, x, lse)) return rc;
    if (n_families > 65536) return GS_ERR_UNSUPPORTED;
    if (b->n_tokens == 0) return GS_OK;
    if (!families || n_families == 0) return GS_ERR_INVALID;
    const size_t need = gs_attn_shared_workspace(c, x->n_heads, b->n, n_families, b->n_tokens);
    if (!need) return GS_ERR_UNSUPPORTED;
    if (!x->ws || ((uintptr_t)x->ws & 15u) || x->ws_bytes < need) return GS_ERR_INVALID;
    // (a grid's threads side by side, of the join)
    if ((uint64_t)b->n_tokens * x->n_heads * (padded(c->d) / 4) > 0xffffffffull - 256) return GS_ERR_UNSUPPORTED;
    gs::AttnArgs a = attn_args(c, layer, b, x, lse);
    const Place p = place(c, x->n_heads, b->n, n_families, b->n_tokens);
    char *ws = (char *)x->ws;
    a.n_families = n_families;
    a.where = (uint32_t *)(ws + p.where);
    a.whole = (float *)(ws + p.whole);
    a.parts = (float *)(ws + p.parts);
    hipStream_t st = (hipStream_t)stream;
    // (16 rows of tokens and heads for each thread to mark)
    const uint64_t marks = ((uint64_t)b->n_tokens * x->n_heads + 16 * gs::kPlan - 1) / (16 * gs::kPlan), most = marks < 256 ? marks : 256;
    hipLaunchKernelGGL(gs::shared_plan_kernel, dim3(n_families > most ? n_families : (unsigned)most), dim3(gs::kPlan), 0, st, a, families, b->n, (gs::Job *)(ws + p.jobs), (int32_t *)(ws + p.pos));
    a.jobs = (const gs::Job *)(ws + p.jobs);
    a.pos = (const int32_t *)(ws + p.pos);
    a.n = b->n + n_families;
    gs::AttnArgs a2 = a;
    a2.parts = (float *)(ws + p.parts2);
    const uint64_t own = (uint64_t)most_tokens(b, x) * a.group, family = (uint64_t)b->n_tokens * a.group;
    const bool f16 = c->type == GS_TYPE_F16;
    if (x->type == GS_TYPE_F32) f16 ? by_head<_Float16, true>(a, a2, own, family, st) : by_head<__bf16, true>(a, a2, own, family, st);
    else f16 ? by_head<_Float16, false>(a, a2, own, family, st) : by_head<__bf16, false>(a, a2, own, family, st);
    return hipGetLastError() == hipSuccess ? GS_OK : GS_ERR_HIP;
}

} // extern "C"
