// gs_attn.hpp -- the kernels of the attention of new tokens over the paged
// cache (include/gs_attn.h).
//
// The work of a call is cut the same way for every shape.  A unit is one head
// of keys and values of one sequence and up to R of its query rows (row r of a
// sequence is token r / G and head r % G of the G that share the keys); a unit
// has one tile per kTile keys that its rows see.  The tiles of all units, one
// after the other, are dealt to the workgroups in equal runs.  So a long row
// and a short one, many and few, cost what their keys cost; a unit that a
// run's end cuts leaves its parts (maximum, sum, weighted values) in the
// workspace, and a second kernel joins them in order.
//
// Each run goes through its keys once, with the running maximum and sum of the
// softmax; the weights do not leave the registers.
//
// Families of rows that begin with the same pages (SHARED): the work is jobs,
// where a sequence is one or two of them: the keys that its family has in
// common, whose job takes the queries of all of the family's sequences beside
// one another, and its own keys.  The parts of both meet in gs_shared.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <cmath>
#include <type_traits>

#include "../../include/gs_attn.h"
#include "gs_cache.hpp"

namespace gs {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

struct AttnArgs {
    const char *k, *v;              // the layer's pages
    const void *q;
    void *out;
    size_t ld_q, ld_out;
    const uint32_t *table, *len, *rows, *start;
    uint32_t n, n_tokens, n_rows, n_pages, ld_table, n_kv, group, d;
    int shift;                      // log2 of the page size
    float scale;                    // of the scores, times log2(e)
    uint32_t window;                // (0xffffffff: none)
    uint32_t n_wg;                  // runs, at most
    uint32_t min_rows, max_rows;    // sequences with fewer or more query rows per head of keys are not this kernel's
    float *parts;                   // [2 n_wg][R][D + 2]: a run's cut units: the one it begins with, the one it ends with
    struct Cut *cuts;               // [n_wg]
    float *lse;                     // [n_tokens][n_kv group] logarithms of the softmax's sums, or null
    float lift;                     // log2 of what the kernel's sums are multiplied by
    // SHARED: `n` jobs, the first n_families of them of common keys
    const struct Job *jobs;
    const int32_t *pos;             // [n_tokens] positions
    uint32_t n_families;
    uint32_t *where;                // [2][n_tokens][heads] where the parts of a row's jobs are (common keys, its own)
    float *whole;                   // [2][n_tokens][heads][D + 4] units that one run has whole
    uint32_t second;                // 0 or kSecond: whose parts they are, of two kernels of a call
};

// What a call wants of the kernels below: gs_attn's result, the softmax's sums
// too, or either for families.
enum Kind { kPlain, kSums, kShared };

// A row of `where`: the unit's first run (9 bits), its parts (10 bits; 0: in
// `whole`), the row's place in the unit (8 bits), and these.
constexpr uint32_t kSecond = 1u << 27;      // parts of the call's second kernel
constexpr uint32_t kCommon = 1u << 28;      // its own keys' job: the row has common keys too
constexpr uint32_t kDone = 1u << 29;        // the result is written

// A unit that a run begins and does not end.
struct Cut {
    uint32_t last;                  // the run that ends it; 0: none
    uint32_t first_token, row0, rows, kvh;
    uint32_t keyless;               // rows before this one see no key
};

// One sequence of the call.
struct Seq {
    uint32_t row, len, first, nq;
    static constexpr uint32_t k0 = 0;
    __device__ __forceinline__ bool family() const { return false; }
};

// A job of a call with families: sequence (or family of sequences) with the
// keys [k0, k1).
struct Job {
    uint32_t row, len, first, nq;   // len kFamily: the family's queries, tokens first .. first + nq - 1
    uint32_t k0, k1;
    int32_t p0, p1;                 // a family: its tokens' lowest and highest position
    __device__ __forceinline__ bool family() const;
};
constexpr uint32_t kFamily = 0xffffffffu;
__device__ __forceinline__ bool Job::family() const { return len == kFamily; }

template <class S> __device__ __forceinline__ S work_of(const AttnArgs &a, uint32_t i);

template <> __device__ __forceinline__ Job work_of<Job>(const AttnArgs &a, uint32_t i)
{
    Job s = a.jobs[i];
    // (held to the call's tokens and the table, whatever the families were)
    s.first = min(s.first, a.n_tokens);
    s.nq = min(s.nq, a.n_tokens - s.first);
    if (s.nq * a.group < a.min_rows || s.nq * a.group > a.max_rows) s.nq = 0;
    s.k1 = min(s.k1, a.ld_table << a.shift);
    return s;
}

template <> __device__ __forceinline__ Seq work_of<Seq>(const AttnArgs &a, uint32_t i)
{
    Seq s;
    s.first = a.start ? min(a.start[i], a.n_tokens) : i;
    const uint32_t end = a.start ? min(a.start[i + 1], a.n_tokens) : i + 1;
    s.nq = end > s.first ? end - s.first : 0;
    if (s.nq * a.group < a.min_rows || s.nq * a.group > a.max_rows) s.nq = 0;
    s.row = a.rows ? a.rows[i] : i;
    s.len = s.row < a.n_rows ? min(a.len[s.row], a.ld_table << a.shift) : 0;
    return s;
}

// The same value in a scalar register, where all lanes have it.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uniform(uint64_t x)
{
    return (uint64_t)uniform((uint32_t)(x >> 32)) << 32 | uniform((uint32_t)x);
}
__device__ __forceinline__ Seq uniform(const Seq &s) { return Seq{uniform(s.row), uniform(s.len), uniform(s.first), uniform(s.nq)}; }
__device__ __forceinline__ Job uniform(const Job &s)
{
    return Job{uniform(s.row), uniform(s.len), uniform(s.first), uniform(s.nq), uniform(s.k0), uniform(s.k1),
               (int32_t)uniform((uint32_t)s.p0), (int32_t)uniform((uint32_t)s.p1)};
}

// The keys that rows r0 .. r1 - 1 of a sequence see, [lo, hi), and the first
// tile; `tiles` is at least 1, so that rows without keys are written too.
template <int kTile> struct Span {
    uint32_t lo, hi, tile0, tiles;
    uint32_t key0;                  // of tile 0 (SHARED: the first key of the job, at a page's begin)
    __device__ __forceinline__ Span(const AttnArgs &a, const Seq &s, uint32_t r0, uint32_t r1)
    {
        const int64_t p0 = (int64_t)s.len - s.nq + r0 / a.group, p1 = (int64_t)s.len - s.nq + (r1 - 1) / a.group;
        hi = (uint32_t)max((int64_t)0, p1 + 1);
        lo = (uint32_t)max((int64_t)0, p0 + 1 - (int64_t)a.window);
        key0 = 0;
        tile0 = lo / kTile;
        tiles = hi > lo ? (hi + kTile - 1) / kTile - tile0 : 1;
    }
    __device__ __forceinline__ Span(const AttnArgs &a, const Job &s, uint32_t r0, uint32_t r1)
    {
        const int64_t base = (int64_t)s.len - s.nq;
        const int64_t p0 = s.family() ? s.p0 : base + r0 / a.group, p1 = s.family() ? s.p1 : base + (r1 - 1) / a.group;
        hi = (uint32_t)min(max((int64_t)0, p1 + 1), (int64_t)s.k1);
        lo = (uint32_t)max((int64_t)s.k0, p0 + 1 - (int64_t)a.window);
        key0 = s.k0;
        tile0 = (lo - key0) / kTile;
        tiles = hi > lo ? (hi - key0 + kTile - 1) / kTile - tile0 : 1;
    }
};

// a / b, by 32-bit division where that is enough (as it is for any call that
// fits the memory; 64 bits are several times as many instructions).
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b)
{
    return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b;
}

// How a kernel deals its work: R rows in a unit, kTile keys in a tile, and a
// unit's beginning and end (its queries, the first keys' way, its rows' way
// out), which are dealt as kSetup tiles before its first.  (us with 0, as it
// is, twice as many: 16 prompts of 512, 28 / 4 heads of 128, kSetup 0, 3, 6:
// 111, 92, 87; one of 2000, 32 / 8 heads, 3 and 6: 80, 84; 64 single tokens
// over 1500, kSetup 0, 1, 2: 39.5, 39.2, 41.4.)
// Where kBase is given, a tile is dealt as kBase pieces and one for each kM rows
// that a wave has of it; a tile is the run's that its first piece is in.
template <int R_, int kTile_, int kSetup_, class S, int kBase = 0, int kM = 1> struct Deal {
    static constexpr int R = R_, kTile = kTile_, kSetup = kSetup_;
    using Work = S;
    static __device__ __forceinline__ uint32_t weight(uint32_t r0, uint32_t r1) { return kBase ? kBase + (r1 - r0 + kM - 1) / kM : 1; }
    // The first tile of a unit whose pieces begin at or after `piece` of its beginning.
    static __device__ __forceinline__ uint32_t tile_at(uint64_t piece, uint32_t weight)
    {
        if constexpr (kBase == 0) return max((uint32_t)piece, (uint32_t)kSetup) - kSetup;
        return max((uint32_t)quotient(piece + weight - 1, weight), (uint32_t)kSetup) - kSetup;
    }
    static __device__ __forceinline__ uint32_t heads(const AttnArgs &a) { return a.n_kv; }
    // Tiles of the unit of rows r ..
    static __device__ __forceinline__ uint32_t unit(const AttnArgs &a, const S &s, uint32_t r)
    {
        const uint32_t r1 = min(r + R, s.nq * a.group);
        return (Span<kTile>(a, s, r, r1).tiles + kSetup) * weight(r, r1);       // (below 2^32: tiles of 32 keys, positions below 2^30)
    }
    // Tiles of a sequence and one head of keys (a chunk of 66000 tokens over 2^23
    // has more than 2^32 of 16 rows), counted by a thread ..
    static __device__ __forceinline__ uint64_t count(const AttnArgs &a, const S &s)
    {
        uint64_t t = 0;
        for (uint32_t r = 0; r < s.nq * a.group; r += R) t += unit(a, s, r);
        return t;
    }
    // .. and by a wave, its lanes side by side
    static __device__ __forceinline__ uint64_t count_wave(const AttnArgs &a, const S &s)
    {
        uint64_t t = 0;
        for (uint32_t r = (threadIdx.x & 63) * R; r < s.nq * a.group; r += 64 * R) t += unit(a, s, r);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) t += __shfl_xor(t, o);
        return t;
    }
    // The first row of the unit that tile `skip` of the sequence is in; skip
    // becomes the tile's number in the unit.  (a wave)
    static __device__ __forceinline__ uint32_t find(const AttnArgs &a, const S &s, uint64_t &skip)
    {
        using Sum = std::conditional_t<kBase == 0, uint32_t, uint64_t>;       // (of 64 units)
        const uint32_t rows = s.nq * a.group, lane = threadIdx.x & 63;
        if (rows <= R) return 0;
        for (uint32_t r = 0;; r += 64 * R) {
            const uint32_t mine = r + lane * R < rows ? unit(a, s, r + lane * R) : 0;
            Sum sum = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const Sum y = __shfl_up(sum, o);
                if (lane >= o) sum += y;
            }
            const uint64_t past = __ballot(sum > skip);
            if (past) {
                const int at = __ffsll((unsigned long long)past) - 1;
                skip -= uniform((Sum)__shfl((Sum)(sum - mine), at));
                return r + at * R;
            }
            skip -= uniform((Sum)__shfl(sum, 63));
        }
    }
};

// The run of this workgroup: its tiles [t0, t1) of `total`, the sequence the
// first of them is in, and how many tiles of that sequence come before it.
// Run g has total / n_wg tiles, the first total % n_wg runs one more.
// Each thread counts a stretch of the sequences, and the one that finds the
// run's first leaves it in LDS.
template <class S> struct Run {
    uint64_t t0, t1, total, skip, per;  // per: tiles of the sequence and one head of keys
    uint32_t n_wg, seq;
    S s;
};

// The run that tile x is in.
template <class S> __device__ __forceinline__ uint32_t run_with(const Run<S> &r, uint64_t x)
{
    const uint64_t q = quotient(r.total, r.n_wg), more = r.total - q * r.n_wg;
    return (uint32_t)(x < more * (q + 1) ? quotient(x, q + 1) : more + quotient(x - more * (q + 1), q));
}

// kLeast: tiles that a run has at least, if there are as many: a shorter one
// costs more to join than it saves.  (The chunk kernel, us with 4, 3, 2: 50
// tokens over 4000, 32 / 8 heads of 128: 33.1, 32.7, 38.0; 300 over 300: 27.3,
// 24.7, 24.7.)
template <class D, int kThreads, int kLeast, class A> __device__ __forceinline__ Run<typename D::Work> run_of(const A &a, uint32_t g)
{
    using S = typename D::Work;
    constexpr uint32_t kWaves = kThreads / 64, kShort = 32;     // up to kShort sequences are counted by waves: theirs may be long
    __shared__ uint64_t s_wave[kWaves];
    __shared__ uint64_t s_per[kShort];
    __shared__ S s_seq[kShort];
    __shared__ Run<S> s_run;
    const uint32_t each = (a.n + kThreads - 1) / kThreads;
    const uint32_t i0 = min(threadIdx.x * each, a.n), i1 = min(i0 + each, a.n);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    S s = {};
    uint64_t per = 0, mine = 0;
    if (a.n <= kShort) {
        for (uint32_t i = w; i < a.n; i += kWaves) {
            s = work_of<S>(a, i);
            per = D::count_wave(a, s);
            if (lane == 0) { s_per[i] = per; s_seq[i] = s; }
        }
        __syncthreads();
        if (threadIdx.x < a.n) {
            s = s_seq[threadIdx.x];
            per = s_per[threadIdx.x];
            mine = per * D::heads(a);
        }
    } else {
        for (uint32_t i = i0; i < i1; i++) {
            s = work_of<S>(a, i);
            per = D::count(a, s);
            mine += per * D::heads(a);
        }
    }
    uint64_t x = mine;
    if (a.n > each) {                       // (one sequence: the first thread has it)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
    }
    if (lane == (a.n > each ? 63 : 0)) s_wave[w] = x;
    __syncthreads();
    uint64_t before = x - mine;
    Run<S> r;
    r.total = 0;
#pragma unroll
    for (int i = 0; i < (int)kWaves; i++) {
        if (i < w) before += s_wave[i];
        r.total += s_wave[i];
    }
    const uint64_t most = quotient(r.total + kLeast - 1, kLeast);
    r.n_wg = (uint32_t)min((uint64_t)a.n_wg, most);
    if (g >= uniform(r.n_wg)) { r.t0 = r.t1 = 0; return r; }
    const uint64_t q = quotient(r.total, r.n_wg), more = r.total - q * r.n_wg;
    r.t0 = g * q + min((uint64_t)g, more);
    r.t1 = r.t0 + q + (g < more);
    if (mine && r.t0 >= before && r.t0 < before + mine) {
        uint32_t i = i0;
        if (each > 1)
            for (;; i++) {
                s = work_of<S>(a, i);
                per = D::count(a, s);
                if (r.t0 < before + per * D::heads(a)) break;
                before += per * D::heads(a);
            }
        r.seq = i; r.skip = r.t0 - before; r.per = per; r.s = s;
        s_run = r;
    }
    __syncthreads();
    const Run<S> u = s_run;
    return Run<S>{uniform(u.t0), uniform(u.t1), uniform(u.total), uniform(u.skip), uniform(u.per), uniform(u.n_wg), uniform(u.seq), uniform(u.s)};
}

// The logarithm of a softmax's sum, of the scores as they came in: `total` is
// the sum of 2^(score - top), lifted.
__device__ __forceinline__ float log_sum(const AttnArgs &a, bool none, float top, float total)
{
    return none ? -INFINITY : (top - a.lift + log2f(total)) * (float)M_LN2;
}

// A maximum as parts of kernels of unlike lifts are joined by.
__device__ __forceinline__ float lifted(const AttnArgs &a, float top) { return top - a.lift; }

// An infinity or NaN among 8 values.
template <class T> __device__ __forceinline__ bool not_finite(u4v x)
{
    constexpr uint32_t e = sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; i++) bad |= (x[i] & e) == e || (x[i] >> 16 & e) == e;
    return bad;
}

// Bits 15 and 31 say the same of the words x of two values each (a half's largest
// exponent and one carry into its sign's place, no further).
template <class T> __device__ __forceinline__ uint32_t exponents(uint32_t x)
{
    return (x & 0x7fff7fffu) + (__is_same(T, _Float16) ? 0x04000400u : 0x00800080u);
}

template <class T> struct Vec;
template <> struct Vec<_Float16> { typedef h8 v8; };
template <> struct Vec<__bf16> { typedef b8 v8; };

// Weights are held times 2^15 where the type's smallest numbers are near: f16
// weights of 2^-15 of the largest would lose bits below 2^-14.
template <class T> constexpr float kLift = __is_same(T, _Float16) ? 15.0f : 0.0f;
template <class T> constexpr float kChunkLift = __is_same(T, _Float16) ? 7.0f : 0.0f;      // (the second kernel's, see there)
// SHARED: the parts in which a weight reaches the values, of 16-bit queries: off
// by 2^-22 (bf16: 2^-24) of it, so that a row's result is that of 32-bit weights,
// rounded once, whichever of its keys are in common.  (us with one part and so: one
// family of 64 rows over 16000, bf16, 63, 82 (two parts: 73); 16 of 16 over 700 to
// 8192, f16, 187, 194; 32 rows of 8 tokens over 30001, heads of 256, bf16, 155, 198.
// Results that are not the exact one's nearest, of these bf16, f16 and bf16:
// 1e-4, 9e-4 and 1e-4 of all; of 32-bit torch operations 2e-4, 2e-3 and 5e-4.)
template <class T> constexpr int kSharedParts = __is_same(T, _Float16) ? 2 : 3;

constexpr int kRowTile = 128;           // keys of a tile: 32 for each wave

// Workgroups of the kernel below that a CU takes at a time, by their
// registers, and so the runs that its work is dealt to: with twice as many the
// second half begins when the first is done (us with 512 and 256 runs: 20
// single tokens over 700 to 8192, 16 / 8 heads of 256, 88, 80; 16 sequences of
// 8 over 500 to 4000, 32 / 8 heads of 128, 46, 35, and of 64, where two fit, 26,
// 28).
constexpr int rows_per_cu(int D, int NT) { return D == 64 || (D == 128 && NT == 1) ? 2 : 1; }

// Up to 16 NT query rows against the keys, for single tokens and few of them:
// what bounds it is the read of K and V, so each wave reads its 32 keys of a
// tile straight to registers, once, K for the next tile while it works on
// this tile's V and the other way round.  The products are S^T = K Q^T and
// O^T = V^T P^T, 16 x 16 x 32: a lane then holds the weights of one query row
// (lane & 15) for exactly the 8 keys that it has to give to the second
// product, if row m of the two K tiles is key 8 (m / 4) + 4 t + m % 4.  V^T's
// columns come from the 8 rows of V in a lane by a transposition of 8 x 8
// values in registers (the value a lane's row m stands for is 8 m + i in
// product i).  Four waves' sums meet in LDS at a unit's end.
// The second product's factors are of T.  With up to 16 rows a bf16 weight goes in
// as two of them, its rounding and the rest, 16 bits together: one product more,
// where the matrix cores have the time.  Others are rounded once, off by 2^-11 of
// themselves (bf16: 2^-8) at most and without a common direction, a quarter of
// what the rounding of the result adds.  (us with one and two: 64 single tokens
// over 1000 to 32768, bf16, 206, 206, the outputs' relative distance to 32-bit
// weights' 6.8e-4, 4e-5; 64 sequences of 8 over 8000, 32 rows of 32 / 8 heads of
// 128, bf16 390, 419; of 64, f16 184, 194.)  Their sum is of the unrounded ones,
// in f32.
// Measured: 64 rows of 16000 tokens, 28 / 4 heads of 128, bf16: 357 us, 5.9
// TB/s, what a read of this size reaches; one token over 4001, f32: 9.7 us of
// kernel, most of them the search for the run's begin and three waits in a row
// for memory (table, keys, values).
// F32: q in three parts of T whose sum is q (scaled by a power of two into
// f16's range), and the weights too, so the products keep 24 bits.
// FULL: heads of just D values (their strides are then constants, which takes
// fewer registers and instructions).
template <class T, int D, int NT, bool F32, bool FULL, Kind KIND>
__global__ void __launch_bounds__(256, rows_per_cu(D, NT)) attn_rows_kernel(const AttnArgs a)
{
    constexpr bool SHARED = KIND == kShared;
    constexpr int R = 16 * NT, NP = F32 ? 3 : 1, NW = F32 ? 3 : SHARED ? kSharedParts<T> : __is_same(T, __bf16) && NT == 1 ? 2 : 1, KS = D / 32;
    constexpr int CW = D >= 128 ? 8 : D / 16, NC = D / (16 * CW);       // values of a lane's V chunk, chunks
    typedef typename Vec<T>::v8 v8;
    typedef T vw __attribute__((ext_vector_type(CW)));
    __shared__ float s_o[4][16][D + 4];
    __shared__ float s_m[4][16], s_l[4][16];

    using S = std::conditional_t<SHARED, Job, Seq>;
    using Dealt = Deal<R, kRowTile, 1, S>;
    Run<S> run = run_of<Dealt, 256, 1>(a, blockIdx.x);
    if (!SHARED && threadIdx.x == 0 && blockIdx.x < a.n_wg) a.cuts[blockIdx.x].last = 0;
    if (run.t0 >= run.t1) return;

    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t page = 1u << a.shift;
    const uint32_t d = FULL ? D : a.d;
    const size_t head = (size_t)d << a.shift;           // values of a head's page

    uint32_t si = run.seq, r0;
    S s = run.s;
    uint64_t t = run.t0;
    uint32_t kvh = (uint32_t)quotient(run.skip, run.per);
    uint64_t before = run.skip - kvh * run.per;
    r0 = Dealt::find(a, s, before);
    uint32_t skip = (uint32_t)before;
    while (t < run.t1) {
        const uint32_t rows = s.nq * a.group;
        if (kvh == a.n_kv || rows == 0) {               // the next sequence
            s = uniform(work_of<S>(a, ++si));
            kvh = 0; r0 = 0;
            continue;
        }
        const uint32_t r1 = min(r0 + R, rows);
        const Span<kRowTile> span(a, s, r0, r1);
        // the run's part of the unit, tiles first .. first + left - 1
        const uint32_t dealt = span.tiles + Dealt::kSetup, part_of = (uint32_t)min((uint64_t)(dealt - skip), run.t1 - t);
        const uint32_t first = max(skip, (uint32_t)Dealt::kSetup) - Dealt::kSetup;
        const uint32_t left = max(skip + part_of, (uint32_t)Dealt::kSetup) - Dealt::kSetup - first;
        if (left == 0) break;                           // (its setup only: the next run begins it)
        const uint64_t end = t - skip + dealt;

        // ---- the keys.  Lane's K rows are in the page of key0 + 8 (m / 4), its V
        // rows in that of key0 + 8 g; the pages' numbers are read a tile ahead
        // of the rows (ahead of K, which is waited for before they are used).
        const uint32_t *table = a.table + (size_t)min(s.row, a.n_rows - 1) * a.ld_table;
        const uint32_t last = span.hi > 0 ? span.hi - 1 : 0;
        auto page_of = [&](uint32_t key) { return table[min(key, last) >> a.shift]; };     // (the key is held to the unit's)
        auto place = [&](uint32_t id) { return ((size_t)min(id, a.n_pages - 1) * a.n_kv + kvh) * head; };
        v8 kf[2][KS];
        vw vf[8][NC];
        auto load_k = [&](uint32_t key0, uint32_t id) {
            const T *p = (const T *)a.k + place(id);
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const T *row = p + (size_t)((key0 + 8 * (m >> 2) + 4 * x + (m & 3)) & (page - 1)) * d;
#pragma unroll
                for (int c = 0; c < KS; c++) {
                    v8 y = {};
                    if (32 * c + 8 * g < d) y = *(const v8 *)(row + 32 * c + 8 * g);
                    kf[x][c] = y;
                }
            }
        };
        auto load_v = [&](uint32_t key0, uint32_t id) {
            const T *p = (const T *)a.v + place(id);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const T *row = p + (size_t)((key0 + 8 * g + j) & (page - 1)) * d;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    vw y = {};
                    if (16 * CW * c + CW * m < d) y = *(const vw *)(row + 16 * CW * c + CW * m);
                    vf[j][c] = y;
                }
            }
        };
        uint32_t key0 = span.key0 + (span.tile0 + first) * kRowTile + 32 * w;
        uint32_t kid = page_of(key0 + 8 * (m >> 2)), vid = page_of(key0 + 8 * g);
        uint32_t kid1 = page_of(key0 + kRowTile + 8 * (m >> 2)), vid1 = page_of(key0 + kRowTile + 8 * g);
        load_k(key0, kid);
        load_v(key0, vid);

        // ---- queries: row r0 + 16 nt + m, values 32 s + 8 g .. + 7
        v8 qf[NT][NP][KS];
        float unscale[NT];
        int64_t pos[NT];
        // SHARED: a row's keys are from[nt] .. pos[nt], held to the job's
        int32_t from[NT];
        auto keys_of = [&](uint32_t tok, int64_t &p, int32_t &f) {
            if constexpr (SHARED) {
                const int64_t at = s.family() ? (a.window == 0xffffffffu ? (int64_t)s.p0 : (int64_t)a.pos[s.first + tok]) : (int64_t)s.len - s.nq + tok;
                f = (int32_t)max((int64_t)s.k0, at + 1 - (int64_t)a.window);
                p = min(at, (int64_t)s.k1 - 1);
            } else {
                p = (int64_t)s.len - s.nq + tok;
                f = 0;
            }
        };
        auto sees = [&](int64_t key, int64_t p, int32_t f) { return SHARED ? key <= p && key >= f : key <= p && key > p - (int64_t)a.window; };
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const uint32_t r = min(r0 + 16 * nt + m, r1 - 1);
            const uint32_t tok = r / a.group, h = kvh * a.group + (r - tok * a.group);
            keys_of(tok, pos[nt], from[nt]);
            const size_t at = (size_t)(s.first + tok) * a.ld_q + (size_t)h * d;
            unscale[nt] = a.scale;
            if constexpr (F32) {
                float x[KS][8], top = 0.0f;
#pragma unroll
                for (int c = 0; c < KS; c++) {
                    if (32 * c + 8 * g < d) load8((const float *)a.q + at + 32 * c + 8 * g, x[c]);
                    else
#pragma unroll
                        for (int e = 0; e < 8; e++) x[c][e] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[c][e]));
                }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                int ex = 0;
                if (__is_same(T, _Float16) && top > 0.0f && top < INFINITY) ex = 14 - ilogbf(top);
                unscale[nt] *= ldexpf(1.0f, -ex);       // (0 for rows below 2^-135: their scores are 0)
#pragma unroll
                for (int c = 0; c < KS; c++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float y = ldexpf(x[c][e], ex);
                        const T p0 = (T)y;
                        const float y1 = y - (float)p0;
                        const T p1 = (T)y1;
                        qf[nt][0][c][e] = p0;
                        qf[nt][1][c][e] = p1;
                        qf[nt][2][c][e] = (T)(y1 - (float)p1);
                    }
            } else {
#pragma unroll
                for (int c = 0; c < KS; c++) {
                    v8 x = {};
                    if (32 * c + 8 * g < d) x = *(const v8 *)((const T *)a.q + at + 32 * c + 8 * g);
                    qf[nt][0][c] = x;
                }
            }
        }

        f4 o[NT][NC][CW];
        float mx[NT], sum[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            mx[nt] = -INFINITY;
            sum[nt] = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < CW; i++) o[nt][c][i] = f4{0, 0, 0, 0};
        }
        // keys that every row of the unit sees: those below all_hi, from all_lo on
        uint32_t all_hi;
        int64_t all_lo;
        if constexpr (SHARED) {
            all_hi = s.family() ? s.k1 : (uint32_t)max((int64_t)0, (int64_t)s.len - s.nq + r0 / a.group + 1);
            all_lo = (s.family() ? (int64_t)s.p1 : (int64_t)s.len - s.nq + (r1 - 1) / a.group) + 1 - (int64_t)a.window;
        } else {
            all_hi = (uint32_t)max((int64_t)0, (int64_t)s.len - s.nq + r0 / a.group + 1);
            all_lo = (int64_t)s.len - s.nq + (r1 - 1) / a.group + 1 - (int64_t)a.window;
        }
        for (uint32_t x = 0; x < left; x++, key0 += kRowTile) {
            // rows that see a part of the 32 keys only
            const bool edge = key0 + 32 > all_hi || (int64_t)key0 < all_lo;
            f4 sc[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    f4 z = {0, 0, 0, 0};
#pragma unroll
                    for (int q = NP - 1; q >= 0; q--)           // (the small parts first)
#pragma unroll
                        for (int c = 0; c < KS; c++) z = mfma(kf[y][c], qf[nt][q][c], z);
                    sc[nt][y] = z;
                }
            const bool more = x + 1 < left;
            if (more) {
                kid = kid1; vid = vid1;
                kid1 = page_of(key0 + 2 * kRowTile + 8 * (m >> 2));
                vid1 = page_of(key0 + 2 * kRowTile + 8 * g);
                load_k(key0 + kRowTile, kid);
            }

            float p[NT][8];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[nt][j] = sc[nt][j >> 2][j & 3] * unscale[nt];
                    if (edge) {
                        const int64_t key = (int64_t)key0 + 8 * g + j;
                        if (!sees(key, pos[nt], from[nt])) p[nt][j] = -INFINITY;
                    }
                    top = fmaxf(top, p[nt][j]);
                }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                top = fmaxf(top, mx[nt]);
                const float ref = top == -INFINITY ? 0.0f : top;
                const float by = __builtin_amdgcn_exp2f(mx[nt] - ref);
                mx[nt] = top;
                float add = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[nt][j] = __builtin_amdgcn_exp2f(p[nt][j] - ref + kLift<T>);
                    add += p[nt][j];
                }
                sum[nt] = sum[nt] * by + add;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int i = 0; i < CW; i++) o[nt][c][i] *= by;
            }

            // Values of keys that no row sees are zeros.  An infinity or a NaN of a
            // key that only some rows see would reach the others as 0 * NaN: such
            // keys (bit 8 g + j of `bad`) are left out of the product and come one
            // by one after it, to the rows that see them.
            uint32_t bad = 0;
            if (edge) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t key = key0 + 8 * g + j;
                    const bool out = key >= span.hi || key < span.lo;
                    bool inf = false;
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        if (out) vf[j][c] = vw{};
                        u4v raw = {};
                        __builtin_memcpy(&raw, &vf[j][c], sizeof(vw));
                        inf |= not_finite<T>(raw);
                    }
                    const uint64_t b = __ballot(inf);
#pragma unroll
                    for (int y = 0; y < 4; y++)
                        if (b >> (16 * y) & 0xffff) bad |= 1u << (8 * y + j);
                    if (bad >> (8 * g + j) & 1)
#pragma unroll
                        for (int c = 0; c < NC; c++) vf[j][c] = vw{};
                }
            }
            v8 pf[NT][NW];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    pf[nt][0][j] = (T)p[nt][j];
                    const float y = p[nt][j] - (float)pf[nt][0][j];
                    if constexpr (NW > 1) pf[nt][1][j] = (T)y;
                    if constexpr (NW > 2) pf[nt][2][j] = (T)(y - (float)pf[nt][1][j]);
                }
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < CW; i++) {
                    v8 x8;
#pragma unroll
                    for (int j = 0; j < 8; j++) x8[j] = vf[j][c][i];
#pragma unroll
                    for (int q = NW - 1; q >= 0; q--)           // (neighbours do not wait for one another)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) o[nt][c][i] = mfma(x8, pf[nt][q], o[nt][c][i]);
                }
            for (; bad; bad &= bad - 1) {
                const uint32_t y = __ffs(bad) - 1;
                const int64_t key = (int64_t)key0 + y;
                const T *row = (const T *)a.v + place(page_of(key0 + y)) + (size_t)((key0 + y) & (page - 1)) * d;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float wt = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (j == (int)(y & 7)) wt = p[nt][j];
                    wt = __shfl(wt, (y >> 3) * 16 + m);         // (the lane that has the key)
                    if (!sees(key, pos[nt], from[nt])) continue;
#pragma unroll
                    for (int c = 0; c < NC; c++)
#pragma unroll
                        for (int i = 0; i < CW; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const uint32_t dv = 16 * CW * c + CW * (4 * g + e) + i;
                                if (dv < d) o[nt][c][i][e] += wt * (float)row[dv];
                            }
                }
            }
            if (more) load_v(key0 + kRowTile, vid);
        }

        // Row r over the wave's keys by the vector units, from the unsplit query
        // and weights, with 64 lanes beside one another along the head; to s_m,
        // s_l and s_o as the products leave them.  A row whose query is not
        // finite, or that has met a NaN, is NaN and costs no more than that.
        auto alone = [&](uint32_t r) {
            constexpr int E = D / 64;
            const uint32_t tok = r / a.group, h = kvh * a.group + (r - tok * a.group), rr = (r - r0) & 15;
            int64_t at;
            int32_t from1;
            keys_of(tok, at, from1);
            const size_t qa = (size_t)(s.first + tok) * a.ld_q + (size_t)h * d;
            float q[E], y[E], top = -INFINITY, l = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const uint32_t dv = 64 * e + lane;
                y[e] = 0.0f;
                q[e] = 0.0f;
                if (dv < d) q[e] = F32 ? ((const float *)a.q)[qa + dv] : (float)((const T *)a.q)[qa + dv];
                l = fmaf(q[e], 0.0f, l);
            }
            if (__any(!(l == 0.0f))) return;
            for (uint32_t x = 0; x < 32 * left && l == l; x++) {
                const uint32_t key = span.key0 + (span.tile0 + first + x / 32) * kRowTile + 32 * w + x % 32;
                if (!sees(key, at, from1)) continue;
                const size_t from = place(page_of(key)) + (size_t)(key & (page - 1)) * d;
                float dot = 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (64 * e + lane < d) dot += q[e] * (float)((const T *)a.k)[from + 64 * e + lane];
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) dot += __shfl_xor(dot, o);
                dot *= a.scale;
                const float up = fmaxf(top, dot), ref = up == -INFINITY ? 0.0f : up, by = __builtin_amdgcn_exp2f(top - ref);
                const float wt = __builtin_amdgcn_exp2f(dot - ref + kLift<T>);
                top = up;
                l = l * by + wt;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    y[e] *= by;
                    if (64 * e + lane < d) y[e] += wt * (float)((const T *)a.v)[from + 64 * e + lane];
                }
            }
            if (lane == 0) { s_m[w][rr] = top; s_l[w][rr] = l; }
#pragma unroll
            for (int e = 0; e < E; e++) s_o[w][rr][64 * e + lane] = y[e];
        };

        // ---- the waves' sums together; the unit's rows or its part
        const bool whole = left == span.tiles;
        const uint32_t heads = a.n_kv * a.group;
        // SHARED: rows that have keys in common with others have two jobs
        const uint32_t common = SHARED && !s.family() && s.k0 ? kCommon : 0;
        const bool here = !SHARED || (!s.family() && !common);
        float *part = a.parts + (size_t)(2 * blockIdx.x + (first == 0)) * R * (D + 2);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float l = sum[nt];
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);
            // A sum that is no finite number may be so by an infinity that met the
            // parts of a query or a weight (inf - inf, 0 inf) where the formula
            // has -inf or inf: such rows are computed again without parts.
            float off = l * 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < CW; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) off = fmaf(o[nt][c][i][e], 0.0f, off);
            uint64_t again = __ballot(!(off == 0.0f));
            again = (again | again >> 32);
            again = (again | again >> 16) & 0xffff;
            __syncthreads();
            if (g == 0) { s_m[w][m] = mx[nt]; s_l[w][m] = l; }
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int i = 0; i < CW; i += 4)
                        *(f4 *)&s_o[w][m][16 * CW * c + CW * (4 * g + e) + i] =
                            f4{o[nt][c][i][e], o[nt][c][i + 1][e], o[nt][c][i + 2][e], o[nt][c][i + 3][e]};
            for (; __builtin_expect(again != 0, 0); again &= again - 1) {
                const uint32_t r = r0 + 16 * nt + __ffsll((unsigned long long)again) - 1;
                if (r < r1) alone(r);
            }
            __syncthreads();
            const uint32_t rr = threadIdx.x >> 4, r = r0 + 16 * nt + rr, c0 = threadIdx.x & 15;
            if (r >= r1) continue;
            float top = fmaxf(fmaxf(s_m[0][rr], s_m[1][rr]), fmaxf(s_m[2][rr], s_m[3][rr])), total = 0.0f, by[4];
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int y = 0; y < 4; y++) {
                by[y] = __builtin_amdgcn_exp2f(s_m[y][rr] - ref);
                total += by[y] * s_l[y][rr];
            }
            const uint32_t tok = r / a.group, h = kvh * a.group + r - tok * a.group;
            const bool none = SHARED && s.family() ? false : (int64_t)s.len - s.nq + tok < 0;
            const float inv = none ? 0.0f : 1.0f / total;               // (no key: zeros)
            if (!whole && c0 == 0) { part[R * D + 16 * nt + rr] = top; part[R * D + R + 16 * nt + rr] = total; }
            if (KIND != kPlain && whole && here && c0 == 0 && a.lse) a.lse[(size_t)(s.first + tok) * heads + h] = log_sum(a, none, top, total);
            float *kept = nullptr;          // SHARED: a whole unit of a row that has another job
            if constexpr (SHARED) {
                const size_t row = (s.family() ? 0 : (size_t)a.n_tokens * heads) + (size_t)(s.first + tok) * heads + h;
                if (c0 == 0 && first == 0)
                    a.where[row] =
                        whole ? here ? kDone : common
                              : blockIdx.x | (run_with(run, end - 1) - blockIdx.x + 1) << 9 | (uint32_t)(16 * nt + rr) << 19 | a.second | common;
                if (whole && !here) kept = a.whole + row * (D + 4);
                if (kept && c0 == 0) { kept[D] = lifted(a, top); kept[D + 1] = total; }
            }
            const size_t to = (size_t)(s.first + tok) * a.ld_out + (size_t)h * d;
#pragma unroll
            for (int c = 0; c < D / 64; c++) {
                const int dv = 64 * c + 4 * c0;
                f4 x = {0, 0, 0, 0};
#pragma unroll
                for (int y = 0; y < 4; y++) x += *(const f4 *)&s_o[y][rr][dv] * by[y];
                if (!whole) *(f4 *)(part + (size_t)(16 * nt + rr) * D + dv) = x;
                else if (SHARED && kept) *(f4 *)(kept + dv) = x;
                else if (dv < (int)d) {
                    x *= inv;
                    if constexpr (F32) *(f4 *)((float *)a.out + to + dv) = x;
                    else {
                        typedef T v4 __attribute__((ext_vector_type(4)));
                        *(v4 *)((T *)a.out + to + dv) = v4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
                    }
                }
            }
        }
        if (!SHARED && !whole && first == 0 && threadIdx.x == 0) {
            Cut c;
            c.last = run_with(run, end - 1);
            c.first_token = s.first; c.row0 = r0; c.rows = r1 - r0; c.kvh = kvh;
            c.keyless = s.nq > s.len ? (s.nq - s.len) * a.group : 0;
            a.cuts[blockIdx.x] = c;
        }
        t += part_of;
        skip = 0;
        r0 += R;
        if (r0 >= rows) { r0 = 0; kvh++; }
    }
}

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f16v mfma(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16v mfma(b8 a, b8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// The largest of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_halves(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The shape of the kernel below for heads of D: eight waves of kM query rows
// (heads of 256 take twice the registers of a row), keys of a tile.
template <int D> struct Chunk {
    static constexpr int kM = D == 256 ? 16 : 32, kTile = D == 256 ? 32 : 64;
    static constexpr int kRows = 8 * kM, kThreads = 512;
    // What a tile costs beside its rows, in eighths of what 8 kM rows add, where
    // units of many and of few rows are dealt together.  (us of a tile of 64 keys
    // of heads of 128, all 256 workgroups at work, 8 waves with rows, 6 and 1: f16
    // 4.3, 3.7, 1.9, bf16 4.9, 4.1, 2.2; of 32 keys of 256: 2.5, 2.2, 1.6 and 2.8,
    // 2.4, 1.6.  One family of 64 rows over 16000 tokens, 28 / 4 heads, bf16: 84 us,
    // with tiles dealt alike 95.)
    static constexpr int kBase = D == 256 ? 24 : 8;
    // (a run is at least as long as the heaviest tile, also where two share little more than twice that)
    static constexpr int kLeast = 3 * (kBase + 1) > 2 * (kBase + 8) ? 3 * (kBase + 1) : 2 * (kBase + 8);
};
constexpr int kChunkRuns = 256;         // one workgroup per CU

// Chunks of many query rows: what bounds it is the matrix cores and, beside
// them, the exponentials.  A wave has kM query rows, and all waves share the
// tiles of K and V in LDS, two of each, so that the next tile's loads (through
// registers) pass while this one is worked on: one barrier per tile.  The
// products are S^T = K Q^T and O^T = V^T P^T again, 32 x 32 x 16 (heads of 256:
// 16 x 16 x 32, as in the kernel above): a lane has
// the scores of query row lane & 31 for keys 8 x + 4 (lane >> 5) + y, x and
// y < 4, of 32, and gives them back, rounded, as the second product's factor;
// V^T's side takes the same keys by transposing reads of LDS, 4 keys of one
// column each.  Rows of LDS are stored with their 16-byte pieces exchanged so
// that neither reading order meets a bank twice.
// The running maximum is raised only when a score passes it by 2^8, so the
// sums are seldom scaled: the weights then reach 2^8, which f32 sums and the
// type's range (f16: 2^7 is the lift here) take without loss.  Each is rounded to
// T once (SHARED: in kSharedParts), off by 2^-11 of itself (bf16: 2^-8) at most and
// without a common direction; the sum is of the unrounded ones.  A second part, as in the kernel
// above, would cost a quarter: 4 x 2048 over 8192, 32 / 8 heads of 128, f16, 1292
// -> 1641 us; one chunk of 8192, bf16, 664 -> 827.  Without it the relative error
// of the output, most of it the result's own rounding, is 2.16e-4 for 2.09e-4
// (f16) and, in a call of chunks and single tokens, 1.74e-3 for 1.66e-3 (bf16).
// Measured: four chunks of 2048 tokens over 8192, 32 / 8 heads of 128, f16: 740
// TFLOP/s, one chunk of 1024 over 32768, bf16: 850 (a library product of 8192 x
// 8192 x 8192: 1140 and 1200), heads of 64 620, of 256 660.  No bank is met twice;
// vector issue is half of the clocks, the matrix cores two fifths.  Each pass of
// keys and values through LDS serves 32 rows of a wave (64 do not fit its
// registers).
template <class T, int D, bool FULL, Kind KIND>
__global__ void __launch_bounds__(Chunk<D>::kThreads, 2) attn_chunk_kernel(const AttnArgs a)
{
    constexpr bool SHARED = KIND == kShared;
    constexpr int R = Chunk<D>::kRows, kTile = Chunk<D>::kTile, kThreads = Chunk<D>::kThreads;
    constexpr int C = D / 8, KP = kTile * C / kThreads;         // 16-byte pieces of a row; pieces of a thread
    constexpr int M = Chunk<D>::kM, KT = kTile / 32, DT = D / M;
    constexpr int NA = M * M / 64, NZ = M / 2;                  // values of a lane: of a product, of the scores of 32 keys
    constexpr int KF = D / 16;                                  // factors of 32 keys, of K and of V
    using Acc = std::conditional_t<M == 32, f16v, f4>;
    constexpr float kUp = kChunkLift<T>, kSlack = 8.0f;
    typedef typename Vec<T>::v8 v8;
    __shared__ __align__(16) T s_k[2][kTile * D], s_v[2][kTile * D];
    __shared__ uint64_t s_bad[3];                               // of this tile, the next, and one that is cleared

    // runs that follow one another, which read the same keys, on one XCD
    const uint32_t g8 = a.n_wg / 8, run_id = a.n_wg % 8 ? blockIdx.x : (blockIdx.x & 7) * g8 + (blockIdx.x >> 3);
    using S = std::conditional_t<SHARED, Job, Seq>;
    using Dealt = Deal<R, kTile, 3, S, SHARED ? Chunk<D>::kBase : 0, M>;
    Run<S> run = run_of<Dealt, kThreads, SHARED ? Chunk<D>::kLeast : 3>(a, run_id);
    if (!SHARED && threadIdx.x == 0) a.cuts[run_id].last = 0;
    if (run.t0 >= run.t1) return;

    const int lane = threadIdx.x & 63, hg = lane / M, col = lane % M, l16 = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t slot = (1u << a.shift) - 1;
    const uint32_t d = FULL ? D : a.d;
    const size_t head = (size_t)d << a.shift;
    const float scale = fabsf(a.scale);

    // this thread's pieces of a tile: rows prow + kStep .., piece pc, and their places in LDS
    const int pc = threadIdx.x % C, prow = threadIdx.x / C;
    constexpr int kStep = kThreads / C;                         // rows from piece to piece
    auto swap_k = [](int row, int c) { return c ^ (M == 32 ? row & (C < 16 ? C - 1 : 15) : (row & 3) | (row >> 1 & 12)); };
    auto swap_v = [](int row, int c) { return C == 8 ? c ^ (row >> 1 & 1) << 2 : M == 32 ? c ^ (row & 3) << 2 : c ^ (row & 3) << 2 ^ (row >> 2 & 2); };
    // What lane and place i stand for: a key of 32, a value of M
    auto key_of = [&](int i) { return M == 32 ? 8 * (i >> 2) + 4 * hg + (i & 3) : 8 * hg + i; };
    auto value_of = [&](int i) { return M == 32 ? 8 * (i >> 2) + 4 * hg + (i & 3) : 4 * hg + i; };
    const bool inside = 8 * pc < (int)d;

    uint32_t si = run.seq, r0;
    S s = run.s;
    uint64_t t = run.t0;
    uint32_t kvh = (uint32_t)quotient(run.skip, run.per);
    uint64_t before = run.skip - kvh * run.per;
    r0 = Dealt::find(a, s, before);
    uint32_t skip = (uint32_t)before;
    while (t < run.t1) {
        const uint32_t rows = s.nq * a.group;
        if (kvh == a.n_kv || rows == 0) {               // the next sequence
            s = uniform(work_of<S>(a, ++si));
            kvh = 0; r0 = 0;
            continue;
        }
        const uint32_t r1 = min(r0 + R, rows);
        const Span<kTile> span(a, s, r0, r1);
        // the run's part of the unit, tiles first .. first + left - 1
        const uint32_t weight = Dealt::weight(r0, r1);
        const uint32_t dealt = (span.tiles + Dealt::kSetup) * weight, part_of = (uint32_t)min((uint64_t)(dealt - skip), run.t1 - t);
        const uint32_t first = Dealt::tile_at(skip, weight), left = Dealt::tile_at((uint64_t)skip + part_of, weight) - first;
        if (!SHARED && left == 0) break;                // (its setup only: the next run begins it)
        if (SHARED && left == 0) {                      // (or a piece of its last tile)
            t += part_of;
            skip = 0;
            r0 += R;
            if (r0 >= rows) { r0 = 0; kvh++; }
            continue;
        }
        const uint64_t end = t - skip + dealt - (weight - 1);       // behind the last tile's first piece
        const int base = (int)s.len - (int)s.nq;        // position of the sequence's first token

        // ---- queries: row col of the wave's M
        const uint32_t w0 = r0 + M * w;
        const bool rows_here = w0 < r1;
        const uint32_t mine = min(w0 + col, r1 - 1), tok = mine / a.group, hq = kvh * a.group + (mine - tok * a.group);
        int pos = base + (int)tok;
        // the wave's first and last row: positions, and the first keys they see
        int pos0 = base + (int)(min(w0, r1 - 1) / a.group), pos1 = base + (int)(min(w0 + M - 1, r1 - 1) / a.group);
        int least = 0;
        if constexpr (SHARED) least = (int)s.k0;
        auto first_of = [&](int p) { return (int)max((int64_t)least, (int64_t)p + 1 - (int64_t)a.window); };
        int lo = first_of(pos), lo0 = first_of(pos0), lo1 = first_of(pos1);
        int unit_pos0 = base + (int)(r0 / a.group), unit_lo1 = first_of(base + (int)((r1 - 1) / a.group));
        if constexpr (SHARED)
            if (s.family()) {       // every row sees the keys up to the last, from its window's begin on
                pos = pos0 = pos1 = unit_pos0 = (int)s.k1 - 1;
                lo = a.window == 0xffffffffu ? 0 : first_of(a.pos[s.first + tok]);
                lo0 = first_of(s.p0);
                lo1 = unit_lo1 = first_of(s.p1);
            }

        // ---- a tile's pieces
        const uint32_t *table = a.table + (size_t)min(s.row, a.n_rows - 1) * a.ld_table;
        const uint32_t last = span.hi > 0 ? span.hi - 1 : 0;
        u4v kr[KP], vr[KP];
        uint32_t id[KP];
        auto pages = [&](uint32_t key0) {
#pragma unroll
            for (int i = 0; i < KP; i++) id[i] = table[min(key0 + prow + kStep * i, last) >> a.shift];
        };
        auto fetch = [&](uint32_t key0) {
#pragma unroll
            for (int i = 0; i < KP; i++) {
                const uint32_t key = key0 + prow + kStep * i;
                const size_t at = ((size_t)min(id[i], a.n_pages - 1) * a.n_kv + kvh) * head + (size_t)(key & slot) * d + 8 * pc;
                kr[i] = vr[i] = u4v{0, 0, 0, 0};
                if (inside) {
                    kr[i] = *(const u4v *)((const T *)a.k + at);
                    vr[i] = *(const u4v *)((const T *)a.v + at);
                }
            }
        };
        // Values of keys that no row of the unit sees are zeros, and so are
        // those of keys that some rows only see if an infinity or a NaN is
        // among them; s_bad says which (bit: the key of the tile).  So are all
        // such values where weights have parts (SHARED), of which some are 0 or
        // below: an infinity would become a NaN.
        auto put = [&](uint32_t key0, int b, int bs) {
            bool look = (int)key0 + kTile > unit_pos0 + 1 || (int)key0 < unit_lo1;
            if (SHARED && !look) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < KP; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) top |= exponents<T>(vr[i][e]);
                look = __any((top & 0x80008000u) != 0);
            }
            if (look) {
                uint64_t bad = 0;
#pragma unroll
                for (int i = 0; i < KP; i++) {
                    const uint32_t row = prow + kStep * i, key = key0 + row;
                    if (key >= span.hi || key < span.lo) vr[i] = u4v{0, 0, 0, 0};
                    const uint64_t v = __ballot(not_finite<T>(vr[i]));
                    constexpr uint64_t kMask = (1ull << C) - 1;
                    if (v >> (lane / C * C) & kMask) { bad |= 1ull << row; vr[i] = u4v{0, 0, 0, 0}; }
                }
                if (bad) atomicOr((unsigned long long *)&s_bad[bs], (unsigned long long)bad);
            }
#pragma unroll
            for (int i = 0; i < KP; i++) {
                const int row = prow + kStep * i;
                *(u4v *)&s_k[b][row * D + 8 * swap_k(row, pc)] = kr[i];
                *(u4v *)&s_v[b][row * D + 8 * swap_v(row, pc)] = vr[i];
            }
        };

        Acc o[DT];
#pragma unroll
        for (int c = 0; c < DT; c++)
#pragma unroll
            for (int i = 0; i < NA; i++) o[c][i] = 0.0f;
        float mx = -INFINITY, sum = 0.0f;

        uint32_t key0 = span.key0 + (span.tile0 + first) * kTile;
        pages(key0);
        constexpr int QF = M == 32 ? KF : KF / 2, kWide = D / QF;       // factors of the queries, their values
        v8 qf[QF];
        const T *q = (const T *)a.q + (size_t)(s.first + tok) * a.ld_q + (size_t)hq * d;
#pragma unroll
        for (int c = 0; c < QF; c++) {
            v8 x = {};
            if (kWide * c + 8 * hg < (int)d) x = *(const v8 *)(q + kWide * c + 8 * hg);
            qf[c] = a.scale < 0.0f ? -x : x;
        }

        fetch(key0);
        pages(key0 + kTile);
        __syncthreads();                                // (the last unit's tiles are read)
        if (threadIdx.x < 3) s_bad[threadIdx.x] = 0;
        __syncthreads();
        put(key0, 0, 0);
        __syncthreads();
        int bs = 0;                                     // x % 3
        for (uint32_t x = 0; x < left; x++, key0 += kTile) {
            const int b = x & 1;
            const bool more = x + 1 < left;
            if (more) {
                fetch(key0 + kTile);
                pages(key0 + 2 * kTile);
            }
            if (rows_here && (int)key0 <= pos1 && (int)key0 + kTile > lo0) {
                // Each group of reads from LDS is under way while the products of
                // the group before it run; the compiler would put every read
                // right before its use.
                constexpr int kGroups = KF / 4;         // of four factors
                constexpr int NP = NZ / 8, NW = SHARED ? kSharedParts<T> : 1;
                Acc z[KT][M == 32 ? 1 : 2];
                v8 pf[KT][NW][NP], kf[2][4], vf[2][4];
                auto read_k = [&](int y, int gr) {      // of keys 32 y ..
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int f = 4 * gr + c;
                        const int row = M == 32 ? col : 8 * (col >> 2) + 4 * (f & 1) + (col & 3), piece = M == 32 ? 2 * f + hg : 4 * (f >> 1) + hg;
                        kf[(y * kGroups + gr) & 1][c] = *(const v8 *)&s_k[b][(32 * y + row) * D + 8 * swap_k(row, piece)];
                    }
                };
                auto read_v = [&](int y, int gr) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int f = 4 * gr + c;       // M 32: 16 keys f / DT, values 32 (f % DT) ..; M 16: values 16 f ..
                        const int row = (M == 32 ? 16 * (f / DT) + 4 * hg : 8 * hg) + (l16 >> 2);
                        const int piece = M == 32 ? 4 * (f % DT) + 2 * (lane >> 4 & 1) + (l16 >> 1 & 1) : 2 * f + (l16 >> 1 & 1);
                        union { s4v half[2]; v8 all; } u;
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            T *at = &s_v[b][(32 * y + row + (M == 32 ? 8 : 4) * e) * D + 8 * swap_v(row, piece) + 4 * (l16 & 1)];
                            u.half[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)at);
                        }
                        vf[(y * kGroups + gr) & 1][c] = u.all;
                    }
                };
                auto score = [&](int y, int gr) {       // the products of a group
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int f = 4 * gr + c, half = M == 32 ? 0 : f & 1;
                        z[y][half] = mfma(kf[(y * kGroups + gr) & 1][c], qf[M == 32 ? f : f >> 1], z[y][half]);
                    }
                };
                auto add_v = [&](int y, int gr) {
#pragma unroll
                    for (int q = NW - 1; q >= 0; q--)   // (the small parts first)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            const int f = 4 * gr + c;
                            o[f % DT] = mfma(vf[(y * kGroups + gr) & 1][c], pf[y][q][f / DT], o[f % DT]);
                        }
                };
                auto score_of = [&](int y, int i) -> float { return z[y][i / NA][i % NA]; };
                float by = 1.0f;
                bool moved = false;
                // the maximum over 32 keys
                const bool edge = (int)key0 + kTile > pos0 + 1 || (int)key0 < lo1;
                auto raise = [&](int y) {
                    if (edge) {
                        const int up = pos - (int)key0 - 32 * y - key_of(0), down = lo - (int)key0 - 32 * y - key_of(0);
#pragma unroll
                        for (int i = 0; i < NZ; i++) {
                            const int key = M == 32 ? 8 * (i >> 2) + (i & 3) : i;      // from the lane's first
                            if (key > up || key < down) z[y][i / NA][i % NA] = -INFINITY;
                        }
                    }
                    float m[4];                         // (four short chains)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        m[i] = fmaxf(score_of(y, i), score_of(y, 4 + i));
                        if constexpr (NZ == 16) m[i] = fmaxf(m[i], fmaxf(score_of(y, 8 + i), score_of(y, 12 + i)));
                    }
                    float top = max_halves(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
                    if constexpr (M == 16) top = fmaxf(top, __shfl_xor(top, 16));
                    top *= scale;
                    const bool up = top > mx + kSlack;  // (each row by itself: its bits do not depend on its neighbours)
                    moved = __any(up);
                    if (moved) {
                        by = up ? __builtin_amdgcn_exp2f(mx - top) : 1.0f;
                        mx = up ? top : mx;
                        sum *= by;
                    }
                };
                auto scale_o = [&] {
#pragma unroll
                    for (int c = 0; c < DT; c++)
#pragma unroll
                        for (int i = 0; i < NA; i++) o[c][i] *= by;
                };
                float ref;
                auto weigh = [&](int y, int i0, int n) {        // the weights of n scores, and their sum
#pragma unroll
                    for (int i = i0; i < i0 + n; i++) {
                        float x = __builtin_amdgcn_exp2f(fmaf(score_of(y, i), scale, -ref));
                        sum += x;
#pragma unroll
                        for (int q = 0; q < NW; q++) {
                            pf[y][q][i >> 3][i & 7] = (T)x;
                            if (q + 1 < NW) x -= (float)pf[y][q][i >> 3][i & 7];
                        }
                    }
                };
                auto hold = [&](int y) {                // (computed here: else they are put off past the branch that follows)
#pragma unroll
                    for (int i = 0; i < NW * NP; i++) asm volatile("" : "+v"(pf[y][i / NP][i % NP]));
                    asm volatile("" : "+v"(sum));
                };
                // one product and its share of the exponentials in turn
                auto in_turn = [&](auto products) {
                    constexpr int kAll = decltype(products)::value;
#pragma unroll
                    for (int i = 0; i < kAll; i++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, NZ * (2 + 5 * NW) / 2 / kAll, 0);
                    }
                };
#pragma unroll
                for (int y = 0; y < KT; y++)
#pragma unroll
                    for (int i = 0; i < NZ; i++) z[y][i / NA][i % NA] = 0.0f;
                read_k(0, 0);
#pragma unroll
                for (int gr = 0; gr < kGroups; gr++) {
                    if (gr + 1 < kGroups) read_k(0, gr + 1);
                    else if (KT > 1) read_k(1, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    score(0, gr);
                    __builtin_amdgcn_sched_barrier(0);
                }
                read_v(0, 0);
                raise(0);
                if (moved) scale_o();
                ref = mx == -INFINITY ? 0.0f : mx - kUp;
                if constexpr (KT > 1) {
                    // the second 32 keys' scores while the first's exponentials run
#pragma unroll
                    for (int gr = 0; gr < kGroups; gr++) {
                        if (gr + 1 < kGroups) read_k(1, gr + 1);
                        score(1, gr);
                        weigh(0, gr * NZ / kGroups, NZ / kGroups);
                    }
                    in_turn(std::integral_constant<int, KF>());
                    hold(0);
                    raise(1);
                    ref = mx == -INFINITY ? 0.0f : mx - kUp;
                    // and the first's values while the second's run
#pragma unroll
                    for (int gr = 0; gr < kGroups; gr++) {
                        if (gr + 1 < kGroups) read_v(0, gr + 1);
                        else read_v(1, 0);
                        add_v(0, gr);
                        weigh(1, gr * NZ / kGroups, NZ / kGroups);
                    }
                    in_turn(std::integral_constant<int, NW * KF>());
                    hold(1);
                    if (moved) scale_o();
                } else weigh(0, 0, NZ);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int gr = 0; gr < kGroups; gr++) {
                    if (gr + 1 < kGroups) read_v(KT - 1, gr + 1);
                    __builtin_amdgcn_sched_barrier(0);
                    add_v(KT - 1, gr);
                    __builtin_amdgcn_sched_barrier(0);
                }
                // The values that were put aside count for the rows that see them.
                // (The first 32 keys' weights are those to the maximum before the
                // second raise, which has scaled the sums since.)
                const float since = KT > 1 && moved ? by : 1.0f;
                if (SHARED || (int)key0 + kTile > unit_pos0 + 1 || (int)key0 < unit_lo1)
                    for (uint64_t bad = s_bad[bs]; bad; bad &= bad - 1) {
                        const int key = __ffsll((unsigned long long)bad) - 1, y = key & 31;
                        // the place and the lane of its weight
                        const int at = NZ * (key >> 5) + (M == 32 ? (y & 3) + 4 * (y >> 3) : y & 7), from = (M == 32 ? y >> 2 & 1 : y >> 3) * M + col;
                        const uint32_t page = min(table[min(key0 + key, last) >> a.shift], a.n_pages - 1);
                        const T *v = (const T *)a.v + ((size_t)page * a.n_kv + kvh) * head + (size_t)((key0 + key) & slot) * d;
                        float wt = 0.0f;
#pragma unroll
                        for (int i = 0; i < NZ * KT; i++)
                            if (i == at) {
                                wt = (float)pf[i / NZ][NW - 1][i % NZ >> 3][i & 7];
#pragma unroll
                                for (int q = NW - 2; q >= 0; q--) wt += (float)pf[i / NZ][q][i % NZ >> 3][i & 7];
                            }
                        wt = __shfl(wt, from);
                        if (key < 32) wt *= since;
                        if ((int)key0 + key > pos || (int)key0 + key < lo) continue;
#pragma unroll
                        for (int c = 0; c < DT; c++)
#pragma unroll
                            for (int i = 0; i < NA; i++) {
                                const int dv = M * c + value_of(i);
                                if (dv < (int)d) o[c][i] += wt * (float)v[dv];
                            }
                    }
            }
            if (!more) break;
            // (s_bad of the tile before this was read before the last barrier,
            // and is written after the next)
            const int next = bs == 2 ? 0 : bs + 1;
            if (threadIdx.x == 0) s_bad[next == 2 ? 0 : next + 1] = 0;
            put(key0 + kTile, b ^ 1, next);
            bs = next;
            __syncthreads();
        }

        // ---- the unit's rows, or its part
        const bool whole = left == span.tiles;
        sum += __shfl_xor(sum, 32);
        if constexpr (M == 16) sum += __shfl_xor(sum, 16);
        const uint32_t heads = a.n_kv * a.group;
        // SHARED: rows that have keys in common with others have two jobs
        uint32_t common = 0;
        bool here = true, family = false;
        if constexpr (SHARED) {
            family = s.family();
            common = !family && s.k0 ? kCommon : 0;
            here = !family && !common;
        }
        if (w0 + col < r1) {
            size_t row = 0;
            if constexpr (SHARED) row = (family ? 0 : (size_t)a.n_tokens * heads) + (size_t)(s.first + tok) * heads + hq;
            if (SHARED && hg == 0 && first == 0)
                a.where[row] = whole ? here ? kDone : common
                                     : run_id | (run_with(run, end - 1) - run_id + 1) << 9 | (uint32_t)(M * w + col) << 19 | a.second | common;
            if (whole && here) {
                const float inv = pos < 0 ? 0.0f : 1.0f / sum;          // (no key: zeros)
                if (KIND != kPlain && hg == 0 && a.lse) a.lse[(size_t)(s.first + tok) * heads + hq] = log_sum(a, pos < 0, mx, sum);
                T *to = (T *)a.out + (size_t)(s.first + tok) * a.ld_out + (size_t)hq * d;
                typedef T v4 __attribute__((ext_vector_type(4)));
#pragma unroll
                for (int c = 0; c < DT; c++)
#pragma unroll
                    for (int i = 0; i < NA / 4; i++) {
                        const int dv = M * c + value_of(4 * i);
                        if (dv < (int)d) {
                            f4 y = {o[c][4 * i], o[c][4 * i + 1], o[c][4 * i + 2], o[c][4 * i + 3]};
                            y *= inv;
                            *(v4 *)(to + dv) = v4{(T)y[0], (T)y[1], (T)y[2], (T)y[3]};
                        }
                    }
            } else if (SHARED && whole) {
                float *kept = a.whole + row * (D + 4);
                if (hg == 0) { kept[D] = lifted(a, mx); kept[D + 1] = sum; }
#pragma unroll
                for (int c = 0; c < DT; c++)
#pragma unroll
                    for (int i = 0; i < NA / 4; i++)
                        *(f4 *)(kept + M * c + value_of(4 * i)) =
                            f4{o[c][4 * i], o[c][4 * i + 1], o[c][4 * i + 2], o[c][4 * i + 3]};
            } else {
                float *part = a.parts + (size_t)(2 * run_id + (first == 0)) * R * (D + 2);
                const int rr = M * w + col;
                if (hg == 0) { part[R * D + rr] = mx; part[R * D + R + rr] = sum; }
#pragma unroll
                for (int c = 0; c < DT; c++)
#pragma unroll
                    for (int i = 0; i < NA / 4; i++)
                        *(f4 *)(part + (size_t)rr * D + M * c + value_of(4 * i)) =
                            f4{o[c][4 * i], o[c][4 * i + 1], o[c][4 * i + 2], o[c][4 * i + 3]};
            }
        }
        if (!SHARED && !whole && first == 0 && threadIdx.x == 0) {
            Cut c;
            c.last = run_with(run, end - 1);
            c.first_token = s.first; c.row0 = r0; c.rows = r1 - r0; c.kvh = kvh;
            c.keyless = s.nq > s.len ? (s.nq - s.len) * a.group : 0;
            a.cuts[run_id] = c;
        }
        t += part_of;
        skip = 0;
        r0 += R;
        if (r0 >= rows) { r0 = 0; kvh++; }
    }
}

// The parts of the unit that run g begins and another ends.  The
// threads of a row (D / 4 of them, 4 values each) first share out its parts'
// maximums and sums, up to kWide at a time, and then add the parts in order,
// eight reads at a time: what bounds it is the chain of reads.  (Of kernel: one
// token over 4001, 4 heads of keys: 5.1 us; four chunks of 2048 over up to 8192:
// 18 us.  Joining in the first kernel by the last run
// to come needs a release to the other XCDs by each run: 64 single tokens 206
// us like this, 368 so.)
template <class TO, int D, int R, bool LSE> __device__ __forceinline__ void join_unit(const AttnArgs &a, uint32_t g)
{
    const Cut c = a.cuts[g];
    if (c.last == 0) return;
    constexpr int kCols = D / 4, kRows = 256 / kCols, kWide = kCols < 32 ? kCols : 32;
    const uint32_t rr = blockIdx.y * kRows + threadIdx.x / kCols, dv = 4 * (threadIdx.x % kCols), j = threadIdx.x % kWide;
    if (blockIdx.y * kRows >= c.rows) return;
    const uint32_t row = min(rr, c.rows - 1);           // (the threads of a row past the unit's help no one)
    constexpr size_t kPart = (size_t)R * (D + 2);
    const uint32_t n = c.last - g + 1;                  // part 0 is the run's second slot, the others their runs' first
    const float *p0 = a.parts + (size_t)(2 * g) * kPart;
    auto part = [&](uint32_t i) { return p0 + (i ? 2 * (size_t)i : 1) * kPart; };
    float top = -INFINITY;
    for (uint32_t i = j; i < n; i += kWide) top = fmaxf(top, part(i)[R * D + row]);
#pragma unroll
    for (int o = 1; o < kWide; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
    f4 x = {0, 0, 0, 0};
    for (uint32_t i0 = 0; i0 < n; i0 += kWide) {
        float by = 0.0f, add = 0.0f;
        if (i0 + j < n) {
            const float *p = part(i0 + j);
            by = __builtin_amdgcn_exp2f(p[R * D + row] - ref);
            add = by * p[R * D + R + row];
        }
        const uint32_t m = min(n - i0, (uint32_t)kWide);
        for (uint32_t i = 0; i < m; i += 8) {
            f4 y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = *(const f4 *)(part(i0 + min(i + e, m - 1)) + (size_t)row * D + dv);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float b = __shfl(by, (int)((threadIdx.x & 63 & ~(kWide - 1)) + ((i + e) & (kWide - 1))));
                if (i + e < m) x += y[e] * b;
            }
        }
#pragma unroll
        for (int o = 1; o < kWide; o <<= 1) add += __shfl_xor(add, o);
        total += add;
    }
    const uint32_t r = c.row0 + rr, tok = r / a.group;
    if (rr >= c.rows || dv >= a.d) return;
    x *= r < c.keyless ? 0.0f : 1.0f / total;
    if (LSE && dv == 0 && a.lse) a.lse[(size_t)(c.first_token + tok) * a.n_kv * a.group + c.kvh * a.group + r - tok * a.group] = log_sum(a, r < c.keyless, top, total);
    const size_t to = (size_t)(c.first_token + tok) * a.ld_out + (size_t)(c.kvh * a.group + r - tok * a.group) * a.d + dv;
    if constexpr (sizeof(TO) == 4) *(f4 *)((float *)a.out + to) = x;
    else {
        typedef TO v4 __attribute__((ext_vector_type(4)));
        *(v4 *)((TO *)a.out + to) = v4{(TO)x[0], (TO)x[1], (TO)x[2], (TO)x[3]};
    }
}

template <class TO, int D, int R, bool LSE>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) { join_unit<TO, D, R, LSE>(a, blockIdx.x); }

// The parts of both kernels of a call that has sequences for each, in one
// launch (a row of one token and one of 100, over up to 1000: 28.3 us with two,
// 25.4; 24 rows over 700 to 8192, heads of 128: 220, 215).
template <class TO, int D, int R, int R2, bool LSE>
__global__ void __launch_bounds__(256) attn_join_both_kernel(const AttnArgs a, const AttnArgs b)
{
    if (blockIdx.x < a.n_wg) join_unit<TO, D, R, LSE>(a, blockIdx.x);
    else join_unit<TO, D, R2, LSE>(b, blockIdx.x - a.n_wg);
}

} // namespace gs

namespace {

constexpr uint32_t kCUs = 256, kRuns = 2 * kCUs;        // runs at most

int padded(uint32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

size_t cuts_bytes() { return kRuns * ((sizeof(gs::Cut) + 15) / 16 * 16); }

// Bytes of a kernel's parts with R rows in a unit.
size_t parts_bytes(uint32_t runs, int R, int D) { return (size_t)2 * runs * R * (D + 2) * sizeof(float); }

// Of the rows kernel's: 16 rows in each of kRuns runs, or 32 (of heads of 64 in
// as many, of others in half of them).
size_t few_bytes(int D) { return parts_bytes(kRuns, D == 64 ? 32 : 16, D); }

// A call's arguments but for its workspace.
inline int check_attn(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_attn_args *x, const float *lse)
{
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_batch(c, b)) return rc;
    if (!x || layer >= c->n_layers || x->n_heads == 0 || x->n_heads % c->n_kv || x->n_heads > 65535) return GS_ERR_INVALID;
    if (x->type != GS_TYPE_F32 && x->type != c->type) return GS_ERR_UNSUPPORTED;
    if (!std::isfinite(x->scale) || ((uintptr_t)lse & 3u)) return GS_ERR_INVALID;
    if (b->n_tokens == 0) return GS_OK;
    const size_t width = (size_t)x->n_heads * c->d;
    if (!x->q || !x->out || x->q == x->out || x->ld_q < width || x->ld_out < width) return GS_ERR_INVALID;
    if ((((uintptr_t)x->q | (uintptr_t)x->out) & 15u) || x->ld_q % 8 || x->ld_out % 8) return GS_ERR_INVALID;
    // (rows of a sequence are counted in 32 bits)
    if ((uint64_t)b->n_tokens * (x->n_heads / c->n_kv) > 0x7fffffffull) return GS_ERR_UNSUPPORTED;
    return GS_OK;
}

// The most new tokens of a sequence.
inline uint32_t most_tokens(const gs_kv_batch *b, const gs_attn_args *x)
{
    return !b->start ? 1 : x->max_q && x->max_q < b->n_tokens ? x->max_q : b->n_tokens;
}

inline gs::AttnArgs attn_args(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_attn_args *x, float *lse)
{
    gs::AttnArgs a = {};
    const size_t plane = (size_t)c->n_pages * c->n_kv * c->page_size * c->d * 2;
    a.k = (const char *)c->k + layer * plane;
    a.v = (const char *)c->v + layer * plane;
    a.q = x->q; a.out = x->out; a.ld_q = x->ld_q; a.ld_out = x->ld_out;
    a.table = c->table; a.len = c->len; a.rows = b->rows; a.start = b->start;
    a.n = b->n; a.n_tokens = b->n_tokens; a.n_rows = c->rows; a.n_pages = c->n_pages; a.ld_table = c->ld_table;
    a.n_kv = c->n_kv; a.group = x->n_heads / c->n_kv; a.d = c->d;
    a.shift = log2_of(c->page_size);
    a.scale = (float)((x->scale == 0.0f ? 1.0 / sqrt((double)c->d) : (double)x->scale) * M_LOG2E);
    a.window = x->window ? x->window : 0xffffffffu;
    a.lse = lse;
    a.max_rows = 0xffffffffu;
    return a;
}

} // namespace
