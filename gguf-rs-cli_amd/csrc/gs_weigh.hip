// gs_weigh.hip -- the weight that cached tokens get from the newest ones
// (gs_attn_weigh, include/gs_attn.h).
//
// With the logarithms of the softmax's sums at hand a weight is one
// exponential of its own score, so keys can be taken in any order and need no
// maximum: keys stay in registers, the query rows that see them pass by, and
// the weights are added up beside the keys, over all heads.  A weight is
//   exp(scale (q . k) - lse) = c 2^(scale2 (q . k) - n),  n = rint(lse2), c = 2^(n - lse2),
// with n and c of the query row: two multiply-adds and an exponential, and the
// one rounding before the exponential is that of a small number where the
// weight is large.  scale2 is scale log2(e) rounded, and lse2 is lse times
// scale2 / scale, so that its rounding counts only for weights far below 1.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "gs_attn.hpp"

namespace gs {

struct WeighArgs : AttnArgs {           // scale: scale2
    const float *sums;                  // [n_tokens][n_kv group] lse
    float *mass;                        // [n_rows][ld_mass]
    size_t ld_mass;
    float keep;
    float base, base_rest;              // scale2 / scale, and what that is off by
    struct Left *left;                  // [n_wg]
};

// A sequence that is this kernel's, or none of its tokens (len 0).
struct WeighSeq : Seq {};

template <> __device__ __forceinline__ WeighSeq work_of<WeighSeq>(const AttnArgs &a, uint32_t i)
{
    WeighSeq s;
    s.first = a.start ? min(a.start[i], a.n_tokens) : i;
    const uint32_t end = a.start ? min(a.start[i + 1], a.n_tokens) : i + 1;
    s.nq = end > s.first ? end - s.first : 0;
    s.row = a.rows ? a.rows[i] : i;
    s.len = s.row < a.n_rows && s.nq * a.group >= a.min_rows && s.nq * a.group <= a.max_rows ? min(a.len[s.row], a.ld_table << a.shift) : 0;
    return s;
}
__device__ __forceinline__ WeighSeq uniform(const WeighSeq &s)
{
    WeighSeq u;
    (Seq &)u = uniform((const Seq &)s);
    return u;
}

// The keys of a sequence whose weights change, kTile at a time: all of its
// tokens where they are scaled, else those that its new tokens see.
template <int kTile> struct Keys {
    uint32_t lo, hi, tile0, tiles;
    __device__ __forceinline__ Keys(const WeighArgs &x, const Seq &s)
    {
        const int64_t p0 = (int64_t)s.len - s.nq;
        hi = s.len;
        lo = x.keep != 1.0f ? 0 : s.nq ? (uint32_t)min((int64_t)s.len, max((int64_t)0, p0 + 1 - (int64_t)x.window)) : s.len;
        tile0 = lo / kTile;
        tiles = hi > lo ? (hi + kTile - 1) / kTile - tile0 : 0;
    }
};

// The query rows of a sequence that see one of the keys key0 .. key0 + n - 1.
struct Seers {
    uint32_t r0, r1;
    __device__ __forceinline__ Seers(const WeighArgs &x, const Seq &s, uint32_t key0, uint32_t n)
    {
        const int64_t base = (int64_t)s.len - s.nq;
        const int64_t t0 = max((int64_t)0, (int64_t)key0 - base), t1 = min((int64_t)s.nq, (int64_t)key0 + n - 1 + (int64_t)x.window - base);
        r0 = (uint32_t)min(t0, (int64_t)s.nq) * x.group;
        r1 = t1 > 0 ? max(r0, (uint32_t)t1 * x.group) : r0;
    }
};

// A sequence of a row that an earlier one has counts there. (a wave)
__device__ __forceinline__ bool is_first(const AttnArgs &a, uint32_t i)
{
    if (!a.rows) return true;
    const uint32_t row = a.rows[i], lane = threadIdx.x & 63;
    for (uint32_t j = 0; j < i; j += 64)
        if (__any(j + lane < i && a.rows[j + lane] == row)) return false;
    return true;
}

// n and c of a query row.  (A sum that is no finite number keeps its meaning.)
__device__ __forceinline__ void base_of(const WeighArgs &x, float lse, float &n, float &c)
{
    const float hi = lse * x.base, lo = fmaf(lse, x.base, -hi) + lse * x.base_rest;
    n = rintf(hi);
    c = __builtin_amdgcn_exp2f((n - hi) - lo);
    if (!(fabsf(hi) < INFINITY)) { n = lse; c = 1.0f; }
}

// A score without the parts of a 32-bit query, which make a NaN of an infinity.
template <class T> __device__ __forceinline__ float dot(const float *q, const T *k, uint32_t d)
{
    float z = 0.0f;
    for (uint32_t c = 0; c < d; c++) z += q[c] * (float)k[c];
    return z;
}

// A token's weight, with what it had before.
__device__ __forceinline__ void add_mass(const WeighArgs &a, uint32_t row, uint32_t key, float sum)
{
    float *mass = a.mass + row * a.ld_mass + key;
    *mass = a.keep == 0.0f ? sum : a.keep * *mass + sum;
}

// The few-rows kernel: kFewKeys keys of a wave, tiles dealt in equal runs.
constexpr int kFewKeys = 32;
struct FewDeal {
    using Work = WeighSeq;
    static __device__ __forceinline__ uint32_t heads(const WeighArgs &) { return 1; }
    static __device__ __forceinline__ uint64_t count(const WeighArgs &a, const WeighSeq &s) { return Keys<kFewKeys>(a, s).tiles; }
    static __device__ __forceinline__ uint64_t count_wave(const WeighArgs &a, const WeighSeq &s) { return count(a, s); }
};

// For single tokens and few of them what bounds it is the read of the keys.  A
// wave takes 32 keys and goes through the heads and the rows, 16 at a time; a
// token's sum is made by one wave, in one order.  Runs of so few tiles that heads
// of keys one after the other would take longer share out the heads instead, and
// the waves' sums are added in order.  (us: one token over 4001, 28 / 4 heads, f32,
// 10.7 and 8.2 so; 64 over 1000 to 32768, bf16, 112, which is 5.2 TB/s.)
template <class T, int D, bool F32>
__global__ void __launch_bounds__(256) weigh_few_kernel(const WeighArgs a)
{
    constexpr int KS = D / 32, NP = F32 ? 3 : 1;
    typedef typename Vec<T>::v8 v8;
    const Run<WeighSeq> run = run_of<FewDeal, 256, 1>(a, blockIdx.x);
    if (run.t0 >= run.t1) return;
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const uint32_t w = uniform(threadIdx.x >> 6);
    const uint32_t page = 1u << a.shift, d = a.d;
    const size_t head = (size_t)d << a.shift;
    uint32_t si = run.seq;
    WeighSeq s = run.s;
    uint64_t before = run.t0 - run.skip;            // tiles of the sequences before
    __shared__ float s_part[4][kFewKeys];
    const bool split = (run.t1 - run.t0) * ((a.n_kv + 3) / 4) < a.n_kv && run.t1 - run.t0 < 4;
    const uint32_t kv0 = split ? w : 0, kv_step = split ? 4 : 1, t_step = split ? 1 : 4;
    for (uint64_t t = run.t0 + (split ? 0 : w);; si++, s = uniform(work_of<WeighSeq>(a, si))) {
        const Keys<kFewKeys> keys(a, s);
        const uint64_t end = min(before + keys.tiles, run.t1);
        if (t < end) {
            const bool mine = is_first(a, si);
            const uint32_t *table = a.table + (size_t)min(s.row, a.n_rows - 1) * a.ld_table;
            const int64_t base = (int64_t)s.len - s.nq;
            for (; t < end; t += t_step) {
                if (!mine) continue;
                const uint32_t key0 = (keys.tile0 + (uint32_t)(t - before)) * kFewKeys;
                const Seers rows(a, s, key0, kFewKeys);
                uint32_t id[2];
#pragma unroll
                for (int y = 0; y < 2; y++) id[y] = min(table[min(key0 + 16 * y + m, s.len - 1) >> a.shift], a.n_pages - 1);
                float sum[2][4] = {};
                for (uint32_t kvh = kv0; kvh < a.n_kv && rows.r0 < rows.r1; kvh += kv_step) {
                    v8 kf[2][KS];
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const T *p = (const T *)a.k + ((size_t)id[y] * a.n_kv + kvh) * head + (size_t)((key0 + 16 * y + m) & (page - 1)) * d;
#pragma unroll
                        for (int c = 0; c < KS; c++) {
                            v8 z = {};
                            if (32 * c + 8 * g < (int)d) z = *(const v8 *)(p + 32 * c + 8 * g);
                            kf[y][c] = z;
                        }
                    }
                    for (uint32_t r = rows.r0; r < rows.r1; r += 16) {
                        const uint32_t rr = min(r + m, rows.r1 - 1), tok = rr / a.group, h = kvh * a.group + (rr - tok * a.group);
                        const size_t at = (size_t)(s.first + tok) * a.ld_q + (size_t)h * d;
                        float n, by;
                        base_of(a, a.sums[(size_t)(s.first + tok) * a.n_kv * a.group + h], n, by);
                        const int64_t pos = r + m < rows.r1 ? base + tok : -1;
                        v8 qf[NP][KS];
                        float unscale = a.scale;
                        if constexpr (F32) {
                            float f[KS][8], top = 0.0f;
#pragma unroll
                            for (int c = 0; c < KS; c++) {
                                if (32 * c + 8 * g < (int)d) load8((const float *)a.q + at + 32 * c + 8 * g, f[c]);
                                else
#pragma unroll
                                    for (int e = 0; e < 8; e++) f[c][e] = 0.0f;
#pragma unroll
                                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(f[c][e]));
                            }
                            top = fmaxf(top, __shfl_xor(top, 16));
                            top = fmaxf(top, __shfl_xor(top, 32));
                            int ex = 0;
                            if (__is_same(T, _Float16) && top > 0.0f && top < INFINITY) ex = 14 - ilogbf(top);
                            unscale *= ldexpf(1.0f, -ex);
#pragma unroll
                            for (int c = 0; c < KS; c++)
#pragma unroll
                                for (int e = 0; e < 8; e++) {
                                    const float y = ldexpf(f[c][e], ex);
                                    const T p0 = (T)y;
                                    const float y1 = y - (float)p0;
                                    const T p1 = (T)y1;
                                    qf[0][c][e] = p0;
                                    qf[1][c][e] = p1;
                                    qf[2][c][e] = (T)(y1 - (float)p1);
                                }
                        } else {
#pragma unroll
                            for (int c = 0; c < KS; c++) {
                                v8 z = {};
                                if (32 * c + 8 * g < (int)d) z = *(const v8 *)((const T *)a.q + at + 32 * c + 8 * g);
                                qf[0][c] = z;
                            }
                        }
                        f4 z[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
                        for (int y = 0; y < 2; y++)
#pragma unroll
                            for (int q = NP - 1; q >= 0; q--)           // (the small parts first)
#pragma unroll
                                for (int c = 0; c < KS; c++) z[y] = mfma(kf[y][c], qf[q][c], z[y]);
                        // lane: keys key0 + 16 y + 4 g + e of row r + m
#pragma unroll
                        for (int y = 0; y < 2; y++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int64_t key = (int64_t)key0 + 16 * y + 4 * g + e;
                                const bool sees = key <= pos && key > pos - (int64_t)a.window;
                                float x = fmaf(z[y][e], unscale, -n);
                                if constexpr (F32)
                                    if (sees && x != x && n == n) {
                                        const uint32_t p = min(table[(uint32_t)key >> a.shift], a.n_pages - 1);
                                        x = dot((const float *)a.q + at, (const T *)a.k + ((size_t)p * a.n_kv + kvh) * head + (size_t)((uint32_t)key & (page - 1)) * d, d) * a.scale - n;
                                    }
                                if (sees) sum[y][e] = fmaf(__builtin_amdgcn_exp2f(x), by, sum[y][e]);
                            }
                    }
                }
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int o = 1; o < 16; o <<= 1) sum[y][e] += __shfl_xor(sum[y][e], o);
                if (split) {
                    __syncthreads();                // (the last tile's sums are read)
                    if (m == 0)
#pragma unroll
                        for (int y = 0; y < 2; y++)
#pragma unroll
                            for (int e = 0; e < 4; e++) s_part[w][16 * y + 4 * g + e] = sum[y][e];
                    __syncthreads();
                    const uint32_t key = key0 + lane;
                    if (w == 0 && lane < kFewKeys && key >= keys.lo && key < keys.hi)
                        add_mass(a, s.row, key, (s_part[0][lane] + s_part[1][lane]) + (s_part[2][lane] + s_part[3][lane]));
                    continue;
                }
                if (m != 0) continue;
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t key = key0 + 16 * y + 4 * g + e;
                        if (key >= keys.lo && key < keys.hi) add_mass(a, s.row, key, sum[y][e]);
                    }
            }
        }
        before += keys.tiles;
        if (before >= run.t1) break;
    }
}

// The shape of the kernel below for heads of D: four waves of kMine keys, tiles
// of kRows query rows (in three parts twice as many would leave room for one
// workgroup in a CU), and the workgroups that a CU takes.  (us with 64 keys of a
// wave, two workgroups, and with 32, three: 4 x 2048 tokens over up to 8192, 350,
// 363; 7 x 32 over up to 12000, 47, 45; one of 2000, 72, 62; 4 x 64 over up to
// 12000, heads of 64, 32, 26.)  With 32-bit queries LDS says how many: 29, 53 and
// 101 KB of 160, of which three of 53 are not to be had.  (us with two for all heads,
// and so: heads of 64, 4 x 1024 over 8192, 298, 236; 7 x 32 over up to 12000, 43, 38;
// one of 2000, 56, 59; of 256, 4 x 256 over 8192, 291, 279; one of 2000, 125, 104.  Of
// 128 with three: 4 x 512 over 8192, 318, 379.)
template <int D, bool F32> struct Many {
    static constexpr int kMine = 32, kKeys = 4 * kMine, kRows = F32 ? 32 : 64, kPerCU = F32 ? D == 64 ? 3 : D == 128 ? 2 : 1 : D == 256 ? 2 : 3;
    static constexpr int kSetup = 1;                // the keys' way and the sums', dealt as tiles of rows
};
constexpr int kManyRuns = 3 * 256;                  // at most

// A block of keys that a run begins and does not end.
struct Left {
    uint32_t last;                                  // the run that ends it; 0: none
    uint32_t row, key0, lo, hi;
};

// How its work is dealt: of a sequence, a block of keys after the other, each
// with all heads of keys one after the other, each with the rows that see one
// of the block's keys, kRows at a time.
template <int D, bool F32> struct ManyDeal {
    using Work = WeighSeq;
    using M = Many<D, F32>;
    static constexpr int kKeys = M::kKeys;
    static __device__ __forceinline__ uint32_t heads(const WeighArgs &a) { return a.n_kv; }
    static __device__ __forceinline__ uint32_t block(const WeighArgs &a, const WeighSeq &s, uint32_t tile)
    {
        const Seers r(a, s, tile * kKeys, kKeys);
        return (r.r1 - r.r0 + M::kRows - 1) / M::kRows + M::kSetup;
    }
    static __device__ __forceinline__ uint64_t count(const WeighArgs &a, const WeighSeq &s)
    {
        const Keys<kKeys> k(a, s);
        uint64_t t = 0;
        for (uint32_t b = 0; b < k.tiles; b++) t += block(a, s, k.tile0 + b);
        return t;
    }
    static __device__ __forceinline__ uint64_t count_wave(const WeighArgs &a, const WeighSeq &s)
    {
        const Keys<kKeys> k(a, s);
        uint64_t t = 0;
        for (uint32_t b = threadIdx.x & 63; b < k.tiles; b += 64) t += block(a, s, k.tile0 + b);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) t += __shfl_xor(t, o);
        return t;
    }
    // The block that tile `skip` of the sequence is in; skip becomes the tile's
    // number in it. (a wave)
    static __device__ __forceinline__ uint32_t find(const WeighArgs &a, const WeighSeq &s, uint64_t &skip)
    {
        const Keys<kKeys> k(a, s);
        const uint32_t lane = threadIdx.x & 63;
        for (uint32_t b = 0;; b += 64) {
            const uint64_t mine = b + lane < k.tiles ? (uint64_t)block(a, s, k.tile0 + b + lane) * a.n_kv : 0;
            uint64_t sum = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint64_t y = __shfl_up(sum, o);
                if (lane >= o) sum += y;
            }
            const uint64_t past = __ballot(sum > skip);
            if (past) {
                const int at = __ffsll((unsigned long long)past) - 1;
                skip -= uniform((uint64_t)__shfl(sum - mine, at));
                return b + at;
            }
            skip -= uniform((uint64_t)__shfl(sum, 63));
        }
    }
};

// For chunks of tokens what bounds it is the matrix cores and, beside them, the
// exponentials.  A wave holds its keys of a head as factors, kRows rows of queries
// at a time pass through LDS for all four waves (two tiles of them, so that the
// next one's loads pass while this one is worked on), and a lane adds up the
// weights of query row lane & 31 for the keys that its results of S^T = K Q^T,
// 32 x 32 x 16, are of.  Measured: 4 x 2048 tokens over 2100 to 8192, 32 / 8 heads
// of 128, bf16: 372 us a call, of which weigh_join_kernel 5, 655 TFLOP/s (a library
// product of 8192 x 8192 x 8192: 1226); by itself, under a profiler, whose load lowers
// the clock, 381 to 437.  Vector issue is 63 % of the clocks, the matrix cores 33 %,
// no bank is met twice.  7 x 32 over 3001 to 12000: 42 us, 2.3 TB/s: each head's keys
// are waited
// for before 128 rows of queries.
template <class T, int D, bool F32>
__global__ void __launch_bounds__(256, (Many<D, F32>::kPerCU)) weigh_many_kernel(const WeighArgs a)
{
    using M = Many<D, F32>;
    constexpr int kMine = M::kMine, kKeys = M::kKeys, kSetup = M::kSetup, kRows = M::kRows, U = kRows / 32;
    constexpr int KF = D / 16, NP = F32 ? 3 : 1, C = D / 8, kEach = C / 8;      // factors; parts; 16-byte pieces of a row, of a thread
    typedef typename Vec<T>::v8 v8;
    // (rows 16 bytes apart beyond their length: 16 of them meet no bank twice, and a
    // lane's factors are at constant distances)
    constexpr int kRow = D + 8;
    __shared__ __align__(16) T s_q[2][NP][kRows * kRow];
    __shared__ float s_n[2][kRows], s_c[2][kRows], s_u[2][kRows];
    __shared__ float s_sum[kKeys];
    using Dealt = ManyDeal<D, F32>;
    const Run<WeighSeq> run = run_of<Dealt, 256, 4>(a, blockIdx.x);
    if (threadIdx.x == 0) a.left[blockIdx.x].last = 0;
    if (run.t0 >= run.t1) return;

    const int lane = threadIdx.x & 63, hg = lane >> 5, col = lane & 31;
    const uint32_t w = uniform(threadIdx.x >> 6);
    const int prow = threadIdx.x >> 3, pc = threadIdx.x & 7;        // this thread's first row of a tile of queries (the others 32 apart); its pieces pc + 8 i
    const uint32_t slot = (1u << a.shift) - 1, d = a.d;
    const size_t head = (size_t)d << a.shift;

    uint32_t si = run.seq;
    WeighSeq s = run.s;
    uint64_t t = run.t0, skip = run.skip;
    uint32_t b = Dealt::find(a, s, skip);
    bool mine = is_first(a, si);
    // Of the waves that want to issue the oldest is taken: the first of a CU's
    // workgroups would be done long before the others.  The one that has more of
    // its run before it goes first, by quarters.  (4 x 2048 tokens over up to 8192:
    // 378 -> 348 us, with two workgroups in a CU.)
    uint32_t done = 0, level = 3;
    const uint32_t quarter = (uint32_t)(run.t1 - run.t0) / 4;
    __builtin_amdgcn_s_setprio(3);
    while (t < run.t1) {
        const Keys<kKeys> keys(a, s);
        if (b >= keys.tiles) {                                      // the next sequence
            s = uniform(work_of<WeighSeq>(a, ++si));
            mine = is_first(a, si);
            b = 0;
            continue;
        }
        const uint32_t key0 = (keys.tile0 + b) * kKeys, w0 = key0 + kMine * w;
        const Seers rows(a, s, key0, kKeys);
        const uint32_t per = (rows.r1 - rows.r0 + kRows - 1) / kRows + kSetup;
        const uint64_t all = (uint64_t)per * a.n_kv, part = min(all - skip, run.t1 - t);
        const int base = (int)s.len - (int)s.nq;
        const uint32_t *table = a.table + (size_t)min(s.row, a.n_rows - 1) * a.ld_table;

        float sum[16];
#pragma unroll
        for (int i = 0; i < 16; i++) sum[i] = 0.0f;
        // the last rows' exponents and factors, whose exponentials are still to come
        float wait[16], wait_by = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) wait[i] = -INFINITY;
        auto weigh = [&](int i0, int i1) {
#pragma unroll
            for (int i = i0; i < i1 && i < 16; i++) {
                sum[i] = fmaf(__builtin_amdgcn_exp2f(wait[i]), wait_by, sum[i]);
                asm volatile("" : "+v"(sum[i]));                    // (here: else it is put off past the branch that follows)
            }
        };
        const uint32_t kv0 = (uint32_t)quotient(skip, per), kv1 = (uint32_t)quotient(skip + part - 1, per);
        // tiles of rows x0 .. x1 - 1 of head kvh are this run's
        auto tiles_of = [&](uint32_t kvh, uint32_t &x0, uint32_t &x1) {
            const uint64_t at = (uint64_t)kvh * per, lo = max(skip, at) - at, hi = min(skip + part, at + per) - at;
            x0 = max((uint32_t)lo, (uint32_t)kSetup) - kSetup;
            x1 = max((uint32_t)hi, (uint32_t)kSetup) - kSetup;
        };
        for (uint32_t kvh = kv0; kvh <= kv1 && mine; kvh++) {
            uint32_t x0, x1;
            tiles_of(kvh, x0, x1);
            if (x0 >= x1) continue;
            v8 kf[KF];
            const uint32_t key = w0 + col, id = min(table[min(key, s.len - 1) >> a.shift], a.n_pages - 1);
            const T *keys_at = (const T *)a.k + ((size_t)id * a.n_kv + kvh) * head + (size_t)(key & slot) * d;
#pragma unroll
            for (int c = 0; c < KF; c++) {
                v8 z = {};
                if (16 * c + 8 * hg < (int)d) z = *(const v8 *)(keys_at + 16 * c + 8 * hg);
                kf[c] = z;
            }
            // A tile of queries through registers to LDS.  The bases of its rows are
            // a wave's, another one's for each tile.
            v8 qr[F32 ? 1 : U][F32 ? 1 : kEach];
            float fr[F32 ? U : 1][F32 ? kEach : 1][8], lse = 0.0f;
            auto row_of = [&](uint32_t r, uint32_t &tok, uint32_t &h) {     // (rows past the last are the last once more)
                r = min(r, rows.r1 - 1);
                tok = r / a.group;
                h = r - tok * a.group;
            };
            // where a thread's rows are: from tile to tile by additions
            const size_t step = (size_t)(kRows / a.group) * a.ld_q + (size_t)(kRows % a.group) * d, wrap = a.ld_q - (size_t)a.group * d;
            size_t at[U];
            uint32_t head_at[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint32_t tok;
                row_of(rows.r0 + kRows * x0 + prow + 32 * u, tok, head_at[u]);
                at[u] = (size_t)(s.first + tok) * a.ld_q + (size_t)(kvh * a.group + head_at[u]) * d;
            }
            auto fetch = [&](uint32_t x) {
                const bool last = rows.r0 + kRows * (x + 1) > rows.r1;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (last && x > x0) {
                        uint32_t tok, h;
                        row_of(rows.r0 + kRows * x + prow + 32 * u, tok, h);
                        at[u] = (size_t)(s.first + tok) * a.ld_q + (size_t)(kvh * a.group + h) * d;
                    }
#pragma unroll
                    for (int i = 0; i < kEach; i++) {
                        const int c = 8 * (pc + 8 * i);
                        if constexpr (F32) {
#pragma unroll
                            for (int e = 0; e < 8; e++) fr[u][i][e] = 0.0f;
                            if (c < (int)d) load8((const float *)a.q + at[u] + c, fr[u][i]);
                        } else {
                            v8 z = {};
                            if (c < (int)d) z = *(const v8 *)((const T *)a.q + at[u] + c);
                            qr[u][i] = z;
                        }
                    }
                    at[u] += step;
                    head_at[u] += kRows % a.group;
                    if (head_at[u] >= a.group) { head_at[u] -= a.group; at[u] += wrap; }
                }
                if (w == (x & 3) && lane < kRows) {
                    uint32_t tok, h;
                    row_of(rows.r0 + kRows * x + lane, tok, h);
                    lse = a.sums[((size_t)(s.first + tok) * a.n_kv + kvh) * a.group + h];
                }
            };
            auto put = [&](uint32_t x, int o) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int row = prow + 32 * u;
                    if constexpr (F32) {
                        float top = 0.0f;
#pragma unroll
                        for (int i = 0; i < kEach; i++)
#pragma unroll
                            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(fr[u][i][e]));
#pragma unroll
                        for (int k = 1; k < 8; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
                        int ex = 0;
                        if (__is_same(T, _Float16) && top > 0.0f && top < INFINITY) ex = 14 - ilogbf(top);
                        if (pc == 0) s_u[o][row] = a.scale * ldexpf(1.0f, -ex);
#pragma unroll
                        for (int i = 0; i < kEach; i++) {
                            v8 p[3];
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                const float y = ldexpf(fr[u][i][e], ex);
                                p[0][e] = (T)y;
                                const float y1 = y - (float)p[0][e];
                                p[1][e] = (T)y1;
                                p[2][e] = (T)(y1 - (float)p[1][e]);
                            }
#pragma unroll
                            for (int q = 0; q < 3; q++) *(v8 *)&s_q[o][q % NP][row * kRow + 8 * (pc + 8 * i)] = p[q];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < kEach; i++) *(v8 *)&s_q[o][0][row * kRow + 8 * (pc + 8 * i)] = qr[u][i];
                    }
                }
                if (w == (x & 3) && lane < kRows) {
                    float n, c;
                    base_of(a, lse, n, c);
                    s_n[o][lane] = n;
                    s_c[o][lane] = rows.r0 + kRows * x + lane < rows.r1 ? c : 0.0f;
                }
            };
            fetch(x0);
            __syncthreads();                                        // (the last head's tiles are read)
            put(x0, 0);
            __syncthreads();
            for (uint32_t x = x0; x < x1; x++) {
                const int o = (x - x0) & 1;
                const bool more = x + 1 < x1;
                if (++done > quarter) {
                    done = 0;
                    if (--level == 2) __builtin_amdgcn_s_setprio(2);
                    else if (level == 1) __builtin_amdgcn_s_setprio(1);
                    else __builtin_amdgcn_s_setprio(0);
                }
                if (more) fetch(x + 1);
#pragma unroll 1
                for (int u = 0; u < U; u++) {
                    // 32 rows at a time: their first and last positions
                    const uint32_t ra = rows.r0 + kRows * x + 32 * u, rb = min(ra + 31, rows.r1 - 1);
                    if (ra >= rows.r1) break;
                    const int pa = base + (int)(ra / a.group), pb = base + (int)(rb / a.group);
                    if ((int)w0 <= pb && (int64_t)w0 + kMine > (int64_t)pa + 1 - (int64_t)a.window) {
                        const float n = s_n[o][32 * u + col], by = s_c[o][32 * u + col], unscale = F32 ? s_u[o][32 * u + col] : a.scale;
                        const bool edge = (int)w0 + kMine > pa + 1 || (int64_t)w0 < (int64_t)pb + 1 - (int64_t)a.window;
                        // these scores while the last ones' exponentials run; the factors
                        // come from LDS kAhead products before theirs
                        constexpr int kAll = NP * KF, kAhead = 4, kFirst = 4, kTurn = (16 - kFirst + kAll - 1) / kAll;
                        v8 f[kAhead];
                        auto factor = [&](int p) {                          // (the small parts first)
                            f[p % kAhead] = *(const v8 *)&s_q[o][NP - 1 - p / KF][(32 * u + col) * kRow + 8 * (2 * (p % KF) + hg)];
                        };
                        f16v z;
#pragma unroll
                        for (int i = 0; i < 16; i++) z[i] = 0.0f;
#pragma unroll
                        for (int p = 0; p < kAhead; p++) factor(p);
                        weigh(0, kFirst);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int p = 0; p < kAll; p++) {
                            z = mfma(kf[p % KF], f[p % kAhead], z);
                            if (p + kAhead < kAll) factor(p + kAhead);
                            weigh(kFirst + kTurn * p, kFirst + kTurn * (p + 1));
                            __builtin_amdgcn_sched_barrier(0);
                        }
#pragma unroll
                        for (int i = 0; i < 16; i++) wait[i] = fmaf(z[i], unscale, -n);
                        wait_by = by;
                        if (edge) {
                            const int pos = base + (int)(min(ra + col, rb) / a.group);
                            const int up = pos - (int)w0 - 4 * hg, down = (int)max((int64_t)-1, (int64_t)pos + 1 - (int64_t)a.window - w0) - 4 * hg;
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const int key = 8 * (i >> 2) + (i & 3);             // from the lane's first
                                if (key > up || key < down) wait[i] = -INFINITY;
                            }
                        }
                    }
                }
                if (more) put(x + 1, o ^ 1);
                __syncthreads();
            }
        }

        weigh(0, 16);

        // ---- the block's sums, or this run's part of them
#pragma unroll
        for (int i = 0; i < 16; i++) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) sum[i] += __shfl_xor(sum[i], o);
            if (col == 0) s_sum[kMine * w + 8 * (i >> 2) + 4 * hg + (i & 3)] = sum[i];
        }
        if constexpr (F32) {                        // keys that met an infinity once more, by 64 lanes beside one another
            for (uint32_t k = 0; k < kMine; k++) {
                const float old = s_sum[kMine * w + k];
                if (__builtin_expect(old == old, 1)) continue;
                const uint32_t key = w0 + k;
                float add = 0.0f;
                bool none = key >= s.len;           // (a NaN that is no infinity's ends it)
                for (uint32_t kvh = kv0; kvh <= kv1 && !none; kvh++) {
                    uint32_t x0, x1;
                    tiles_of(kvh, x0, x1);
                    const uint32_t id = min(table[key >> a.shift], a.n_pages - 1), end = min(rows.r0 + kRows * x1, rows.r1);
                    const T *p = (const T *)a.k + ((size_t)id * a.n_kv + kvh) * head + (size_t)(key & slot) * d;
                    for (uint32_t r0 = rows.r0 + kRows * x0; r0 < end && !none; r0 += 64) {
                        const uint32_t r = min(r0 + lane, end - 1), tok = r / a.group, h = kvh * a.group + (r - tok * a.group);
                        const int pos = base + (int)tok;
                        if (r0 + lane < end && (int)key <= pos && (int64_t)key > (int64_t)pos - (int64_t)a.window) {
                            float n, c;
                            base_of(a, a.sums[(size_t)(s.first + tok) * a.n_kv * a.group + h], n, c);
                            float x = n;
                            if (n == n) x = fmaf(dot((const float *)a.q + (size_t)(s.first + tok) * a.ld_q + (size_t)h * d, p, d), a.scale, -n);
                            add += c * __builtin_amdgcn_exp2f(x);
                        }
                        none = __any(add != add);
                    }
                }
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) add += __shfl_xor(add, o);
                if (lane == 0) s_sum[kMine * w + k] = add;
            }
        }
        const bool whole = skip == 0 && part == all;
        float *parts = a.parts + (size_t)(2 * blockIdx.x + (skip == 0)) * kKeys;
        if (lane < kMine) {
            const uint32_t key = w0 + lane;
            const float x = s_sum[kMine * w + lane];
            if (!whole) parts[kMine * w + lane] = x;
            else if (mine && key >= keys.lo && key < keys.hi) add_mass(a, s.row, key, x);
        }
        if (!whole && skip == 0 && mine && threadIdx.x == 0)
            a.left[blockIdx.x] = Left{run_with(run, t + all - 1), s.row, key0, keys.lo, keys.hi};
        t += part;
        skip = 0;
        b++;
    }
}

// The parts of the block that run blockIdx.x begins and another ends, in order.
// (4 to 5 us: three reads in a row and a launch.)
__global__ void __launch_bounds__(256) weigh_join_kernel(const WeighArgs a, int keys)
{
    const Left l = a.left[blockIdx.x];
    const uint32_t key = l.key0 + threadIdx.x;
    if (l.last == 0 || (int)threadIdx.x >= keys || key < l.lo || key >= l.hi) return;
    const float *p = a.parts + (size_t)2 * blockIdx.x * keys + threadIdx.x;
    float sum = p[keys];                            // part 0 is the run's second slot, the others their runs' first
    for (uint32_t i = 1; i <= l.last - blockIdx.x; i++) sum += p[(size_t)2 * i * keys];
    add_mass(a, l.row, key, sum);
}

} // namespace gs

namespace {

constexpr size_t kLeftBytes = (gs::kManyRuns * sizeof(gs::Left) + 15) / 16 * 16;
// Query rows per head of keys that the first kernel takes.  (us with 16, 32, 64; 16
// sequences over up to 8000, 32 / 8 heads of 128, f16, 24 rows: 65, 56, 56; 32: 65, 59,
// 59; 48: 66, 66, 67; 64: 67, 67, 77.  f32, 8 sequences, 24: 45, 51, 51; 48: 58, 58, 66;
// 64: 58, 58, 78.  Four, heads of 64, 32: 16, 10, 10; heads of 256, eight, 24 to 64:
// within 2 of one another.)
constexpr uint32_t kFewRows = 32;

template <class T, int D, bool F32> void by_rows(gs::WeighArgs a, uint64_t rows, hipStream_t st)
{
    const bool few = rows <= kFewRows, alike = (uint64_t)a.n_tokens * a.group == rows * a.n;
    if (few || !alike) {
        a.max_rows = few ? 0xffffffffu : kFewRows;
        // (us with 512, 1024, 2048 runs: 16 single tokens over up to 4000, 28 / 4 heads,
        // bf16: 16.7, 14.9, 17.9; 64 over up to 32768: 115, 112, 108; 8 x 4 over up to
        // 6000, 32 / 8, f16: 22.4, 20.4, 23.2; heads of 256, f32, 4 over up to 12000: 47,
        // 53, 53)
        a.n_wg = 1024;
        hipLaunchKernelGGL((gs::weigh_few_kernel<T, D, F32>), dim3(a.n_wg), dim3(256), 0, st, a);
    }
    if (few) return;
    a.min_rows = alike ? 0 : kFewRows + 1;
    a.max_rows = 0xffffffffu;
    a.n_wg = 256 * gs::Many<D, F32>::kPerCU;
    hipLaunchKernelGGL((gs::weigh_many_kernel<T, D, F32>), dim3(a.n_wg), dim3(256), 0, st, a);
    hipLaunchKernelGGL(gs::weigh_join_kernel, dim3(a.n_wg), dim3(256), 0, st, a, gs::Many<D, F32>::kKeys);
}

template <class T, bool F32> void by_head(const gs::WeighArgs &a, uint64_t rows, hipStream_t st)
{
    switch (padded(a.d)) {
    case 64: return by_rows<T, 64, F32>(a, rows, st);
    case 128: return by_rows<T, 128, F32>(a, rows, st);
    default: return by_rows<T, 256, F32>(a, rows, st);
    }
}

} // namespace

extern "C" {

size_t gs_attn_weigh_workspace(const gs_kv_cache *c)
{
    return check_cache(c) ? 0 : kLeftBytes + (size_t)2 * gs::kManyRuns * gs::Many<128, false>::kKeys * sizeof(float);
}

int gs_attn_weigh(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_weigh_args *x, void *stream)
{
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_batch(c, b)) return rc;
    if (!x || layer >= c->n_layers || x->n_heads == 0 || x->n_heads % c->n_kv || x->n_heads > 65535) return GS_ERR_INVALID;
    if (x->type != GS_TYPE_F32 && x->type != c->type) return GS_ERR_UNSUPPORTED;
    if (!std::isfinite(x->scale) || !std::isfinite(x->keep)) return GS_ERR_INVALID;
    if (b->n == 0) return GS_OK;
    if (!x->mass || ((uintptr_t)x->mass & 3u) || x->ld_mass < (size_t)c->ld_table * c->page_size) return GS_ERR_INVALID;
    if (x->ld_mass > (size_t)1 << 40) return GS_ERR_UNSUPPORTED;
    if (b->n_tokens) {
        if (!x->q || ((uintptr_t)x->q & 15u) || x->ld_q % 8 || x->ld_q < (size_t)x->n_heads * c->d) return GS_ERR_INVALID;
        if (!x->lse || ((uintptr_t)x->lse & 3u)) return GS_ERR_INVALID;
    }
    if (!x->ws || ((uintptr_t)x->ws & 15u) || x->ws_bytes < gs_attn_weigh_workspace(c)) return GS_ERR_INVALID;
    // (rows of a sequence are counted in 32 bits)
    if ((uint64_t)b->n_tokens * (x->n_heads / c->n_kv) > 0x7fffffffull) return GS_ERR_UNSUPPORTED;
    const gs_attn_args q = {x->type, x->n_heads, x->q, x->ld_q, nullptr, 0, x->scale, x->window, x->max_q, nullptr, 0};
    gs::WeighArgs a = {};
    (gs::AttnArgs &)a = attn_args(c, layer, b, &q, nullptr);
    const double scale = x->scale == 0.0f ? 1.0 / sqrt((double)c->d) : (double)x->scale, base = (double)a.scale / scale;
    a.sums = x->lse;
    a.mass = x->mass;
    a.ld_mass = x->ld_mass;
    a.keep = x->keep;
    a.base = (float)base;
    a.base_rest = (float)(base - (double)a.base);
    a.left = (gs::Left *)x->ws;
    a.parts = (float *)((char *)x->ws + kLeftBytes);
    const uint64_t rows = (uint64_t)most_tokens(b, &q) * a.group;
    hipStream_t st = (hipStream_t)stream;
    const bool f16 = c->type == GS_TYPE_F16;
    if (x->type == GS_TYPE_F32) f16 ? by_head<_Float16, true>(a, rows, st) : by_head<__bf16, true>(a, rows, st);
    else f16 ? by_head<_Float16, false>(a, rows, st) : by_head<__bf16, false>(a, rows, st);
    return hipGetLastError() == hipSuccess ? GS_OK : GS_ERR_HIP;
}

} // extern "C"
