// gs_weigh.hip -- the weight that cached tokens get from the newest ones
// (gs_attn_weigh, include/gs_attn.h).
//
// With the logarithms of the softmax's sums at hand a weight is one
// exponential of its own score, so keys can be taken in any order and need no
// maximum: a wave takes 32 keys of a sequence, goes through the heads and the
// query rows that see them, and adds their weights up in registers.  Each
// token's sum is made by one wave, in one order.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "gs_attn.hpp"

namespace gs {

constexpr int kKeys = 32;               // of a wave

struct WeighArgs {
    AttnArgs a;
    const float *lse;                   // [n_tokens][n_kv group]
    float *mass;                        // [n_rows][ld_mass]
    size_t ld_mass;
    float keep, scale;                  // scale: of the scores
};

// The keys of a sequence whose weights change: all of its tokens where they are
// scaled, else those that its new tokens see.
struct Keys {
    uint32_t lo, hi, tile0, tiles;
    __device__ __forceinline__ Keys(const WeighArgs &x, const Seq &s)
    {
        const int64_t p0 = (int64_t)s.len - s.nq;
        hi = s.len;
        lo = x.keep != 1.0f ? 0 : s.nq ? (uint32_t)min((int64_t)s.len, max((int64_t)0, p0 + 1 - (int64_t)x.a.window)) : s.len;
        tile0 = lo / kKeys;
        tiles = hi > lo ? (hi + kKeys - 1) / kKeys - tile0 : 0;
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

template <class T, int D, bool F32>
__global__ void __launch_bounds__(256) weigh_kernel(const WeighArgs x)
{
    constexpr int KS = D / 32, NP = F32 ? 3 : 1;
    typedef typename Vec<T>::v8 v8;
    const AttnArgs &a = x.a;
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const uint32_t w = uniform(threadIdx.x >> 6);
    const uint32_t page = 1u << a.shift, d = a.d;
    const size_t head = (size_t)d << a.shift;
    // wave `item` of the call takes tiles item, item + waves, ..
    const uint64_t waves = (uint64_t)gridDim.x * 4;
    uint64_t item = (uint64_t)blockIdx.x * 4 + w, before = 0;
    for (uint32_t i = 0; i < a.n; i++) {
        const Seq s = uniform(work_of<Seq>(a, i));
        const Keys keys(x, s);
        if (item >= before + keys.tiles) { before += keys.tiles; continue; }
        const bool mine = is_first(a, i);
        const uint32_t *table = a.table + (size_t)min(s.row, a.n_rows - 1) * a.ld_table;
        const int64_t base = (int64_t)s.len - s.nq;
        for (; item < before + keys.tiles; item += waves) {
            if (!mine) continue;
            const uint32_t key0 = (keys.tile0 + (uint32_t)(item - before)) * kKeys;
            // rows that see one of the keys
            const int64_t t0 = max((int64_t)0, (int64_t)key0 - base), t1 = min((int64_t)s.nq, (int64_t)key0 + kKeys - 1 + (int64_t)a.window - base);
            const uint32_t r0 = (uint32_t)min(t0, (int64_t)s.nq) * a.group, r1 = t1 > t0 ? (uint32_t)t1 * a.group : 0;
            uint32_t id[2];
#pragma unroll
            for (int y = 0; y < 2; y++) id[y] = min(table[min(key0 + 16 * y + m, s.len - 1) >> a.shift], a.n_pages - 1);
            float sum[2][4] = {};
            for (uint32_t kvh = 0; kvh < a.n_kv && r0 < r1; kvh++) {
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
                for (uint32_t r = r0; r < r1; r += 16) {
                    const uint32_t rr = min(r + m, r1 - 1), tok = rr / a.group, h = kvh * a.group + (rr - tok * a.group);
                    const size_t at = (size_t)(s.first + tok) * a.ld_q + (size_t)h * d;
                    const float lse = x.lse[(size_t)(s.first + tok) * a.n_kv * a.group + h];
                    const int64_t pos = r + m < r1 ? base + tok : -1;
                    v8 qf[NP][KS];
                    float unscale = x.scale;
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
                            float score = z[y][e] * unscale;
                            if constexpr (F32)
                                if (sees && score != score) {       // an infinity met the parts of a query: once more, without
                                    const uint32_t p = min(table[(uint32_t)key >> a.shift], a.n_pages - 1);
                                    const T *row = (const T *)a.k + ((size_t)p * a.n_kv + kvh) * head + (size_t)((uint32_t)key & (page - 1)) * d;
                                    score = 0.0f;
                                    for (uint32_t c = 0; c < d; c++) score += ((const float *)a.q)[at + c] * (float)row[c];
                                    score *= x.scale;
                                }
                            const float wt = __builtin_amdgcn_exp2f((score - lse) * (float)M_LOG2E);
                            sum[y][e] += sees ? wt : 0.0f;
                        }
                }
            }
#pragma unroll
            for (int y = 0; y < 2; y++)
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) sum[y][e] += __shfl_xor(sum[y][e], o);
            if (m != 0) continue;
            float *mass = x.mass + s.row * x.ld_mass;
#pragma unroll
            for (int y = 0; y < 2; y++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t key = key0 + 16 * y + 4 * g + e;
                    if (key < keys.lo || key >= keys.hi) continue;
                    mass[key] = x.keep == 0.0f ? sum[y][e] : x.keep * mass[key] + sum[y][e];
                }
        }
        before += keys.tiles;
    }
}

} // namespace gs

namespace {

template <class T, bool F32> void launch(const gs::WeighArgs &x, hipStream_t st)
{
    const dim3 grid(1024), block(256);
    switch (padded(x.a.d)) {
    case 64: hipLaunchKernelGGL((gs::weigh_kernel<T, 64, F32>), grid, block, 0, st, x); break;
    case 128: hipLaunchKernelGGL((gs::weigh_kernel<T, 128, F32>), grid, block, 0, st, x); break;
    default: hipLaunchKernelGGL((gs::weigh_kernel<T, 256, F32>), grid, block, 0, st, x); break;
    }
}

} // namespace

extern "C" {

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
    // (rows of a sequence are counted in 32 bits)
    if ((uint64_t)b->n_tokens * (x->n_heads / c->n_kv) > 0x7fffffffull) return GS_ERR_UNSUPPORTED;
    const gs_attn_args q = {x->type, x->n_heads, x->q, x->ld_q, nullptr, 0, x->scale, x->window, x->max_q, nullptr, 0};
    gs::WeighArgs w = {};
    w.a = attn_args(c, layer, b, &q, nullptr);
    w.lse = x->lse;
    w.mass = x->mass;
    w.ld_mass = x->ld_mass;
    w.keep = x->keep;
    w.scale = x->scale == 0.0f ? (float)(1.0 / sqrt((double)c->d)) : x->scale;
    hipStream_t st = (hipStream_t)stream;
    const bool f16 = c->type == GS_TYPE_F16;
    if (x->type == GS_TYPE_F32) f16 ? launch<_Float16, true>(w, st) : launch<__bf16, true>(w, st);
    else f16 ? launch<_Float16, false>(w, st) : launch<__bf16, false>(w, st);
    return hipGetLastError() == hipSuccess ? GS_OK : GS_ERR_HIP;
}

} // extern "C"
