// gs_rope.hip -- rotary positions (include/gs_rope.h) and the write of new
// tokens to the paged cache (gs_kv_append, include/gs_cache.h).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <new>
#include <vector>

#include "../../include/gs_cache.h"
#include "gs_cache.hpp"

namespace gs {

constexpr int kRopeThreads = 256;
constexpr int kRopeTokens = 4;          // most tokens of one workgroup

struct RopeArgs {
    // the rotation (rot 0: none)
    const uint64_t *turns;
    int rot, d, half;
    float gain;
    // heads that are turned and go to q_out, then those that go to the cache
    const void *q, *k, *v;
    void *q_out;
    size_t ld_q, ld_out, ld_k, ld_v;
    int n_heads, n_kv;                  // (n_kv 0: no cache)
    int n_tokens;
    const int32_t *pos;                 // or, where null, from the rows:
    const uint32_t *rows, *start, *len, *table;
    uint32_t n, n_rows, ld_table, n_pages;
    int shift;                          // log2 of the page size
    void *kc, *vc;                      // the layer's pages
    // work items: a vector of 8 values, or two that the half layout turns together (in the pair form two values)
    int turned, per_head, per_v;        // items of a head that are turned, all of its items, those of a head of v
    int tokens;                         // of a workgroup
    int first;                          // token of the launch
    uint32_t by_head, by_token, by_v, by_vtoken;   // 2^32 / (per_head, items of a token, per_v, items of v of a token), up
};

// n / d for n d < 2^32, m = ceil(2^32 / d)
__device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t d, uint32_t m) { return d == 1 ? n : __umulhi(n, m); }

// Each value is read once and written once; a token's angles are computed once
// by its workgroup and serve all heads from LDS.  What bounds it is the
// traffic, so neighbouring threads have neighbouring vectors of 8 values (for
// the half layout's turned values two each, rot / 2 apart), and two such items
// at a time.  VEC: the pair form otherwise, for heads, parts or strides that
// are not multiples of the vectors.
// PAST: written past the caches.
// Measured: 12001 x 32 x 96, bf16, 148 MB: 24.6 us, 6.0 TB/s; the new tokens of
// one layer, 4 x 2048 x (32 + 2 x 8) x 128, f16, 201 MB: 34 us, 5.9 TB/s; one
// token 2.3 to 3.1 us of kernel (one that reads a word and ends: 1.3).
template <class TI, class TO, class TC, bool VEC, bool PAST>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a)
{
    constexpr int kItems = 2, kW = VEC ? 8 : 1;
    __shared__ float2 cs[kRopeTokens * 256];
    __shared__ int64_t place[kRopeTokens];      // of a token's slot in a head's pages, in slots; -1: not written
    const int t0 = a.first + blockIdx.x * a.tokens, nt = min(a.tokens, a.n_tokens - t0);
    const int pairs = a.rot >> 1;
    const size_t head = ((size_t)1 << a.shift) * a.d;

    if (a.pos) {
        for (int i = threadIdx.x; i < nt * pairs; i += kRopeThreads) {
            const int t = i / pairs;
            cs[t * 256 + i - t * pairs] = turn_of(a.turns[i - t * pairs], a.pos[t0 + t], a.gain);
        }
    } else {
        // a wave finds the position of its token and the page
        for (int t = threadIdx.x >> 6; t < nt; t += kRopeThreads / 64) {
            const uint32_t token = t0 + t;
            uint32_t i = token, first = token, count = 1;
            if (a.start) {
                i = sequence_of(a.start, a.n, token);
                first = a.start[i];
                count = a.start[i + 1] - first;
            }
            const uint32_t row = a.rows ? a.rows[i] : i;
            int64_t pos = -1;
            if (row < a.n_rows) pos = (int64_t)a.len[row] - count + (token - first);
            if ((threadIdx.x & 63) == 0) {
                int64_t at = -1;
                if (pos >= 0 && (uint64_t)pos < (uint64_t)a.ld_table << a.shift) {
                    const uint32_t page = a.table[(size_t)row * a.ld_table + (pos >> a.shift)];
                    // (head 0 of the page; head h is n_kv pages of one head further)
                    if (page < a.n_pages) at = ((int64_t)page * a.n_kv << a.shift) + (pos & ((1 << a.shift) - 1));
                }
                place[t] = at;
            }
            for (int i = threadIdx.x & 63; i < pairs; i += 64) cs[t * 256 + i] = turn_of(a.turns[i], pos, a.gain);
        }
    }
    __syncthreads();

    // kItems items of a thread at a time: their reads are under way together
    const int heads = a.n_heads + a.n_kv;
    const uint32_t per_token = heads * a.per_head, step = gridDim.y * kRopeThreads;
    for (uint32_t i0 = blockIdx.y * kRopeThreads + threadIdx.x; i0 < nt * per_token; i0 += kItems * step) {
        float u[kItems][kW], w[kItems][kW];
        int p[kItems], q[kItems];
        uint32_t cj[kItems];                // the item's first angle
        TO *yq[kItems];
        TC *yk[kItems];
        bool live[kItems], turned[kItems];
#pragma unroll
        for (int s = 0; s < kItems; s++) {
            const uint32_t i = i0 + s * step;
            live[s] = i < nt * per_token;
            if (!live[s]) continue;
            const uint32_t t = quotient(i, per_token, a.by_token), r = i - t * per_token;
            const uint32_t h = quotient(r, a.per_head, a.by_head), j = r - h * a.per_head;
            const size_t token = t0 + t;
            const bool isq = (int)h < a.n_heads;
            const TI *x = isq ? (const TI *)a.q + token * a.ld_q + (size_t)h * a.d
                              : (const TI *)a.k + token * a.ld_k + (size_t)(h - a.n_heads) * a.d;
            const int64_t at = isq ? 0 : place[t];
            yq[s] = isq ? (TO *)a.q_out + token * a.ld_out + (size_t)h * a.d : nullptr;
            yk[s] = (TC *)a.kc + (h - a.n_heads) * head + at * a.d;
            live[s] = at >= 0;
            if (!live[s]) continue;
            turned[s] = (int)j < a.turned;
            if constexpr (VEC) {
                // one vector of 8, or for pairs of the half layout two
                cj[s] = t * 256 + (a.half ? 8 : 4) * j;
                p[s] = q[s] = turned[s] ? 8 * j : a.rot + 8 * (j - a.turned);
                if (turned[s] && a.half) q[s] += pairs;
                load8(x + p[s], u[s]);
                if (q[s] != p[s]) load8(x + q[s], w[s]);
            } else {
                cj[s] = t * 256 + j;
                p[s] = turned[s] && a.half ? j : 2 * j;
                q[s] = turned[s] && a.half ? j + pairs : 2 * j + 1;
                u[s][0] = (float)x[p[s]];
                w[s][0] = (float)x[q[s]];
            }
        }
#pragma unroll
        for (int s = 0; s < kItems; s++) {
            if (!live[s]) continue;
            const float2 *c = cs + cj[s];
            if (turned[s]) {
                if constexpr (VEC) {
                    if (a.half) {
#pragma unroll
                        for (int e = 0; e < 8; e++) turn_pair(u[s][e], w[s][e], c[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) turn_pair(u[s][2 * e], u[s][2 * e + 1], c[e]);
                    }
                } else turn_pair(u[s][0], w[s][0], c[0]);
            }
            if constexpr (VEC) {
                if (yq[s]) {
                    store8<PAST>(yq[s] + p[s], u[s]);
                    if (q[s] != p[s]) store8<PAST>(yq[s] + q[s], w[s]);
                } else {
                    store8<PAST>(yk[s] + p[s], u[s]);
                    if (q[s] != p[s]) store8<PAST>(yk[s] + q[s], w[s]);
                }
            } else {
                if (yq[s]) { yq[s][p[s]] = (TO)u[s][0]; yq[s][q[s]] = (TO)w[s][0]; }
                else { yk[s][p[s]] = (TC)u[s][0]; yk[s][q[s]] = (TC)w[s][0]; }
            }
        }
    }
    if (a.n_kv == 0) return;
    const uint32_t v_token = a.n_kv * a.per_v;
    for (uint32_t i = blockIdx.y * kRopeThreads + threadIdx.x; i < nt * v_token; i += gridDim.y * kRopeThreads) {
        const uint32_t t = quotient(i, v_token, a.by_vtoken), r = i - t * v_token;
        const uint32_t h = quotient(r, a.per_v, a.by_v), j = r - h * a.per_v;
        if (place[t] < 0) continue;
        const TI *x = (const TI *)a.v + (size_t)(t0 + t) * a.ld_v + (size_t)h * a.d;
        TC *y = (TC *)a.vc + h * head + place[t] * a.d;
        if constexpr (VEC) {
            float u[8];
            load8(x + 8 * j, u);
            store8<PAST>(y + 8 * j, u);
        } else {
            y[2 * j] = (TC)(float)x[2 * j];
            y[2 * j + 1] = (TC)(float)x[2 * j + 1];
        }
    }
}

} // namespace gs

namespace {

using gs::RopeArgs;

uint32_t over(uint32_t d) { return (uint32_t)(((1ull << 32) + d - 1) / d); }

size_t bytes_of(uint32_t type) { return type == GS_TYPE_F32 ? 4 : 2; }

bool vectors(const void *p, size_t ld, uint32_t type) { return ((uintptr_t)p & 15u) == 0 && (ld * bytes_of(type)) % 16 == 0; }

// Calls f with a value of the type.
template <class Fn> int with_type(uint32_t type, Fn f)
{
    switch (type) {
    case GS_TYPE_F32: return f(float());
    case GS_TYPE_F16: return f(_Float16());
    case GS_TYPE_BF16: return f(__bf16());
    default: return GS_ERR_UNSUPPORTED;
    }
}

template <class TI, class TO, class TC>
int launch(RopeArgs &a, bool vec, hipStream_t st)
{
    a.turned = !vec ? a.rot / 2 : a.half ? a.rot / 16 : a.rot / 8;
    a.per_head = a.turned + (vec ? (a.d - a.rot) / 8 : (a.d - a.rot) / 2);
    a.per_v = vec ? a.d / 8 : a.d / 2;
    const uint64_t per_token = (uint64_t)(a.n_heads + a.n_kv) * a.per_head, items = per_token + (uint64_t)a.n_kv * a.per_v;
    if (per_token > 65535 || (uint64_t)a.n_kv * a.per_v > 65535) return GS_ERR_UNSUPPORTED;     // (quotient)
    // One token per workgroup until there are several workgroups per CU, then
    // four: with one, the angles and the places leave most lanes idle.  (us, one
    // and four, bf16: 1024 x 32 x 128 4.7, 6.4; 16384 x 32 x 128 40.6, 41.6; 16384
    // x 8 x 64 16.0, 8.5; 12001 x 32 x 96 28.8, 25.1; 4 x 2048 tokens written,
    // 16 / 2 heads of 64, 20.8, 11.4.)
    // (quotient: values are twice the items of their keys at most, and
    // 4 * 32768 * 32768 = 2^32)
    a.tokens = a.n_tokens >= 4096 && per_token <= 16384 ? gs::kRopeTokens : 1;
    const unsigned blocks = ((unsigned)a.n_tokens + a.tokens - 1) / a.tokens;
    // Few tokens: a token's items are spread over workgroups, each with one
    // round of them; the angles are computed by each.  (One token of 128 heads
    // of 256: 3.0 us, by one workgroup 8.8; of 32 heads of 128 either way 2.6.)
    unsigned y = blocks <= 256 ? (unsigned)((items + gs::kRopeThreads - 1) / gs::kRopeThreads) : 1;
    if (y > 64) y = 64;
    a.by_head = over(a.per_head);
    a.by_token = over((uint32_t)per_token);
    a.by_v = over(a.per_v);
    a.by_vtoken = over(a.n_kv ? a.n_kv * a.per_v : 1);
    const size_t written = (size_t)a.n_tokens * a.d * (a.n_heads * sizeof(TO) + 2 * a.n_kv * sizeof(TC));
    // (a grid has less than 2^32 threads side by side)
    constexpr unsigned kMost = 1u << 23;
    for (unsigned done = 0; done < blocks; done += kMost) {
        a.first = (int)(done * a.tokens);
        const dim3 grid(blocks - done < kMost ? blocks - done : kMost, y), block(gs::kRopeThreads);
        if (!vec) hipLaunchKernelGGL((gs::rope_kernel<TI, TO, TC, false, false>), grid, block, 0, st, a);
        else if (written > kPastCaches) hipLaunchKernelGGL((gs::rope_kernel<TI, TO, TC, true, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((gs::rope_kernel<TI, TO, TC, true, false>), grid, block, 0, st, a);
    }
    return hipGetLastError() == hipSuccess ? GS_OK : GS_ERR_HIP;
}

void set_rope(RopeArgs &a, const gs_rope *r)
{
    a.turns = r ? r->turns : nullptr;
    a.rot = r ? (int)r->rot : 0;
    a.half = r && r->layout == GS_ROPE_HALF;
    a.gain = r ? r->gain : 1.0f;
}

} // namespace

extern "C" {

int gs_rope_create(const gs_rope_params *p, gs_rope **out)
{
    if (!out) return GS_ERR_INVALID;
    *out = nullptr;
    if (!p || p->d == 0 || p->d % 2 || p->rot < 2 || p->rot % 2 || p->rot > p->d) return GS_ERR_INVALID;
    if (p->layout > GS_ROPE_HALF || !(p->base > 1.0) || !std::isfinite(p->base)) return GS_ERR_INVALID;
    if (p->d > 512 || p->scaling > GS_ROPE_YARN) return GS_ERR_UNSUPPORTED;
    const bool yarn = p->scaling == GS_ROPE_YARN;
    if (p->scaling != GS_ROPE_NONE && (!(p->factor >= 1.0) || !std::isfinite(p->factor))) return GS_ERR_INVALID;
    if (!std::isfinite(p->gain) || p->gain < 0.0) return GS_ERR_INVALID;
    const double fast = p->beta_fast == 0.0 ? 32.0 : p->beta_fast, slow = p->beta_slow == 0.0 ? 1.0 : p->beta_slow;
    if (yarn && (p->context == 0 || !(fast > 0.0) || !(slow > 0.0) || !std::isfinite(fast) || !std::isfinite(slow))) return GS_ERR_INVALID;
    const int n = (int)p->rot / 2;
    double low = 0.0, high = 0.0;
    if (yarn) {
        const double two_pi = 2.0 * M_PI, ln = 2.0 * log(p->base);
        low = fmax(floor(p->rot * log(p->context / (two_pi * fast)) / ln), 0.0);
        high = fmin(ceil(p->rot * log(p->context / (two_pi * slow)) / ln), (double)p->rot - 1.0);
    }
    gs_rope *r = new (std::nothrow) gs_rope();
    if (!r) return GS_ERR_NOMEM;
    r->d = p->d; r->rot = p->rot; r->layout = p->layout;
    r->gain = p->gain > 0.0 ? (float)p->gain : yarn ? (float)(0.1 * log(p->factor) + 1.0) : 1.0f;
    uint64_t turns[256];
    for (int i = 0; i < n; i++) {
        // (80-bit: the angle of the farthest position keeps its bits)
        long double f = powl((long double)p->base, -2.0L * i / p->rot) / (2.0L * 3.14159265358979323846264338327950288L);
        if (p->divisors) {
            if (!(p->divisors[i] > 0.0f) || !std::isfinite(p->divisors[i])) { delete r; return GS_ERR_INVALID; }
            f /= p->divisors[i];
        }
        if (p->scaling == GS_ROPE_LINEAR) f /= p->factor;
        if (yarn) {
            const long double y = fmin(fmax((i - low) / fmax(high - low, 0.001), 0.0), 1.0);
            f = f * (1.0L - y) + f / p->factor * y;
        }
        f -= floorl(f);                 // whole turns (a divisor below 1 / (2 pi))
        turns[i] = (uint64_t)(f * 18446744073709551616.0L);
    }
    if (hipGetDevice(&r->device) != hipSuccess) { delete r; return GS_ERR_HIP; }
    if (hipMalloc((void **)&r->turns, n * sizeof(uint64_t)) != hipSuccess) {
        (void)hipGetLastError();
        delete r;
        return GS_ERR_NOMEM;
    }
    if (hipMemcpy(r->turns, turns, n * sizeof(uint64_t), hipMemcpyHostToDevice) != hipSuccess) {
        (void)hipFree(r->turns);
        delete r;
        return GS_ERR_HIP;
    }
    *out = r;
    return GS_OK;
}

int gs_rope_destroy(gs_rope *r)
{
    if (!r) return GS_ERR_INVALID;
    int dev;
    (void)hipGetDevice(&dev);
    (void)hipSetDevice(r->device);
    (void)hipDeviceSynchronize();
    (void)hipFree(r->turns);
    (void)hipSetDevice(dev);
    delete r;
    return GS_OK;
}

int gs_rope_apply(const gs_rope *r, uint32_t type, const void *x, size_t ld_x, void *out, size_t ld_out,
                  size_t n_tokens, uint32_t n_heads, const int32_t *pos, void *stream)
{
    if (!r) return GS_ERR_INVALID;
    if (type != GS_TYPE_F32 && type != GS_TYPE_F16 && type != GS_TYPE_BF16) return GS_ERR_UNSUPPORTED;
    if (n_tokens == 0 || n_heads == 0) return GS_OK;
    if (!x || !out || !pos) return GS_ERR_INVALID;
    if (ld_x < (size_t)n_heads * r->d || ld_out < (size_t)n_heads * r->d) return GS_ERR_INVALID;
    if (x == out && ld_x != ld_out) return GS_ERR_INVALID;
    if (!is_here(r)) return GS_ERR_INVALID;
    if (((uintptr_t)x | (uintptr_t)out) % bytes_of(type)) return GS_ERR_INVALID;
    if (n_tokens > 0x3fffffff) return GS_ERR_UNSUPPORTED;
    RopeArgs a = {};
    set_rope(a, r);
    a.d = (int)r->d;
    a.q = x; a.ld_q = ld_x;
    a.q_out = out; a.ld_out = ld_out;
    a.n_heads = (int)n_heads;
    a.n_tokens = (int)n_tokens;
    a.pos = pos;
    const bool vec = r->rot % (a.half ? 16 : 8) == 0 && r->d % 8 == 0 && vectors(x, ld_x, type) && vectors(out, ld_out, type);
    return with_type(type, [&](auto t) { return launch<decltype(t), decltype(t), _Float16>(a, vec, (hipStream_t)stream); });
}

int gs_kv_append(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_rope *rope, const gs_kv_new *x,
                 void *stream)
{
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_batch(c, b)) return rc;
    if (!x || layer >= c->n_layers) return GS_ERR_INVALID;
    if (rope && (rope->d != c->d || !is_here(rope))) return GS_ERR_INVALID;
    if (x->type != GS_TYPE_F32 && x->type != c->type) return GS_ERR_UNSUPPORTED;
    if (x->q && x->q_out_type != x->type && x->q_out_type != c->type) return GS_ERR_UNSUPPORTED;
    if (b->n_tokens == 0) return GS_OK;
    const size_t kv = (size_t)c->n_kv * c->d, w = bytes_of(x->type);
    if (!x->k || !x->v || x->ld_k < kv || x->ld_v < kv) return GS_ERR_INVALID;
    if (((uintptr_t)x->k | (uintptr_t)x->v | (uintptr_t)x->q) % w) return GS_ERR_INVALID;
    RopeArgs a = {};
    set_rope(a, rope);
    a.d = (int)c->d;
    a.k = x->k; a.ld_k = x->ld_k;
    a.v = x->v; a.ld_v = x->ld_v;
    a.n_kv = (int)c->n_kv;
    bool vec = a.rot % (a.half ? 16 : 8) == 0 && vectors(x->k, x->ld_k, x->type) && vectors(x->v, x->ld_v, x->type);
    if (x->q) {
        const size_t q = (size_t)x->n_heads * c->d;
        if (x->n_heads == 0 || !x->q_out || x->ld_q < q || x->ld_q_out < q) return GS_ERR_INVALID;
        if (x->n_heads > 65535 || (uintptr_t)x->q_out % bytes_of(x->q_out_type)) return GS_ERR_INVALID;
        if (x->q == x->q_out && (x->ld_q != x->ld_q_out || x->type != x->q_out_type)) return GS_ERR_INVALID;
        a.q = x->q; a.ld_q = x->ld_q;
        a.q_out = x->q_out; a.ld_out = x->ld_q_out;
        a.n_heads = (int)x->n_heads;
        vec = vec && vectors(x->q, x->ld_q, x->type) && vectors(x->q_out, x->ld_q_out, x->q_out_type);
    }
    a.n_tokens = (int)b->n_tokens;
    a.rows = b->rows; a.start = b->start; a.len = c->len; a.table = c->table;
    a.n = b->n; a.n_rows = c->rows; a.ld_table = c->ld_table; a.n_pages = c->n_pages;
    a.shift = log2_of(c->page_size);
    const size_t plane = (size_t)c->n_pages * c->n_kv * c->page_size * c->d * 2;
    a.kc = (char *)c->k + layer * plane;
    a.vc = (char *)c->v + layer * plane;
    hipStream_t st = (hipStream_t)stream;
    return with_type(c->type, [&](auto tc) -> int {
        using TC = decltype(tc);
        if constexpr (sizeof(TC) == 4) return GS_ERR_UNSUPPORTED;
        else if (x->type != GS_TYPE_F32) return launch<TC, TC, TC>(a, vec, st);
        else if (x->q && x->q_out_type != GS_TYPE_F32) return launch<float, TC, TC>(a, vec, st);
        else return launch<float, float, TC>(a, vec, st);
    });
}

} // extern "C"
