// gs_cache.hpp -- what the kernels of the paged cache share: value types, a
// row's sequence in a call, and the host's check of a cache.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/gs_cache.h"

// The plan of gs_rope_create (include/gs_rope.h).
struct gs_rope {
    uint32_t d, rot, layout;
    float gain;
    int device;
    uint64_t *turns;        // [rot / 2] 2^64 times the turns per position, whole turns dropped
};

namespace gs {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

// 8 consecutive values as f32; the addresses are 16-byte aligned.
__device__ __forceinline__ void load8(const float *p, float (&x)[8])
{
    const f4v a = *(const f4v *)p, b = *(const f4v *)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; i++) { x[i] = a[i]; x[4 + i] = b[i]; }
}
template <class T> __device__ __forceinline__ void load8(const T *p, float (&x)[8])
{
    typedef T v8 __attribute__((ext_vector_type(8)));
    const v8 a = *(const v8 *)p;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)a[i];
}
// A vector's write; PAST: around the caches, for more than they hold.
template <bool PAST, class V> __device__ __forceinline__ void store(V *p, V x)
{
    if constexpr (PAST) __builtin_nontemporal_store(x, p);
    else *p = x;
}
template <bool PAST> __device__ __forceinline__ void store8(float *p, const float (&x)[8])
{
    store<PAST>((f4v *)p, f4v{x[0], x[1], x[2], x[3]});
    store<PAST>((f4v *)(p + 4), f4v{x[4], x[5], x[6], x[7]});
}
// (rounded to nearest, ties to even)
template <bool PAST, class T> __device__ __forceinline__ void store8(T *p, const float (&x)[8])
{
    typedef T v8 __attribute__((ext_vector_type(8)));
    v8 a;
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = (T)x[i];
    store<PAST>((v8 *)p, a);
}

// cos and sin of a pair's angle at position pos, times gain.  The product
// modulo 2^64 is the fraction of a turn, exact to pos 2^-65; as a signed
// number it lies in [-1/2, 1/2) and rounds to f32 with a relative error of
// 2^-24, so small angles keep all their bits.
__device__ __forceinline__ float2 turn_of(uint64_t turns, int64_t pos, float gain)
{
    const int64_t part = (int64_t)(turns * (uint64_t)pos);
    float s, c;
    sincospif((float)part * 0x1p-63f, &s, &c);
    return make_float2(c * gain, s * gain);
}

// (a, b) turned: the products are rounded once each way, in f32.
__device__ __forceinline__ void turn_pair(float &a, float &b, float2 cs)
{
    const float x = a;
    a = fmaf(x, cs.x, -(b * cs.y));
    b = fmaf(b, cs.x, x * cs.y);
}

// The sequence of a token, found by a wave: how many sequences end at or
// before it.  start: [n + 1]
__device__ __forceinline__ uint32_t sequence_of(const uint32_t *start, uint32_t n, uint32_t token)
{
    const uint32_t lane = threadIdx.x & 63;
    uint32_t k = 0;
    for (uint32_t j = 0; j < n; j += 64)
        k += __popcll(__ballot(j + lane < n && start[j + lane + 1] <= token));
    return k < n ? k : n - 1;
}

} // namespace gs

namespace {

// The sizes that every call on a cache relies on.
inline int check_cache(const gs_kv_cache *c)
{
    if (!c || !c->k || !c->v || !c->table || !c->len || !c->ref) return GS_ERR_INVALID;
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15u) return GS_ERR_INVALID;
    if (c->n_layers == 0 || c->n_pages == 0 || c->n_kv == 0 || c->rows == 0 || c->ld_table == 0 || c->d == 0) return GS_ERR_INVALID;
    if (c->type != GS_TYPE_F16 && c->type != GS_TYPE_BF16) return GS_ERR_UNSUPPORTED;
    if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return GS_ERR_UNSUPPORTED;
    if (c->d % 8 || c->d > GS_KV_MAX_HEAD) return GS_ERR_UNSUPPORTED;
    if ((uint64_t)c->ld_table * c->page_size > 1ull << 30) return GS_ERR_UNSUPPORTED;     // (positions are added to in 32 bits)
    if (c->n_kv > 4096 || c->n_layers > 65535 || c->n_pages > 0x7fffffffu || c->rows > 0x7fffffffu) return GS_ERR_UNSUPPORTED;
    return GS_OK;
}

// A plan's turns are memory of the device it was made on.
inline bool is_here(const gs_rope *r)
{
    int device;
    return hipGetDevice(&device) == hipSuccess && device == r->device;
}

inline int check_batch(const gs_kv_cache *c, const gs_kv_batch *b)
{
    if (!b) return GS_ERR_INVALID;
    if (!b->start && b->n_tokens != b->n) return GS_ERR_INVALID;
    if (b->n > 65536 || b->n_tokens > 0x7fffffffu) return GS_ERR_UNSUPPORTED;
    if (b->n == 0 && b->n_tokens) return GS_ERR_INVALID;
    if (!b->rows && b->n > c->rows) return GS_ERR_INVALID;
    return GS_OK;
}

// Calls that write more than this write past the caches: the L2s of the eight
// XCDs hold 32 MB together.  (us per call, written the usual way and past:
// 12001 x 32 x 96 bf16 turned, 74 MB written: 34.5, 25.4; 256 rows forked
// from 16, 340 MB: 185, 113; 4 x 2048 tokens of a layer, f16, 101 MB: 46.5,
// 42.0.  Fewer bytes are read again soon, by the attention, from L2.)
constexpr size_t kPastCaches = (size_t)32 << 20;

inline int log2_of(uint32_t x)
{
    int s = 0;
    while ((1u << s) < x) s++;
    return s;
}

} // namespace
