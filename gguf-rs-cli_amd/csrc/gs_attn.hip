// gs_attn.hip -- attention of new tokens over the paged cache
// (include/gs_attn.h): which kernels of gs_attn.hpp a call takes.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <cmath>
#include <type_traits>

#include "../../include/gs_attn.h"
#include "gs_attn.hpp"

namespace {

template <int D, int R> dim3 join_grid(uint32_t runs)
{
    constexpr int kRows = 256 / (D / 4);        // of a workgroup
    return dim3(runs, (R + kRows - 1) / kRows);
}

template <class TO, int D, int R, bool LSE> int join(const gs::AttnArgs &a, hipStream_t st)
{
    hipLaunchKernelGGL((gs::attn_join_kernel<TO, D, R, LSE>), (join_grid<D, R>(a.n_wg)), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? GS_OK : GS_ERR_HIP;
}

template <class T, int D, int NT, bool F32, bool LSE> void rows_launch(gs::AttnArgs &a, hipStream_t st)
{
    a.n_wg = kCUs * gs::rows_per_cu(D, NT);
    a.lift = gs::kLift<T>;
    if (a.d == D) hipLaunchKernelGGL((gs::attn_rows_kernel<T, D, NT, F32, true, LSE ? gs::kSums : gs::kPlain>), dim3(a.n_wg), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((gs::attn_rows_kernel<T, D, NT, F32, false, LSE ? gs::kSums : gs::kPlain>), dim3(a.n_wg), dim3(256), 0, st, a);
}

template <class T, int D, int NT, bool F32, bool LSE> int rows_call(gs::AttnArgs &a, hipStream_t st)
{
    rows_launch<T, D, NT, F32, LSE>(a, st);
    return join<std::conditional_t<F32, float, T>, D, 16 * NT, LSE>(a, st);
}

template <class T, int D, bool LSE> void chunk_launch(gs::AttnArgs &a, hipStream_t st)
{
    a.n_wg = gs::kChunkRuns;
    a.lift = gs::kChunkLift<T>;
    const dim3 grid(a.n_wg), block(gs::Chunk<D>::kThreads);
    if (a.d == D) hipLaunchKernelGGL((gs::attn_chunk_kernel<T, D, true, LSE ? gs::kSums : gs::kPlain>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((gs::attn_chunk_kernel<T, D, false, LSE ? gs::kSums : gs::kPlain>), grid, block, 0, st, a);
}

// `rows`: the most query rows per head of keys that a sequence may have.
template <class T, int D, bool F32, bool LSE> int by_rows(gs::AttnArgs &a, uint64_t rows, hipStream_t st)
{
    a.min_rows = 0;
    a.max_rows = 0xffffffffu;
    if (rows <= 16) return rows_call<T, D, 1, F32, LSE>(a, st);
    if constexpr (F32) {
        // f32 queries of any number go to the first kernel: its products are
        // three for one, and four chunks of 512 tokens over 8192, 32 / 8 heads
        // of 128, take 1230 us (650 TFLOP/s of products; a bf16 cache: 1130).
        if constexpr (D == 256) return rows_call<T, D, 1, F32, LSE>(a, st);      // (two tiles of rows spill)
        else return rows_call<T, D, 2, F32, LSE>(a, st);
    } else {
        if constexpr (D != 256)
            if (rows <= 32) return rows_call<T, D, 2, F32, LSE>(a, st);
        // Sequences of a few rows go to the first kernel, the others to the
        // second.  (us, first and second, f16; 64 sequences of 8000, 8 heads of
        // keys: of 64, 32 rows: 204, 295; 48: 367, 287; of 128, 32 rows: 362,
        // 384; 48: 713, 425; of 256, 16 rows: 688, 736; 24: 1366, 739.  Four of
        // 4000, where the time is launches and waits: of 128, 16 rows: 23, 25;
        // 32: 30, 26; of 256, 16: 35, 33.)
        constexpr int kFew = D == 256 ? 16 : 32;
        constexpr int R = gs::Chunk<D>::kRows;
        if ((uint64_t)a.n_tokens * a.group == rows * a.n) {     // (all of the same length, or the caller's most is wrong)
            chunk_launch<T, D, LSE>(a, st);
            return join<T, D, R, LSE>(a, st);
        }
        gs::AttnArgs b = a;
        b.cuts = (gs::Cut *)((char *)a.cuts + cuts_bytes());
        b.parts = (float *)((char *)a.parts + few_bytes(D));
        a.max_rows = kFew;
        b.min_rows = kFew + 1;
        rows_launch<T, D, kFew / 16, F32, LSE>(a, st);
        chunk_launch<T, D, LSE>(b, st);
        hipLaunchKernelGGL((gs::attn_join_both_kernel<T, D, kFew, R, LSE>), (join_grid<D, R>(a.n_wg + b.n_wg)), dim3(256), 0, st, a, b);
        return hipGetLastError() == hipSuccess ? GS_OK : GS_ERR_HIP;
    }
}

template <class T, bool F32, bool LSE> int by_head(gs::AttnArgs &a, uint64_t rows, hipStream_t st)
{
    switch (padded(a.d)) {
    case 64: return by_rows<T, 64, F32, LSE>(a, rows, st);
    case 128: return by_rows<T, 128, F32, LSE>(a, rows, st);
    default: return by_rows<T, 256, F32, LSE>(a, rows, st);
    }
}

template <bool LSE> int by_type(const gs_kv_cache *c, const gs_attn_args *x, gs::AttnArgs &a, uint64_t rows, hipStream_t st)
{
    const bool f16 = c->type == GS_TYPE_F16;
    if (x->type == GS_TYPE_F32) return f16 ? by_head<_Float16, true, LSE>(a, rows, st) : by_head<__bf16, true, LSE>(a, rows, st);
    return f16 ? by_head<_Float16, false, LSE>(a, rows, st) : by_head<__bf16, false, LSE>(a, rows, st);
}

} // namespace

extern "C" {

size_t gs_attn_workspace(const gs_kv_cache *c, uint32_t n_heads)
{
    if (check_cache(c) || n_heads == 0 || n_heads % c->n_kv) return 0;
    const int D = padded(c->d);
    return 2 * cuts_bytes() + few_bytes(D) + parts_bytes(gs::kChunkRuns, D == 256 ? gs::Chunk<256>::kRows : gs::Chunk<128>::kRows, D);
}

int gs_attn(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_attn_args *x, void *stream)
{
    return gs_attn_lse(c, layer, b, x, nullptr, stream);
}

int gs_attn_lse(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_attn_args *x, float *lse, void *stream)
{
    if (int rc = check_attn(c, layer, b, x, lse)) return rc;
    if (b->n_tokens == 0) return GS_OK;
    if (!x->ws || ((uintptr_t)x->ws & 15u) || x->ws_bytes < gs_attn_workspace(c, x->n_heads)) return GS_ERR_INVALID;
    gs::AttnArgs a = attn_args(c, layer, b, x, lse);
    a.cuts = (gs::Cut *)x->ws;
    a.parts = (float *)((char *)x->ws + 2 * cuts_bytes());
    const uint64_t rows = (uint64_t)most_tokens(b, x) * a.group;
    hipStream_t st = (hipStream_t)stream;
    // (kernels of their own: those of a call without sums do without the registers and
    // instructions that sums take; us of 4 chunks of 1024 over 4000, 16 / 4 heads of 192,
    // f16: 425, and 451 with one kernel for both)
    return lse ? by_type<true>(c, x, a, rows, st) : by_type<false>(c, x, a, rows, st);
}

} // extern "C"
