// gfx950 kernels of the paged-cache operators, a code object of their own
// (hipcc --genco --offload-arch=gfx950): the decode step's kernels in the
// other one keep their places in the instruction caches.
#include "device/paged.h"
#include "device/paged_attn.h"

using namespace ifr;

extern "C" __global__ void __launch_bounds__(PG_PLAN_THREADS) paged_plan_k(PagedPlanArgs a) { paged_plan_body(a); }
extern "C" __global__ void __launch_bounds__(256) paged_rows_k(PagedPlanArgs a) { paged_rows_body(a); }
extern "C" __global__ void __launch_bounds__(PG_ROPE_THREADS) paged_rope_k(PagedRopeArgs a) { paged_rope_body(a); }

// (two waves per SIMD: the registers of the next key tile's rows)
#define PA_ROWS16(NAME, HSP, T)                                                                           \
    extern "C" __global__ void __launch_bounds__(64 * PAD_WAVES) __attribute__((amdgpu_waves_per_eu(2, 8))) \
    paged_rows16_##NAME##_h##HSP(PagedAttnArgs a) {                                                       \
        pa_rows16_body<HSP, T, 1>(a);                                                                       \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) paged_merge16_##NAME##_h##HSP(PagedAttnArgs a) {    \
        pa_merge_body<HSP, T, 16 * PAD_NU<HSP, T>, 1>(a);                                                 \
    }

PA_ROWS16(f16, 64, PA_H)
PA_ROWS16(f16, 128, PA_H)
PA_ROWS16(mixed, 64, PA_M)
PA_ROWS16(mixed, 128, PA_M)
PA_ROWS16(f32, 64, PA_S)
PA_ROWS16(f32, 128, PA_S)

// f32 rows of chunks: two blocks of 16 rows (their merges are those of one)
extern "C" __global__ void __launch_bounds__(64 * PAD_WAVES) __attribute__((amdgpu_waves_per_eu(2, 8)))
paged_rows32_f32_h64(PagedAttnArgs a) { pa_rows16_body<64, PA_S, 2>(a); }
extern "C" __global__ void __launch_bounds__(64 * PAD_WAVES) __attribute__((amdgpu_waves_per_eu(2, 8)))
paged_rows32_f32_h128(PagedAttnArgs a) { pa_rows16_body<128, PA_S, 2>(a); }

#define PA_TILE(NAME, HSP, T, WPE)                                                                             \
    extern "C" __global__ void __launch_bounds__(64 * PAT_WAVES) __attribute__((amdgpu_waves_per_eu(WPE, 8))) \
    paged_tile_##NAME##_h##HSP(PagedAttnArgs a) {                                                           \
        pa_tile_body<HSP, T>(a);                                                                            \
    }                                                                                                       \
    extern "C" __global__ void __launch_bounds__(256) paged_merge128_##NAME##_h##HSP(PagedAttnArgs a) {      \
        pa_merge_body<HSP, T, PAT_KT, 4>(a);                                                                \
    }

PA_TILE(f16, 64, PA_H, 3)
PA_TILE(f16, 128, PA_H, 2)
PA_TILE(mixed, 64, PA_M, 2)
PA_TILE(mixed, 128, PA_M, 2)
