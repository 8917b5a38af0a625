// How the experts' products are cut into tiles: what expert_kernel derives from the counts alone.  Shared with the host,
// where only the tests ask for it (mc_ep_debug_expert_plan): which tile shapes a call runs is decided by the prices here.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

namespace mcep {

// The plans a block can choose from: an expert's rows spread over as few tiles as give none more than 32 * blocks rows,
// tiles of 256 or (the last four; not for fp8 gate_up, whose scale groups want 256) 128 weight rows.
constexpr int kPlans = 12, kWidePlans = 8;
__host__ __device__ __forceinline__ bool plan_wide(int plan) { return plan < kWidePlans; }
__host__ __device__ __forceinline__ int plan_blocks(int plan) { return plan_wide(plan) ? plan + 1 : plan + 1 - kWidePlans; }
__host__ __device__ __forceinline__ int plan_columns(int plan, bool gate_up) { return (plan_wide(plan) ? 256 : 128) / (gate_up ? 2 : 1); }

constexpr int kStep = 128;             // bytes of a row per K step
__host__ __device__ __forceinline__ int steps_of(int row_bytes) { return (row_bytes + kStep - 1) / kStep; }

// What a K step of a tile costs, in ns, by its blocks of 32 rows, and a tile besides (fitted to calls of every plan; the plan
// that comes out is within 3 % of the best of the twelve for 4 to 256 experts of 24 to 512 rows, where the best is anything
// from 32 x 256 and 64 x 128 to 256 x 256 and the worst takes 1.5 to 4 times as long).
__host__ __device__ __forceinline__ int step_cost(bool wide, int blocks) { return wide ? 350 + 150 * blocks : 250 + 90 * blocks; }
constexpr int kTileCost = 4000;

// The tiles that n rows are spread over: (n + most - 1) / most, by x * divisor(most) >> 32, exact for the x there are.
__host__ __device__ __forceinline__ uint32_t divisor(int most) { return 0xffffffffu / (uint32_t)most + 1; }
__host__ __device__ __forceinline__ int row_tiles(int n, int most, uint32_t divisor_of_most) {
    return (int)(((uint64_t)(uint32_t)(n + most - 1) * divisor_of_most) >> 32);
}

// 1 / x for a price: the hardware's own where the kernel asks.
__host__ __device__ __forceinline__ float price_reciprocal(float x) {
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_rcpf(x);
#else
    return 1.0f / x;
#endif
}

// A K step of all of an expert's `down` tiles of n rows together.
__host__ __device__ __forceinline__ int rows_cost(int n, int down, bool wide) {
    return n > 0 ? down * step_cost(wide, (int)ceilf((float)n * price_reciprocal((float)down) * 0.03125f)) : 0;
}

// A call of `tiles` tiles of rows, whose K steps cost `cost` together (past 31 bits from 1.4 million tiles on), by `across`
// tiles of columns on `blocks` blocks: rounds of the blocks, each as long as a tile of middling cost.
__host__ __device__ __forceinline__ float plan_time(int tiles, uint64_t cost, int across, int blocks, int steps) {
    const float rounds = ceilf((float)tiles * (float)across / (float)blocks);
    return rounds * ((float)cost * price_reciprocal((float)(tiles > 0 ? tiles : 1)) * steps + kTileCost);
}

// Few rows (all experts' are one tile each, and at most 32): the weights are read once and are the whole cost, and they can
// be read without a place in the caches.  That pays wherever they are not in the last-level cache (256 MiB) already - a
// product of 50 to 450 MiB after others' weights: 4 to 13 % (8 experts of fp8 7168 x 2048, a row each: 224 + 112 MiB, 56 + 25 us
// kept, 52 + 23 not; 28 MiB the same, 45) - and costs where they are: up to 250 MiB read again at once 38 us kept and 52
// not, 12 + 7 for 20 MB (11 + 7), beyond what the cache holds 66 and 59.  Weights that are read again before 256 MiB of
// others are those of a program of few, small layers: a product of 64 MiB or more is a layer or two of it at most.  (Tiles
// of 128 weight rows have no such form: they are chosen for products of too few tiles to be bound by the reads.)
constexpr int64_t kStreamed = 64 << 20;
__host__ __device__ __forceinline__ bool streamed(int tiles, int experts, int across, int weight_rows, int row_bytes) {
    return tiles == experts && (int64_t)tiles * across * weight_rows * row_bytes >= kStreamed;
}

}  // namespace mcep
