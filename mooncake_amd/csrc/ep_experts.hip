// The experts between dispatch and combine: two products per local expert over the packed layout,
//   act = silu(x Wg^T) * (x Wu^T)      out = act Wd^T
// for the first packed_recv_count[e] rows of expert e, x as dispatch leaves it (bf16, or fp8 e4m3 with a scale per
// 128 elements stored column-major), and the entry points mc_ep_expert_gate_up and mc_ep_expert_down around them.
//
// How the work is cut.  The counts are only known on the GPU, so one block per CU walks a list of tiles that
// every block derives from the counts by itself (no host round trip, no work list in memory).  A tile is up to BM rows of
// one expert by BN rows of its weights.  An expert's rows are spread evenly over its tiles (140 rows and BM = 128: two
// tiles of 70 rows, run in the shape for 96).  The list is cut into eight consecutive parts, one per XCD, with
// the tiles that share weights next to each other: they run at the same time behind one L2.
//
// Operands.  Both are K-contiguous.  A K step is 128 bytes of every row (64 bf16 or 128 fp8), loaded straight into
// LDS 16 bytes a lane; the 16-byte chunks of a row are stored at chunk ^ (row & 7), so that the 16 rows a matrix
// instruction reads lie in different banks.  Rows past the count, columns past the weights and a last K step that is
// not full are zeros by the buffer descriptor's range check: nothing out of range is read.
// The weights are the matrix instructions' first operand and the tokens the second: a lane then holds results of one
// token, for weight rows that this kernel is free to choose.  It takes them so that a lane's results are consecutive
// columns (wide stores) and, for the first product, gate and up of the same columns (SwiGLU without an exchange).
//
// fp8: a 16x16x128 instruction is exactly one scale group of the payload and one of the weights' blocks, so its result
// starts from zero and enters the 32-bit sums times (row scale * block scale).  Inside, the instruction takes the products of
// eight consecutive elements together and cuts each off 2^-13 below the largest of the eight; from eight to eight, and from
// group to group, sums have 32 bits.  (The other fp8 instructions do the same: there is no wider fp8 product.)
// Between the products the activations are rounded to the payload's type (bf16, or fp8 with a scale per 128): that is what the
// second product's matrix instructions take, and half or a quarter of the traffic of 32 bits.
//
// What bounds it, and what it measured (both products, weights not in the caches; matrix units busy by the counters):
//   8 experts of 4096 x 8192, 14700 rows, bf16: the matrix units, busy 72-75 % of the time at the 1.5 GHz that the card
//     holds under them: 2.38-2.49 ms = 1190-1250 TFLOP/s (the library's product of 16384^3: 1539);
//   8 experts of 7168 x 2048, 15000 rows, skewed, fp8: matrix units busy 50-56 %, 1.7 GHz: 646-683 us = 1940-2050 TFLOP/s
//     (library 3139, without block scales).  A step has the loads, LDS reads, barrier and matrix cycles (2.0 thousand) of a
//     step in bf16 and takes 3.7 thousand cycles where that takes 2.7: its vector instructions are 1.4 thousand more, of
//     which the rest would be what the matrix instructions do not cover;
//   8 experts of 4096 x 2048, 256 rows each, bf16: every weight is read once, at 2.8 TB/s (3.2 for 128 such experts), and the
//     matrix units are busy 40 %: neither is near its limit, waves wait 42 % of their time (27 % in the large calls) for a
//     step's loads and barrier with one step in flight behind the one that is multiplied.  152-157 us;
//   8 experts of 7168 x 2048, 128 rows each, fp8: the same, 102 us = 3.7 TB/s; 256 such experts at once 2.34-2.38 ms = 4.7
//     TB/s;
//   8 of 256 such experts with a row each: HBM, 76-78 us = 4.6 TB/s (the first product is 128 tiles, half the CUs).
// A call of few tiles besides spends 3 to 4 us on reading the counts and on the first fetch of its code.
#include "../../include/mooncake_ep_hip.h"

#include <hip/hip_runtime.h>

#include <string>
#include <type_traits>

#include "ep_debug.h"
#include "ep_expert_plan.h"
#include "ep_operators.h"

namespace mcep {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr int kMaxLocalExperts = 2048;
constexpr int kXCDs = 8;
constexpr int kMaxGroups = 256;        // scale groups of a row: fp8 rows of at most 32768

struct ExpertArgs {
    const char* x;          // [L, RM, K]
    const float* xs;        // [L, K/128, RM], fp8 only
    const int32_t* count;   // [L]
    const char* w;          // gate_up: [L, 2N, K], gate rows first; down: [L, N, K]
    const float* ws;        // a scale per 128 x 128 block of w, fp8 only
    char* out;              // [L, RM, N]: gate_up bf16 or fp8, down bf16
    float* outs;            // gate_up in fp8: [L, N/128, RM]
    int L, RM, N;
    int Kb;                 // bytes of a row of x and of w
};



// The buffer descriptor of `bytes` bytes at p: loads past them give zeros.
__device__ __forceinline__ v4i span(const char* p, int bytes) {
    const uint64_t at = (uint64_t)p;
    return v4i{(int)(uint32_t)at, (int)(at >> 32), bytes, 0x00027000};
}

// The address of a __shared__ object inside the block's LDS.
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(const lds_void*)p; }

// 16 (4) bytes a lane from r + offset into consecutive LDS addresses from `lds` (the same in all lanes) on.  Written out because the
// compiler, which cannot tell the stages apart, makes every later LDS read wait for all such loads; nothing is returned in
// registers, and the reads wait for the count of loads they need (vmcnt) and for the barrier.  (m0 is a reserved register: it
// can't be listed as overwritten, and the compiler keeps nothing in it.)
__device__ __forceinline__ void load_to_lds16(v4i r, uint32_t lds, int offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(r) : "memory");
}
// (the same, for what is read once: not kept in L2 in place of what is read again)
__device__ __forceinline__ void stream_to_lds16(v4i r, uint32_t lds, int offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(lds), "v"(offset), "s"(r) : "memory");
}
__device__ __forceinline__ void load_to_lds4(v4i r, uint32_t lds, int offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(r) : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    v2bf v;
    v[0] = (__bf16)a;
    v[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, v);
}

// g / (1 + e^-g) * u with the hardware's exponential and reciprocal, within (8 + |g|) 2^-23 of itself: the rounding of the
// exponential's argument grows with g (for gates below -87.33, whose quotient is less than the smallest normal number, zero).
// The result is rounded to bf16 or fp8, 2^-8 or 2^-4 of itself.
__device__ __forceinline__ float swiglu(float g, float u) {
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504f)) * u;
}

// A tile's shape: 32 * BLOCKS rows by BN weight rows over 2 x 4 waves, 128 bytes of K a step, STAGES steps in LDS.
// ONCE: nothing else reads its weights (see kStreamed).
template <bool FP8_, bool GATE_UP_, int BLOCKS_, int BN_, bool ONCE_ = false>
struct Config {
    static constexpr bool FP8 = FP8_, GATE_UP = GATE_UP_, ONCE = ONCE_;
    static constexpr int BLOCKS = BLOCKS_, BM = 32 * BLOCKS, BN = BN_, WN = 4;
    static constexpr int STAGES = BN < 256 ? 4 : BLOCKS <= 4 ? 3 : 2;
    static constexpr int LDS_ROWS = (BM + 63) / 64 * 64;           // what whole loads by all waves fill
    static constexpr int WAVE_M = BM / 2, WAVE_N = BN / WN;
    static constexpr int MT = WAVE_M / 16, NT = WAVE_N / 16;
    static constexpr int COLUMNS = GATE_UP ? BN / 2 : BN;          // output columns of a tile
    static constexpr int LANE_COLUMNS = GATE_UP ? NT * 2 : NT * 4;   // consecutive ones in a lane
    static constexpr int LOADS_A = LDS_ROWS / 64, LOADS_B = BN / 64;   // of 1 KiB, per wave and step
    static constexpr int LOADS = LOADS_A + LOADS_B + (FP8 ? 1 : 0);
    static constexpr int STAGE_BYTES = (LDS_ROWS + BN) * kStep + (FP8 ? LDS_ROWS * 4 : 0);
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES + (FP8 && GATE_UP ? WN * BM * 4 : 0);   // last: WN waves' largest activations
    static constexpr int AHEAD = MT < 2 || (FP8 && MT >= 8) ? 1 : 2;               // (eight: for the registers)
    static constexpr int LAG = NT < 3 ? NT : 3;
    static constexpr int PER_MT = FP8 ? NT : 2 * NT;                // matrix instructions of 16 rows
};
constexpr int kScaleBytes = 2 * (2 * kMaxGroups + 4) * 4;          // the weights' scales of two tiles
constexpr int kLdsBytes = 3 * (128 + 256) * kStep + 3 * 128 * 4 + 4 * 128 * 4;   // the largest LDS_BYTES

// blocks of 32 rows
__device__ __forceinline__ int blocks_of(int rows) { return (rows + 31) / 32; }

// rows m0 .. m0 + rows of expert e by output columns n0 .. n0 + COLUMNS; rows == 0: none
struct Tile {
    int e, m0, rows, n0;
};

// The tiles of one shape that follow each other on a block's list, from `tile` on: what a tile begins with is loaded while
// the one before it ends.  `next_of` gives the block's next tile; returns the first of another shape.
template <class C, class Next>
__device__ __forceinline__ Tile run_tiles(const ExpertArgs& a, Tile tile, const Next& next_of, char* smem, float* scales_lds) {
    static_assert(C::LDS_BYTES <= kLdsBytes, "");
    float* amax_lds = (float*)(smem + C::STAGES * C::STAGE_BYTES);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / C::WN, wn = wave % C::WN;
    const int quarter = lane >> 4, l16 = lane & 15;
    const int Kb = a.Kb;
    const int steps = steps_of(Kb);
    const int groups = Kb / kStep;                 // scale groups of a row (fp8: Kb is whole steps)

    // --- addresses of the loads: row of the tile = load * 64 + wave * 8 + lane / 8, 16-byte chunk (lane & 7) ^ (row & 7)
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    const int off_a = (wave * 8 + (lane >> 3)) * Kb + chunk;
    // which weight row is row r of the tile: see LANE_COLUMNS; from load to load 64 rows further, which is so many output columns
    int off_b;
    {
        const int r = wave * 8 + (lane >> 3), w = r / C::WAVE_N, nt = (r % C::WAVE_N) / 16, q = (r % 16) / 4, j = r % 4;
        off_b = (C::GATE_UP ? (j & 1) * a.N + w * (C::WAVE_N / 2) + q * (C::NT * 2) + nt * 2 + (j >> 1)
                            : w * C::WAVE_N + q * (C::NT * 4) + nt * 4 + j) * Kb + chunk;
    }
    constexpr int FURTHER = C::GATE_UP ? 32 : 64;
    // the rows' scales: 64 a load, by every wave (one of the places, so that all waves have as many loads under way)
    const int place_s = (wave % C::LOADS_A) * 64;

    struct Source {
        const char *a, *b;
        const float *s, *w;
        int left_a, left_b, rows;
    };
    const auto source_of = [&](const Tile& t) {
        Source o;
        o.a = a.x + ((int64_t)t.e * a.RM + t.m0) * Kb;
        o.b = a.w + ((int64_t)t.e * (C::GATE_UP ? 2 : 1) * a.N + t.n0) * Kb;
        o.left_a = t.rows * Kb;
        o.left_b = ((C::GATE_UP ? 2 : 1) * a.N - t.n0) * Kb;
        o.rows = t.rows;
        if (C::FP8) {
            o.s = a.xs + (int64_t)t.e * groups * a.RM + t.m0;
            // the scales of the weights' blocks: gate and up of the tile's columns, or its two halves (even and odd waves)
            const int blocks = a.N / 128, half = wave & 1;
            const int b = t.n0 / 128 + (C::GATE_UP ? half * blocks : half);
            o.w = a.ws + ((int64_t)t.e * (C::GATE_UP ? 2 : 1) * blocks + (C::GATE_UP || b < blocks ? b : blocks - 1)) * groups;
        }
        return o;
    };
    // load i of step k into a stage: the rows, the weights, the scales
    const auto load = [&](const Source& o, int i, int k, int stage) {
        const uint32_t st = lds_address(smem) + stage * C::STAGE_BYTES;
        const int done = k * kStep;
        // a last step that is not full: the chunks past the row's end come from out of range
        const int cut = !C::FP8 && Kb - done < kStep && chunk >= Kb - done ? (int)0x80000000 : 0;
        if (i < C::LOADS_A) {
            const int at = done + i * 64 * Kb;
            load_to_lds16(span(o.a + at, max(o.left_a - at, 0)), st + (i * 64 + wave * 8) * kStep, off_a | cut);
        } else if (i < C::LOADS_A + C::LOADS_B) {
            const int l = i - C::LOADS_A, at = done + l * FURTHER * Kb;
            const v4i from = span(o.b + at, max(o.left_b - at, 0));
            const uint32_t to = st + (C::LDS_ROWS + l * 64 + wave * 8) * kStep;
            if constexpr (C::ONCE) stream_to_lds16(from, to, off_b | cut);
            else load_to_lds16(from, to, off_b | cut);
        } else {
            load_to_lds4(span((const char*)(o.s + (int64_t)k * a.RM), o.rows * 4),
                         st + (C::LDS_ROWS + C::BN) * kStep + place_s * 4, (place_s + lane) * 4);
        }
    };
    // all block scales of a tile, in front of its first step
    const auto load_wscales = [&](const Source& o, int parity) {
        load_to_lds4(span((const char*)o.w, groups * 4),
                     lds_address(scales_lds) + (parity * (2 * kMaxGroups + 4) + (wave & 1) * kMaxGroups + (wave >> 1) * 64) * 4,
                     ((wave >> 1) * 64 + lane) * 4);
    };

    // --- where the lane's operands lie in a stage (the second part of a row's 128 bytes: ^ 64)
    const int read_a = (wm * C::WAVE_M + l16) * kStep + ((quarter ^ (lane & 7)) << 4);
    const int read_b = (C::LDS_ROWS + wn * C::WAVE_N + l16) * kStep + ((quarter ^ (lane & 7)) << 4);
    const int read_s = (C::LDS_ROWS + C::BN) * kStep + (wm * C::WAVE_M + l16) * 4;
    const int my_half = C::GATE_UP ? 0 : (wn * C::WAVE_N / 128) * kMaxGroups;

    // Operands in registers: the wave's weights of a step, and sixteen of its rows at a time, read AHEAD blocks of rows before
    // they are multiplied.
    v4i b[C::NT][2];
    float w[2];
    struct Rows {
        v4i a[2];
        float s;
    } ahead[C::AHEAD];
    const auto read_weights = [&](int nt, int part, const char* st) {
        b[nt][part] = *(const v4i*)(st + (part ? read_b ^ 64 : read_b) + nt * 16 * kStep);
    };
    const auto read_wscale = [&](int k, int parity) {
        const float* at = scales_lds + parity * (2 * kMaxGroups + 4) + my_half + k;
        w[0] = at[0];
        w[1] = C::GATE_UP ? at[kMaxGroups] : w[0];
    };
    const auto read_rows = [&](Rows& o, int mt, const char* st) {
#pragma unroll
        for (int part = 0; part < 2; ++part)
            o.a[part] = *(const v4i*)(st + (part ? read_a ^ 64 : read_a) + mt * 16 * kStep);
        if (C::FP8) o.s = *(const float*)(st + read_s + mt * 64);
    };
    // The loads of all but the newest `newer` steps are done, and every wave has read what it wanted of the stages.
#define MC_STEP_BARRIER(newer)                                                                    \
    do {                                                                                          \
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(C::LOADS * (newer)) : "memory");      \
        __builtin_amdgcn_s_barrier();                                                             \
        asm volatile("" ::: "memory");                                                            \
    } while (0)

    Source now = source_of(tile), then = now;
    int parity = 0;
    if (C::FP8) load_wscales(now, 0);
    // (a tile of fewer steps than there are stages takes no tile's loads behind its own)
    const bool chained = steps >= C::STAGES;
#pragma unroll
    for (int k = 0; k < C::STAGES; ++k)
        if (k < steps)
#pragma unroll
            for (int i = 0; i < C::LOADS; ++i) load(now, i, k, k);
    if (chained) MC_STEP_BARRIER(C::STAGES - 1);
    else MC_STEP_BARRIER(0);
#pragma unroll
    for (int i = 0; i < C::NT * 2; ++i) read_weights(i % C::NT, i / C::NT, smem);
    if (C::FP8) read_wscale(0, 0);
#pragma unroll
    for (int i = 0; i < C::AHEAD; ++i) read_rows(ahead[i], i, smem);
    int stage = 0;

    for (;;) {
    Tile next = next_of();
    const bool follows = chained && next.rows > 0 && blocks_of(next.rows) == C::BLOCKS;
    if (follows) then = source_of(next);
    const int my_rows = tile.rows - wm * C::WAVE_M;      // of this wave's
    v4f acc[C::MT][C::NT];
#pragma unroll
    for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) acc[mt][nt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    // Step k.  Its last rows are read when there are AHEAD blocks of them left to multiply: then the waves meet, the stage
    // takes step k + STAGES, and what step k + 1 begins with is read behind the last products of this one, the weights
    // each as soon as its last product has begun.  The order is the one written here (sched_barrier): a matrix instruction,
    // and in its shadow a read or load and, in fp8, the four multiply-adds that take the result of the instruction LAG
    // before it into the sums.  Measured in a loop of nothing else: fp8 instructions with four such multiply-adds each 14.9
    // ns, without any 14.9; in blocks of four and sixteen they add up.  (In the whole step they are not all covered: see top.)
    const auto step = [&](int k, auto steady) {
        const char* st = smem + stage * C::STAGE_BYTES;
        const int next_stage = stage == C::STAGES - 1 ? 0 : stage + 1;
        const char* next_st = smem + next_stage * C::STAGE_BYTES;
        v4f p[C::LAG + 1];
        float t0[2], t1[2];
        const auto take = [&](int i) {          // the result of instruction i into the sums
            v4f& sum = acc[i / C::NT][i % C::NT];
            const v4f& r = p[i % (C::LAG + 1)];
            const int of = i / C::NT % 2;
            sum[0] += r[0] * t0[of];
            sum[1] += r[1] * t1[of];
            sum[2] += r[2] * t0[of];
            sum[3] += r[3] * t1[of];
            asm volatile("" : "+v"(sum));       // here and no later: results that wait cost registers
        };
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
            const Rows rows_now = ahead[0];
#pragma unroll
            for (int i = 0; i + 1 < C::AHEAD; ++i) ahead[i] = ahead[i + 1];
            if (mt + C::AHEAD == C::MT) {
                if (steady || follows || k + C::STAGES - 1 < steps) MC_STEP_BARRIER(C::STAGES - 2);
                else MC_STEP_BARRIER(0);
            }
            const bool behind = mt + C::AHEAD >= C::MT;      // behind the barrier
            read_rows(ahead[C::AHEAD - 1], (mt + C::AHEAD) % C::MT, behind ? next_st : st);
            if (C::FP8) {
                t0[mt % 2] = rows_now.s * w[0];
                t1[mt % 2] = C::GATE_UP ? rows_now.s * w[1] : t0[mt % 2];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < C::PER_MT; ++j) {
                const int nt = j % C::NT, part = j / C::NT;
                if constexpr (C::FP8) {
                    const int i = mt * C::NT + nt;
                    const v8i av = __builtin_shufflevector(rows_now.a[0], rows_now.a[1], 0, 1, 2, 3, 4, 5, 6, 7);
                    const v8i bv = __builtin_shufflevector(b[nt][0], b[nt][1], 0, 1, 2, 3, 4, 5, 6, 7);
                    p[i % (C::LAG + 1)] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bv, av, v4f{0.0f, 0.0f, 0.0f, 0.0f},
                                                                                           0, 0, 0, 0, 0, 0);
                } else {
                    acc[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, b[nt][part]),
                                                                          __builtin_bit_cast(v8bf, rows_now.a[part]),
                                                                          acc[mt][nt], 0, 0, 0);
                }
                if (mt == C::MT - 1) {
                    read_weights(nt, part, next_st);
                    if (C::FP8) read_weights(nt, 1, next_st);
                    if (C::FP8 && j == 0) read_wscale(steady || k + 1 < steps ? k + 1 : 0, steady || k + 1 < steps ? parity : parity ^ 1);
                }
                if (C::FP8 && mt * C::NT + nt >= C::LAG) take(mt * C::NT + nt - C::LAG);
                const int slot = (mt + C::AHEAD - C::MT) * C::PER_MT + j;        // behind the barrier
                if (behind)
#pragma unroll
                    for (int q = slot * C::LOADS / (C::AHEAD * C::PER_MT); q < (slot + 1) * C::LOADS / (C::AHEAD * C::PER_MT); ++q) {
                        if (steady) {
                            load(now, q, k + C::STAGES, stage);
                        } else if (follows) {
                            if (C::FP8 && q == 0 && k + C::STAGES == steps) load_wscales(then, parity ^ 1);
                            load(then, q, k + C::STAGES - steps, stage);
                        }
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (C::FP8)
#pragma unroll
            for (int i = C::MT * C::NT - C::LAG; i < C::MT * C::NT; ++i) take(i);
        stage = next_stage;
    };
    int k = 0;
    for (; k + C::STAGES < steps; ++k) step(k, std::true_type());
    for (; k < steps; ++k) step(k, std::false_type());
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");

    // --- results
    const int column = tile.n0 + wn * (C::GATE_UP ? C::WAVE_N / 2 : C::WAVE_N) + quarter * C::LANE_COLUMNS;
    const int64_t first = (int64_t)tile.e * a.RM + tile.m0 + wm * C::WAVE_M;
    if (C::GATE_UP) {
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                acc[mt][nt][0] = swiglu(acc[mt][nt][0], acc[mt][nt][1]);
                acc[mt][nt][1] = swiglu(acc[mt][nt][2], acc[mt][nt][3]);
            }
    }
    if constexpr (C::GATE_UP && C::FP8) {
        // a token's 128 columns of the tile are one scale group: the lanes' largest, then the waves' through LDS
        static_assert(C::COLUMNS == 128, "a tile is one scale group of the activations");
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
            float top = 0.0f;
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) top = fmaxf(top, fmaxf(fabsf(acc[mt][nt][0]), fabsf(acc[mt][nt][1])));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            if (quarter == 0) amax_lds[wn * C::BM + wm * C::WAVE_M + mt * 16 + l16] = top;
        }
        // (not __syncthreads, which would wait for the next tile's loads)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
            const int r = mt * 16 + l16;
            float amax = 1e-4f;
#pragma unroll
            for (int i = 0; i < C::WN; ++i) amax = fmaxf(amax, amax_lds[i * C::BM + wm * C::WAVE_M + r]);
            if (r >= my_rows) continue;
            const float inverse = 448.0f / amax;
            uint32_t q[C::NT / 2];
#pragma unroll
            for (int i = 0; i < C::NT / 2; ++i) {
                const int v = __builtin_amdgcn_cvt_pk_fp8_f32(acc[mt][2 * i][0] * inverse, acc[mt][2 * i][1] * inverse, 0, false);
                q[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(acc[mt][2 * i + 1][0] * inverse,
                                                                 acc[mt][2 * i + 1][1] * inverse, v, true);
            }
            uint32_t* o = (uint32_t*)(a.out + (first + r) * a.N + column);
#pragma unroll
            for (int i = 0; i < C::NT / 2; ++i) o[i] = q[i];
            if (wn == 0 && quarter == 0)
                a.outs[((int64_t)tile.e * (a.N / 128) + tile.n0 / 128) * a.RM + tile.m0 + wm * C::WAVE_M + r] = amax / 448.0f;
        }
    } else {
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt) {
            const int r = mt * 16 + l16;
            if (r >= my_rows || column >= a.N) break;
            uint32_t* o = (uint32_t*)(a.out + ((first + r) * a.N + column) * 2);
            uint32_t v[C::LANE_COLUMNS / 2];
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                if (C::GATE_UP) {
                    v[nt] = pack_bf16(acc[mt][nt][0], acc[mt][nt][1]);
                } else {
                    v[2 * nt] = pack_bf16(acc[mt][nt][0], acc[mt][nt][1]);
                    v[2 * nt + 1] = pack_bf16(acc[mt][nt][2], acc[mt][nt][3]);
                }
            }
            __builtin_memcpy(__builtin_assume_aligned(o, C::LANE_COLUMNS >= 8 ? 16 : C::LANE_COLUMNS * 2), v, sizeof(v));
        }
    }
    if (!follows) return next;
    tile = next;
    now = then;
    parity ^= 1;
    }
}

template <bool FP8, bool GATE_UP>
__global__ __launch_bounds__(kThreads, 2) void expert_kernel(ExpertArgs a) {
    __shared__ __align__(1024) char smem[kLdsBytes];
    __shared__ float scales_lds[FP8 ? kScaleBytes / 4 : 1];
    __shared__ int begin[kMaxLocalExperts + 1];     // tiles of rows in front of each expert
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // --- the plan.  A lane in sixteen tries a plan, on every 32nd expert; its sums meet in LDS (behind which the stages begin
    // later).  Code that runs once is fetched for it: this is written to be short.
    unsigned long long* cost_sums = (unsigned long long*)smem;      // cost and tiles by plan
    int* tile_sums = (int*)(cost_sums + 16);
    if (threadIdx.x < 16) {
        cost_sums[threadIdx.x] = 0;
        tile_sums[threadIdx.x] = 0;
    }
    const int choice = lane & 15, choice_most = 32 * plan_blocks(choice);
    const bool wide = plan_wide(choice);
    const uint32_t per_most = divisor(choice_most);
    int tiles_sum = 0;
    unsigned long long cost_sum = 0;
    __syncthreads();
    for (int e = wave * 4 + (lane >> 4); e < a.L; e += 4 * kWaves) {
        int n = a.count[e];
        n = n < 0 ? 0 : (n > a.RM ? a.RM : n);
        const int down = row_tiles(n, choice_most, per_most);
        tiles_sum += down;
        cost_sum += rows_cost(n, down, wide);
    }
    atomicAdd(&tile_sums[choice], tiles_sum);
    atomicAdd(&cost_sums[choice], cost_sum);
    __syncthreads();
    int plan;
    {
        const int columns = plan_columns(choice, GATE_UP);
        float time = plan_time(tile_sums[choice], cost_sums[choice], (a.N + columns - 1) / columns, gridDim.x, steps_of(a.Kb));
        if (choice >= (FP8 && GATE_UP ? kWidePlans : kPlans)) time = INFINITY;
        float least = time;
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) least = fminf(least, __shfl_xor(least, d));
        plan = __builtin_ctz((uint32_t)__ballot(time == least) & 0xffff);
    }
    const int most = 32 * plan_blocks(plan), bn = plan_wide(plan) ? 256 : 128;
    // --- begin[e], by every wave for itself (the same values)
    int experts;               // that have rows
    {
        const uint32_t per = divisor(most);
        int total = 0;
        experts = 0;
        for (int e0 = 0; e0 < a.L; e0 += 64) {
            int n = e0 + lane < a.L ? a.count[e0 + lane] : 0;
            n = n < 0 ? 0 : (n > a.RM ? a.RM : n);
            int sum = row_tiles(n, most, per);
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int v = __shfl_up(sum, d);
                if (lane >= d) sum += v;
            }
            experts += __popcll(__ballot(n > 0));
            if (e0 + lane < a.L) begin[e0 + lane + 1] = total + sum;
            total += __builtin_amdgcn_readlane(sum, 63);
        }
        begin[0] = 0;
    }
    __syncthreads();           // (the sums have been read: the stages are there now)

    const int columns = plan_columns(plan, GATE_UP);
    const uint32_t across = (uint32_t)((a.N + columns - 1) / columns);
    const uint64_t tiles = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane(begin[a.L]) * across;      // (less than 2^31: checked)
    const bool once = streamed(__builtin_amdgcn_readfirstlane(begin[a.L]), experts, (int)across, bn, a.Kb);
    const uint32_t xcd = blockIdx.x % kXCDs, slots = gridDim.x / kXCDs;
    const uint32_t end = (uint32_t)(tiles * (xcd + 1) / kXCDs);
    uint32_t t = (uint32_t)(tiles * xcd / kXCDs) + blockIdx.x / kXCDs;
    const auto next_of = [&]() {
        if (t >= end) return Tile{0, 0, 0, 0};
        const int row_tile = (int)(t / across);      // the expert is the last whose first tile of rows is not behind it
        int e = 0;
        for (int e0 = 0; e0 < a.L; e0 += 64) {
            const uint64_t past = __ballot(e0 + lane < a.L && begin[e0 + lane + 1] <= row_tile);
            e += __popcll(past);
            if (past != ~0ull) break;
        }
        e = __builtin_amdgcn_readfirstlane(e);
        const int first = __builtin_amdgcn_readfirstlane(begin[e]);
        const uint32_t down = (uint32_t)(__builtin_amdgcn_readfirstlane(begin[e + 1]) - first);
        const uint32_t local = t - (uint32_t)first * across;
        const uint32_t n = local / down, m = local - n * down;
        int count = __builtin_amdgcn_readfirstlane(a.count[e]);
        count = count > a.RM ? a.RM : count;
        const int each = (int)((count + down - 1) / down), m0 = (int)m * each;
        t += slots;
        return Tile{e, m0, count - m0 < each ? count - m0 : each, (int)n * columns};
    };
    Tile tile = next_of();
    while (tile.rows > 0) {
#define MC_RUN(blocks, width) run_tiles<Config<FP8, GATE_UP, blocks, width>>(a, tile, next_of, smem, scales_lds)
        const int blocks = blocks_of(tile.rows);
        if constexpr (!(FP8 && GATE_UP)) {
            if (bn == 128) {
                switch (blocks) {
                    case 1: tile = MC_RUN(1, 128); break;
                    case 2: tile = MC_RUN(2, 128); break;
                    case 3: tile = MC_RUN(3, 128); break;
                    default: tile = MC_RUN(4, 128); break;
                }
                __syncthreads();
                continue;
            }
        }
        switch (blocks) {
            case 1:
                tile = once ? run_tiles<Config<FP8, GATE_UP, 1, 256, true>>(a, tile, next_of, smem, scales_lds) : MC_RUN(1, 256);
                break;
            case 2: tile = MC_RUN(2, 256); break;
            case 3: tile = MC_RUN(3, 256); break;
            case 4: tile = MC_RUN(4, 256); break;
            case 5: tile = MC_RUN(5, 256); break;
            case 6: tile = MC_RUN(6, 256); break;
            case 7: tile = MC_RUN(7, 256); break;
            default: tile = MC_RUN(8, 256); break;
        }
        __syncthreads();       // the stages are another shape's
#undef MC_RUN
    }
}

template <bool GATE_UP>
int launch(const ExpertArgs& a, bool fp8, hipStream_t stream) {
    int device = 0, cus = 0;
    OP_HIP(hipGetDevice(&device));
    OP_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device));
    const int blocks = cus < kXCDs ? kXCDs : cus / kXCDs * kXCDs;
    if (fp8) expert_kernel<true, GATE_UP><<<blocks, kThreads, 0, stream>>>(a);
    else expert_kernel<false, GATE_UP><<<blocks, kThreads, 0, stream>>>(a);
    OP_HIP(hipGetLastError());
    return MC_EP_OK;
}

constexpr int64_t kMostBytes = (int64_t)1 << 31;   // of one expert's weights and a tile past them: offsets within are 32 bits
constexpr int kMostRows = 1 << 24;                 // of an expert: up to there the plan's divisions by multiplication are exact

// Other blocks still read what one writes over: input and output have to lie apart.
bool apart(uint64_t a, int64_t a_bytes, uint64_t b, int64_t b_bytes) {
    return a + (uint64_t)a_bytes <= b || b + (uint64_t)b_bytes <= a;
}

}  // namespace
}  // namespace mcep

using namespace mcep;

extern "C" {

int mc_ep_expert_gate_up(uint64_t packed_recv_x_ptr, uint64_t packed_recv_x_scales_ptr, uint64_t packed_recv_count_ptr,
                         uint64_t w_ptr, uint64_t w_scales_ptr, uint64_t act_ptr, uint64_t act_scales_ptr,
                         int num_local_experts, int rows_per_expert, int hidden, int intermediate, int use_fp8,
                         uint64_t stream_ptr) {
    OP_ASSERT(num_local_experts >= 0 && num_local_experts <= kMaxLocalExperts);
    OP_ASSERT(rows_per_expert >= 0 && rows_per_expert <= kMostRows);
    OP_ASSERT(hidden > 0 && hidden % 128 == 0);
    OP_ASSERT(intermediate > 0 && intermediate % (use_fp8 ? 128 : 8) == 0);
    if (num_local_experts == 0 || rows_per_expert == 0) return MC_EP_OK;
    OP_ASSERT(packed_recv_x_ptr != 0 && packed_recv_count_ptr != 0 && w_ptr != 0 && act_ptr != 0);
    OP_ASSERT(!use_fp8 || (packed_recv_x_scales_ptr != 0 && w_scales_ptr != 0 && act_scales_ptr != 0));
    OP_ASSERT(packed_recv_x_ptr % 16 == 0 && w_ptr % 16 == 0 && act_ptr % 16 == 0);
    const int64_t row = (int64_t)hidden * (use_fp8 ? 1 : 2);
    OP_ASSERT((2 * (int64_t)intermediate + 256) * row < kMostBytes);
    OP_ASSERT(!use_fp8 || hidden <= kMaxGroups * 128);
    OP_ASSERT((int64_t)num_local_experts * (rows_per_expert / 32 + 1) * (intermediate / 64 + 1) < kMostBytes);
    const int64_t rows = (int64_t)num_local_experts * rows_per_expert;
    OP_ASSERT(apart(packed_recv_x_ptr, rows * row, act_ptr, rows * intermediate * (use_fp8 ? 1 : 2)));
    OP_ASSERT(!use_fp8 || apart(packed_recv_x_scales_ptr, rows * (hidden / 128) * 4, act_scales_ptr,
                                rows * (intermediate / 128) * 4));
    ExpertArgs a{(const char*)packed_recv_x_ptr, (const float*)packed_recv_x_scales_ptr, (const int32_t*)packed_recv_count_ptr,
                 (const char*)w_ptr, (const float*)w_scales_ptr, (char*)act_ptr, (float*)act_scales_ptr, num_local_experts,
                 rows_per_expert, intermediate, (int)row};
    return launch<true>(a, use_fp8 != 0, (hipStream_t)stream_ptr);
}

int mc_ep_expert_down(uint64_t act_ptr, uint64_t act_scales_ptr, uint64_t packed_recv_count_ptr, uint64_t w_ptr,
                      uint64_t w_scales_ptr, uint64_t out_ptr, int num_local_experts, int rows_per_expert, int hidden,
                      int intermediate, int use_fp8, uint64_t stream_ptr) {
    OP_ASSERT(num_local_experts >= 0 && num_local_experts <= kMaxLocalExperts);
    OP_ASSERT(rows_per_expert >= 0 && rows_per_expert <= kMostRows);
    OP_ASSERT(hidden > 0 && hidden % 128 == 0);
    OP_ASSERT(intermediate > 0 && intermediate % (use_fp8 ? 128 : 8) == 0);
    if (num_local_experts == 0 || rows_per_expert == 0) return MC_EP_OK;
    OP_ASSERT(act_ptr != 0 && packed_recv_count_ptr != 0 && w_ptr != 0 && out_ptr != 0);
    OP_ASSERT(!use_fp8 || (act_scales_ptr != 0 && w_scales_ptr != 0));
    OP_ASSERT(act_ptr % 16 == 0 && w_ptr % 16 == 0 && out_ptr % 16 == 0);
    const int64_t row = (int64_t)intermediate * (use_fp8 ? 1 : 2);
    OP_ASSERT(((int64_t)hidden + 256) * row < kMostBytes);
    OP_ASSERT(!use_fp8 || intermediate <= kMaxGroups * 128);
    OP_ASSERT((int64_t)num_local_experts * (rows_per_expert / 32 + 1) * (hidden / 128 + 1) < kMostBytes);
    const int64_t rows = (int64_t)num_local_experts * rows_per_expert;
    OP_ASSERT(apart(act_ptr, rows * row, out_ptr, rows * hidden * 2));
    ExpertArgs a{(const char*)act_ptr, (const float*)act_scales_ptr, (const int32_t*)packed_recv_count_ptr,
                 (const char*)w_ptr, (const float*)w_scales_ptr, (char*)out_ptr, nullptr, num_local_experts,
                 rows_per_expert, hidden, (int)row};
    return launch<false>(a, use_fp8 != 0, (hipStream_t)stream_ptr);
}

int mc_ep_debug_expert_plan(const int32_t* counts, int num_local_experts, int rows_per_expert, int columns, int row_bytes,
                            int use_fp8, int gate_up, int blocks, int32_t* tile_rows, int32_t* weight_rows, int32_t* tiles,
                            int32_t* streamed_weights) {
    OP_ASSERT(num_local_experts >= 0 && num_local_experts <= kMaxLocalExperts);
    OP_ASSERT(rows_per_expert >= 0 && rows_per_expert <= kMostRows);
    OP_ASSERT(columns > 0 && row_bytes > 0 && blocks > 0);
    float least = INFINITY;
    for (int plan = 0; plan < (use_fp8 && gate_up ? kWidePlans : kPlans); ++plan) {
        const int most = 32 * plan_blocks(plan), across = (columns - 1) / plan_columns(plan, gate_up) + 1;
        int sum = 0, experts = 0;
        uint64_t cost = 0;
        for (int e = 0; e < num_local_experts; ++e) {
            const int n = counts[e] < 0 ? 0 : counts[e] > rows_per_expert ? rows_per_expert : counts[e];
            const int down = row_tiles(n, most, divisor(most));
            sum += down;
            cost += rows_cost(n, down, plan_wide(plan));
            experts += n > 0;
        }
        const float time = plan_time(sum, cost, across, blocks, steps_of(row_bytes));
        if (!(time < least)) continue;
        least = time;
        *tile_rows = most;
        *weight_rows = plan_wide(plan) ? 256 : 128;
        *tiles = sum;
        *streamed_weights = plan == 0 && streamed(sum, experts, across, 256, row_bytes);
    }
    return MC_EP_OK;
}

}  // extern "C"
