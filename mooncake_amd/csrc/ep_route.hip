// The router: logits of every token over all experts -> the topk_idx / topk_weights that dispatch and combine take, and
// the entry point mc_ep_route.
//
//   scores   s = softmax over the experts, or sigmoid, of the logits, in 32 bits
//   choice   c = s + bias where there is a bias, else the logits themselves (both scores rise with them)
//   groups   a group of experts counts as its largest choice, with a bias as the sum of its two largest; experts
//            outside the best topk_groups groups are left out
//   top-k    the largest choices in order, the lowest index first among equals
//   weights  the chosen experts' scores (without the bias), divided by their sum if asked for, times a factor
//
// A logit of -inf or NaN, or a choice of -inf or NaN, is never chosen: such places of topk_idx are -1 with weight 0, as
// for a masked token; +inf counts as the largest finite number.
//
// What bounds it: a token's logits are read once and stay in registers; the arithmetic of the scores and of K dependent
// searches is what costs, so values are compared as integers in the floats' order, a search is one instruction per
// halving of the wave and scalar instructions besides, and a lane's values are put in order once.  131072 tokens: 256
// experts, sigmoid, bias, eight groups 80-85 us (1.7 TB/s of logits; 420 vector instructions a token, a third of them the
// scores, issued at 1.2 a CU cycle, which is all there is), softmax without groups 65; 128 experts 54, 64 experts 44, 512
// experts 106.  4096 tokens of 256 5.5 us and fewer 5.3, which is the host's call (3.0 from a graph).
#include "../../include/mooncake_ep_hip.h"

#include <hip/hip_runtime.h>

#include <cfloat>
#include <climits>
#include <string>

#include "ep_operators.h"

namespace mcep {
namespace {

constexpr int kMaxTopK = 16;
constexpr int kMaxExperts = 1024;
constexpr int kMaxGroups = 64;
constexpr int kWavesPerBlock = 4;

struct RouteArgs {
    const char* logits;       // [T, E] f32 or bf16, rows row_stride elements apart
    const float* bias;        // [E] or null
    const uint8_t* mask;      // [T] or null: 0 masks the token
    int64_t* idx;             // [T, K]
    float* weights;           // [T, K]
    int64_t row_stride;
    int T, E, K;
    int groups, topk_groups, group_size;
    float scale;
    int renormalize;
    int vector;               // rows can be loaded in aligned pieces
};

template <bool HALF>
__device__ __forceinline__ float raw_logit(const char* row, int e) {
    return HALF ? __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[e] << 16) : ((const float*)row)[e];
}

// as the operator takes it: never chosen (-inf), or finite
__device__ __forceinline__ float taken_logit(float v) {
    if (!(v > -INFINITY)) v = -INFINITY;
    return fminf(v, FLT_MAX);
}

// Scores of logits as taken_logit gives them: the same values as 1 / (1 + exp(-x)) on a tensor has, to the last bit, which
// decides between nearly equal scores.  The quotient: the hardware's reciprocal and one Newton step are the correctly
// rounded 1 / d for every d from 1 to 2^126 (all mantissas tried); beyond that the score is less than the smallest normal
// number, which the reciprocal does not give, and is divided out (zero from the overflow of the exponential on, for logits
// below -88.72).  One branch for all of a lane's, the biases asked for in front of it: 131072 tokens of 256 experts 84 us
// and of 384 113, as without it (83, 111); with the biases behind it 88 and 122, with a branch for each 90 and 129.
template <int N>
__device__ __forceinline__ void sigmoids(const float (&x)[N], float (&s)[N]) {
    bool small = false;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float d = 1.0f + expf(-x[j]);
        const float r = __builtin_amdgcn_rcpf(d);
        const float q = fmaf(fmaf(-d, r, 1.0f), r, r);
        s[j] = d < 0x1p126f ? q : 0.0f;
        small |= !(d < 0x1p126f) & (x[j] > -INFINITY);
    }
    if (__builtin_expect(small, 0)) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (s[j] == 0.0f) s[j] = 1.0f / (1.0f + expf(-x[j]));
    }
}
__device__ __forceinline__ float sigmoid(float x) {
    const float of[1] = {x};
    float s[1];
    sigmoids(of, s);
    return s[0];
}

// floats in their order as integers (both zeros the same one), and back
__device__ __forceinline__ int ordered(float v) {
    const int i = __builtin_bit_cast(int, v + 0.0f);
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) { return __builtin_bit_cast(float, i ^ ((i >> 31) & 0x7fffffff)); }
constexpr int kNever = (int)0x807fffff;      // ordered(-inf)

// lanes' values moved by a DPP control; lanes that get none have the least integer, which a maximum takes into its own
// instruction
template <int CTRL>
__device__ __forceinline__ int moved(int v) {
    return __builtin_amdgcn_update_dpp(INT_MIN, v, CTRL, 0xf, 0xf, false);
}
// the same for permutations, where every lane gets one
template <int CTRL>
__device__ __forceinline__ int permuted(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float permuted(float v) {
    return __builtin_bit_cast(float, permuted<CTRL>(__builtin_bit_cast(int, v)));
}
constexpr int kRowShr = 0x110, kBcast15 = 0x142, kBcast31 = 0x143, kHalfMirror = 0x141, kMirror = 0x140;
constexpr int kXor1 = 0xb1, kXor2 = 0x4e;    // quad permutations

// the wave's largest value, in a scalar register
__device__ __forceinline__ int wave_max(int v) {
    v = max(v, moved<kRowShr + 1>(v));
    v = max(v, moved<kRowShr + 2>(v));
    v = max(v, moved<kRowShr + 4>(v));
    v = max(v, moved<kRowShr + 8>(v));
    v = max(v, moved<kBcast15>(v));
    v = max(v, moved<kBcast31>(v));
    return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// (largest, second largest) of two such pairs
__device__ __forceinline__ void join_top2(int& a1, int& a2, int b1, int b2) {
    a2 = max(min(a1, b1), max(a2, b2));
    a1 = max(a1, b1);
}

// what a group counts as, from its two largest choices
__device__ __forceinline__ int group_value(int m1, int m2, bool both) {
    if (!both) return m1;
    const float sum = from_ordered(m1) + from_ordered(m2);
    return sum > -INFINITY ? ordered(sum) : kNever;
}

// A wave per token; lane l holds experts l * NV .. l * NV + NV - 1.
//   FAST_GROUPS  groups are whole lanes, a power of two of them up to sixteen: their largest are found across lanes
//   SORTED       a lane's values are put in order for the searches, which then look at the lists' heads only
template <bool HALF, bool SOFTMAX, int NV, bool FAST_GROUPS, bool SORTED>
__global__ __launch_bounds__(64 * kWavesPerBlock) void route_wave_kernel(RouteArgs a) {
    __shared__ __align__(16) float lds_logits[kWavesPerBlock][64 * NV];
    __shared__ __align__(16) int2 lds_sorted[SORTED ? kWavesPerBlock : 1][SORTED ? 64 * (NV + 1) : 1];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * kWavesPerBlock + wave;
    if (t >= a.T) return;
    int64_t* idx_row = a.idx + (int64_t)t * a.K;
    float* weight_row = a.weights + (int64_t)t * a.K;
    if (a.mask != nullptr && a.mask[t] == 0) {
        if (lane < a.K) {
            idx_row[lane] = -1;
            weight_row[lane] = 0.0f;
        }
        return;
    }
    const char* row = a.logits + (int64_t)t * a.row_stride * (HALF ? 2 : 4);
    float x[NV];
    if (a.vector) {      // rows of whole, aligned lanes
        const bool in = lane * NV < a.E;
        if (HALF) {
            uint16_t v[NV];
            __builtin_memcpy(v, __builtin_assume_aligned(row + (in ? lane * NV * 2 : 0), NV >= 8 ? 16 : NV * 2), sizeof(v));
#pragma unroll
            for (int j = 0; j < NV; ++j) x[j] = in ? __builtin_bit_cast(float, (uint32_t)v[j] << 16) : -INFINITY;
        } else {
            float v[NV];
            __builtin_memcpy(v, __builtin_assume_aligned(row + (in ? lane * NV * 4 : 0), NV >= 4 ? 16 : NV * 4), sizeof(v));
#pragma unroll
            for (int j = 0; j < NV; ++j) x[j] = in ? v[j] : -INFINITY;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = lane * NV + j;
            x[j] = e < a.E ? raw_logit<HALF>(row, e) : -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        x[j] = taken_logit(x[j]);
        lds_logits[wave][lane * NV + j] = x[j];
    }
    int c[NV];
    float top = 0.0f, total = 0.0f;
    if (SOFTMAX) {
        int m = kNever;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            c[j] = ordered(x[j]);
            m = max(m, c[j]);
        }
        m = wave_max(m);
        top = m == kNever ? 0.0f : from_ordered(m);
#pragma unroll
        for (int j = 0; j < NV; ++j) total += expf(x[j] - top);
        total = wave_sum(total);
    } else if (a.bias == nullptr) {
#pragma unroll
        for (int j = 0; j < NV; ++j) c[j] = ordered(x[j]);
    }
    if (a.bias != nullptr) {
        float s[NV], b[NV];       // (on their way while the scores are computed: see sigmoids)
#pragma unroll
        for (int j = 0; j < NV; ++j) b[j] = a.bias[lane * NV + j < a.E ? lane * NV + j : 0];
        if (SOFTMAX) {
#pragma unroll
            for (int j = 0; j < NV; ++j) s[j] = expf(x[j] - top) / total;
        } else {
            sigmoids(x, s);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const float v = s[j] + b[j];
            c[j] = x[j] > -INFINITY && v > -INFINITY ? ordered(v) : kNever;
        }
    }
    if (a.groups > 1) {
        const bool both = a.bias != nullptr && a.group_size > 1;
        if (FAST_GROUPS) {
            int m1 = c[0], m2 = kNever;
#pragma unroll
            for (int j = 1; j < NV; ++j) join_top2(m1, m2, c[j], kNever);
            const int lanes = a.group_size / NV;
            if (lanes > 1) join_top2(m1, m2, permuted<kXor1>(m1), permuted<kXor1>(m2));
            if (lanes > 2) join_top2(m1, m2, permuted<kXor2>(m1), permuted<kXor2>(m2));
            if (lanes > 4) join_top2(m1, m2, permuted<kHalfMirror>(m1), permuted<kHalfMirror>(m2));
            if (lanes > 8) join_top2(m1, m2, permuted<kMirror>(m1), permuted<kMirror>(m2));
            const int best = group_value(m1, m2, both);
            int before = 0;
            for (int first = 0; first < a.E / NV; first += lanes) {
                const int other = __builtin_amdgcn_readlane(best, first);
                // a group further on also gives way to an equal one
                before += other > best - (lane >= first + lanes);
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) c[j] = before >= a.topk_groups ? kNever : c[j];
        } else {
            // lane g finds group g's two largest choices, in LDS (the logits are written again below)
            int* all = (int*)lds_logits[wave];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
            for (int j = 0; j < NV; ++j) all[lane * NV + j] = c[j];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            int m1 = kNever, m2 = kNever;
            if (lane < a.groups)
                for (int i = 0; i < a.group_size; ++i) join_top2(m1, m2, all[lane * a.group_size + i], kNever);
            const int best = group_value(m1, m2, both);
            int before = 0;
            for (int g = 0; g < a.groups; ++g) {
                const int other = __builtin_amdgcn_readlane(best, g);
                before += other > best || (other == best && g < lane);
            }
            const uint64_t taken = __ballot(lane < a.groups && before < a.topk_groups);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = lane * NV + j;
                if (e < a.E && !((taken >> (e / a.group_size)) & 1)) c[j] = kNever;
                lds_logits[wave][e] = x[j];
            }
        }
    }
    // --- the K largest, one after another: lane k keeps the k-th
    int mine = -1;
    if (SORTED) {
        int at[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) at[j] = lane * NV + j;
        const auto order = [&](int p, int q) {           // the larger first, of equals the lower index
            const bool swap = c[q] > c[p] || (c[q] == c[p] && at[q] < at[p]);
            const int u = c[p], v = c[q], i = at[p], k = at[q];
            c[p] = swap ? v : u;
            c[q] = swap ? u : v;
            at[p] = swap ? k : i;
            at[q] = swap ? i : k;
        };
        if (NV == 2) order(0, 1 % NV);
        if (NV == 4) {
            order(0, 1 % NV);
            order(2 % NV, 3 % NV);
            order(0, 2 % NV);
            order(1 % NV, 3 % NV);
            order(1 % NV, 2 % NV);
        }
        if (NV == 8) {
            constexpr int network[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                            {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
            for (int i = 0; i < 19; ++i) order(network[i][0] % NV, network[i][1] % NV);
        }
        int2* list = lds_sorted[wave] + lane * (NV + 1);
#pragma unroll
        for (int j = 1; j < NV; ++j) list[j] = make_int2(c[j], at[j]);
        list[NV] = make_int2(kNever, 0);
        int head = c[0], head_at = at[0];
        for (int k = 0; k < a.K; ++k) {
            const int m = wave_max(head);
            if (m == kNever) break;
            const int winner = __builtin_ctzll(__ballot(head == m));
            const int won = __builtin_amdgcn_readlane(head_at, winner);
            mine = lane == __builtin_amdgcn_readfirstlane(k) ? won : mine;
            if (lane == winner) {
                const int2 next = *++list;
                head = next.x;
                head_at = next.y;
            }
        }
    } else {
        for (int k = 0; k < a.K; ++k) {
            int m = c[0];
#pragma unroll
            for (int j = 1; j < NV; ++j) m = max(m, c[j]);
            m = wave_max(m);
            if (m == kNever) break;
            int j_of = NV;
#pragma unroll
            for (int j = NV - 1; j >= 0; --j) j_of = c[j] == m ? j : j_of;
            const int winner = __builtin_ctzll(__ballot(j_of < NV));
            const int j_won = __builtin_amdgcn_readlane(j_of, winner);
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (lane == winner && j == j_won) c[j] = kNever;
            if (lane == k) mine = winner * NV + j_won;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    float w = 0.0f;
    if (mine >= 0) {
        const float v = lds_logits[wave][mine];
        w = SOFTMAX ? expf(v - top) / total : sigmoid(v);
    }
    if (a.renormalize) {
        // (K <= 16: the first sixteen lanes' sum, the same in all of them)
        float sum = w + permuted<kXor1>(w);
        sum += permuted<kXor2>(sum);
        sum += permuted<kHalfMirror>(sum);
        sum += permuted<kMirror>(sum);
        if (sum > 0.0f) w /= sum;
    }
    if (lane < a.K) {
        idx_row[lane] = mine;
        weight_row[lane] = w * a.scale;
    }
}

// A thread per token, for up to N experts: a wave per token would have most of its lanes idle.
template <bool HALF, bool SOFTMAX, int N>
__global__ __launch_bounds__(64) void route_thread_kernel(RouteArgs a) {
    const int t = blockIdx.x * 64 + threadIdx.x;
    if (t >= a.T) return;
    int64_t* idx_row = a.idx + (int64_t)t * a.K;
    float* weight_row = a.weights + (int64_t)t * a.K;
    if (a.mask != nullptr && a.mask[t] == 0) {
        for (int k = 0; k < a.K; ++k) {
            idx_row[k] = -1;
            weight_row[k] = 0.0f;
        }
        return;
    }
    const char* row = a.logits + (int64_t)t * a.row_stride * (HALF ? 2 : 4);
    float x[N], top = -INFINITY, total = 0.0f;
    if (a.vector && a.E == N) {
        if (HALF) {
            uint16_t v[N];
            __builtin_memcpy(v, __builtin_assume_aligned(row, 16), sizeof(v));
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = __builtin_bit_cast(float, (uint32_t)v[j] << 16);
        } else {
            __builtin_memcpy(x, __builtin_assume_aligned(row, 16), sizeof(x));
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = j < a.E ? raw_logit<HALF>(row, j) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        x[j] = taken_logit(x[j]);
        top = fmaxf(top, x[j]);
    }
    if (top == -INFINITY) top = 0.0f;
    float s[N];
    if (SOFTMAX) {
#pragma unroll
        for (int j = 0; j < N; ++j) s[j] = expf(x[j] - top);
    } else {
        sigmoids(x, s);
    }
    if (SOFTMAX) {      // in pairs of pairs, as the lanes of a wave add
        float part[N];
#pragma unroll
        for (int j = 0; j < N; ++j) part[j] = s[j];
#pragma unroll
        for (int d = N / 2; d > 0; d >>= 1)
#pragma unroll
            for (int j = 0; j < N / 2; ++j)
                if (j < d) part[j] += part[j + d];
        total = part[0];
    }
    int c[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (SOFTMAX) s[j] = s[j] / total;
        if (a.bias != nullptr) {
            const float v = s[j] + a.bias[j < a.E ? j : 0];
            c[j] = x[j] > -INFINITY && v > -INFINITY ? ordered(v) : kNever;
        } else {
            c[j] = ordered(x[j]);
        }
    }
    if (a.groups > 1) {
        const bool both = a.bias != nullptr && a.group_size > 1;
        int best[N];                 // of the group that expert j belongs to
#pragma unroll
        for (int j = 0; j < N; ++j) {
            int m1 = kNever, m2 = kNever;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i / a.group_size == j / a.group_size) join_top2(m1, m2, c[i], kNever);
            best[j] = group_value(m1, m2, both);
        }
        bool out[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            int before = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < a.E && i % a.group_size == 0)
                    before += best[i] > best[j] || (best[i] == best[j] && i / a.group_size < j / a.group_size);
            out[j] = before >= a.topk_groups;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) c[j] = out[j] ? kNever : c[j];
    }
    float sum = 0.0f, w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        w[k] = 0.0f;
        if (k >= a.K) continue;
        int m = kNever, at = -1;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c[j] > m) {
                m = c[j];
                at = j;
                w[k] = s[j];
            }
#pragma unroll
        for (int j = 0; j < N; ++j) c[j] = j == at ? kNever : c[j];
        idx_row[k] = at;
        sum += w[k];
    }
    if (!a.renormalize || !(sum > 0.0f)) sum = 1.0f;
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (k < a.K) weight_row[k] = w[k] / sum * a.scale;
}

template <bool HALF, bool SOFTMAX, int NV, bool SORTED>
void launch_wave(const RouteArgs& a, hipStream_t stream) {
    const int blocks = (a.T + kWavesPerBlock - 1) / kWavesPerBlock;
    const dim3 threads(64 * kWavesPerBlock);
    const int lanes = a.group_size % NV == 0 ? a.group_size / NV : 0;
    RouteArgs b = a;
    // what a lane loads lies in one aligned piece
    const int piece = NV * (HALF ? 2 : 4) < 16 ? NV * (HALF ? 2 : 4) : 16;
    b.vector = a.E % NV == 0 && (uint64_t)a.logits % piece == 0 && a.row_stride * (HALF ? 2 : 4) % piece == 0;
    if (a.groups == 1 || lanes == 1 || lanes == 2 || lanes == 4 || lanes == 8 || lanes == 16)
        route_wave_kernel<HALF, SOFTMAX, NV, true, SORTED><<<blocks, threads, 0, stream>>>(b);
    else
        route_wave_kernel<HALF, SOFTMAX, NV, false, SORTED><<<blocks, threads, 0, stream>>>(b);
}

template <bool HALF, bool SOFTMAX, int N>
void launch_thread(const RouteArgs& a, hipStream_t stream) {
    RouteArgs b = a;
    b.vector = (uint64_t)a.logits % 16 == 0 && a.row_stride * (HALF ? 2 : 4) % 16 == 0;
    route_thread_kernel<HALF, SOFTMAX, N><<<(a.T + 63) / 64, 64, 0, stream>>>(b);
}

template <bool HALF, bool SOFTMAX>
void launch_route(const RouteArgs& a, hipStream_t stream) {
    if (a.E <= 8) launch_thread<HALF, SOFTMAX, 8>(a, stream);
    else if (a.E <= 64) launch_wave<HALF, SOFTMAX, 1, true>(a, stream);
    else if (a.E <= 128) launch_wave<HALF, SOFTMAX, 2, true>(a, stream);
    else if (a.E <= 256) launch_wave<HALF, SOFTMAX, 4, true>(a, stream);
    // eight values a lane are put in order (19 exchanges) for more than five searches: 131072 tokens of 512 experts, top 4
    // 90 us against 84 searched as they lie, top 8 104 against 117, top 16 128 against 186
    else if (a.E <= 512 && a.K > 5) launch_wave<HALF, SOFTMAX, 8, true>(a, stream);
    else if (a.E <= 512) launch_wave<HALF, SOFTMAX, 8, false>(a, stream);
    // sixteen never: 60 exchanges, and lists that leave room for fewer waves
    else launch_wave<HALF, SOFTMAX, 16, false>(a, stream);
}

}  // namespace
}  // namespace mcep

using namespace mcep;

extern "C" int mc_ep_route(uint64_t logits_ptr, int logits_bf16, int64_t logits_row_stride, uint64_t bias_ptr,
                           uint64_t token_mask_ptr, int num_tokens, int num_experts, int num_topk, int sigmoid_scores,
                           int num_groups, int num_topk_groups, int renormalize, float scale, uint64_t topk_idx_ptr,
                           uint64_t topk_weights_ptr, uint64_t stream_ptr) {
    OP_ASSERT(num_tokens >= 0);
    OP_ASSERT(num_experts > 0 && num_experts <= kMaxExperts);
    OP_ASSERT(num_topk > 0 && num_topk <= kMaxTopK && num_topk <= num_experts);
    OP_ASSERT(num_groups > 0 && num_groups <= kMaxGroups && num_experts % num_groups == 0);
    OP_ASSERT(num_topk_groups > 0 && num_topk_groups <= num_groups);
    OP_ASSERT(num_tokens <= 1 || logits_row_stride >= num_experts);
    if (num_tokens == 0) return MC_EP_OK;
    OP_ASSERT(logits_ptr != 0 && topk_idx_ptr != 0 && topk_weights_ptr != 0);
    const RouteArgs a{(const char*)logits_ptr, (const float*)bias_ptr, (const uint8_t*)token_mask_ptr, (int64_t*)topk_idx_ptr,
                      (float*)topk_weights_ptr, logits_row_stride, num_tokens, num_experts, num_topk, num_groups,
                      num_topk_groups, num_experts / num_groups, scale, renormalize, 0};
    const hipStream_t stream = (hipStream_t)stream_ptr;
    if (logits_bf16) {
        if (sigmoid_scores) launch_route<true, false>(a, stream);
        else launch_route<true, true>(a, stream);
    } else {
        if (sigmoid_scores) launch_route<false, false>(a, stream);
        else launch_route<false, true>(a, stream);
    }
    OP_HIP(hipGetLastError());
    return MC_EP_OK;
}
