// route.hip - the router of a mixture of experts: scores of a token's E logits, the choice of its top_k experts, their weights.
//
//   s = softmax(z) or 1 / (1 + exp(-z));   c = s + bias (no bias: the order of z, which is that of s without its rounding)
//   a group's score = its largest c, or the sum of its two largest; the experts of the top_groups best groups stand for choice
//   ids = the top_k largest c among them, ties to the lowest index;   weights = s[ids] (/ their sum) * scale
//
// One wave per token: lane l holds experts l, l + 64, ..  A round of the choice is a wave maximum and one ballot per 64 experts, which finds
// the lowest index that holds it.  Scores, and c where a bias is added, are fp64: which of two experts is chosen, and with it a whole row of
// the products behind it, hangs on the last bits of c.  Without a bias c is the logit itself, fp32, and where no other score is needed (no
// groups, no softmax over all that is not divided out again) the scores of the chosen alone are formed, one per lane.
//
// What bounds it is the length of one wave's chain: a launch with no work is 2 us, a trip to memory 1 us.  Lanes meet through DPP and the
// row swaps, a few cycles each; through ds_bpermute (two per fp64 step, 100 cycles and more) a maximum took 900 cycles.  us before that / with
// it / now (fp32 keys of c, groups' scores through LDS): one token of 128 experts 5.5 / 3.7 / 3.7 - 4.5 (the host), 48 tokens of 160 experts in 8 groups
// 9.7 / 7.6 / 5.5, 8192 tokens of 256 experts in 8 groups 36 / 23.5 / 17 - 19, where what is left are the fp64 exponentials and divisions of 2 M scores and
// eight rounds of some 200 cycles, eight waves to a SIMD.
#include <type_traits>

#include "cybq_internal.h"

namespace cybq {

namespace {

constexpr double kNone = -__builtin_inf();

// The logits' type is the kernel's: with branches on it between the loads the compiler once (a variant of the rounds, E > 512, a bias) left the
// index of the bias undefined where the logits were bf16.
template <int LDT>
__device__ __forceinline__ float logit_at(const void* z, int64_t i)
{
    if constexpr (LDT == kF32) return static_cast<const float*>(z)[i];
    else if constexpr (LDT == kF16) return (float)static_cast<const _Float16*>(z)[i];
    else return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(z)[i] << 16);
}

// v of the lane that step STEP pairs this one with: 0 .. 3 within 16 lanes (mirrors pair lanes whose groups agree in themselves by then),
// 4 and 5 the neighbouring 16 and 32
template <int STEP>
__device__ __forceinline__ uint32_t partner(uint32_t v)
{
    if constexpr (STEP < 4) {
        constexpr int ctrl[4] = {0xB1, 0x4E, 0x141, 0x140};      // quad permutations [1 0 3 2], [2 3 0 1], half row mirror, row mirror
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl[STEP], 0xf, 0xf, true);
    } else {
        // the swap leaves even rows (halves) of v in both places of one result, odd ones in both of the other
        const auto r = STEP == 4 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        const bool odd = threadIdx.x & (STEP == 4 ? 16 : 32);
        return odd ? r[0] : r[1];
    }
}

template <int STEP>
__device__ __forceinline__ float partner(float v) { return __builtin_bit_cast(float, partner<STEP>(__builtin_bit_cast(uint32_t, v))); }

template <int STEP>
__device__ __forceinline__ double partner(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)partner<STEP>((uint32_t)(u >> 32)) << 32 | partner<STEP>((uint32_t)u));
}

__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }

template <int STEP = 0, class V>
__device__ __forceinline__ V wave_max(V v)
{
    v = larger(v, partner<STEP>(v));
    if constexpr (STEP < 5) return wave_max<STEP + 1>(v);
    else return v;
}

template <int STEP = 0>
__device__ __forceinline__ double wave_sum(double v)
{
    v += partner<STEP>(v);
    if constexpr (STEP < 5) return wave_sum<STEP + 1>(v);
    else return v;
}

// the two largest of 2^steps neighbouring lanes' pairs a >= b
template <int STEP = 0>
__device__ __forceinline__ void best_two(double& a, double& b, int steps)
{
    if (STEP >= steps) return;
    const double a2 = partner<STEP>(a), b2 = partner<STEP>(b);
    b = fmax(fmax(b, b2), fmin(a, a2));
    a = fmax(a, a2);
    if constexpr (STEP < 5) best_two<STEP + 1>(a, b, steps);
}

__device__ __forceinline__ double lane_value(double v, int lane)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)u, lane));
}

// the softmax term of logit z next to the largest, `top`: all -inf: zero; some +inf: they share the whole
__device__ __forceinline__ double term(float z, float top)
{
    const float none = -__builtin_inff();
    return z == none ? 0.0 : top == -none ? (z == top ? 1.0 : 0.0) : exp((double)z - (double)top);
}

__device__ __forceinline__ double sigmoid(float z) { return 1.0 / (1.0 + exp(-(double)z)); }

template <bool BIAS> struct ChoiceType { typedef float type; };
template <> struct ChoiceType<true> { typedef double type; };

// PER: experts per lane
template <int PER, bool BIAS, int LDT>
__global__ __launch_bounds__(256) void route_kernel(const void* __restrict__ logits, int T, int E, int top_k, int score,
                                                    const float* __restrict__ bias, int groups, int top_groups, int group_best, int renormalise,
                                                    float scale, int32_t* __restrict__ ids, float* __restrict__ weights)
{
    typedef typename ChoiceType<BIAS>::type Choice;
    extern __shared__ double group_lds[];                        // [waves][E], where there are groups
    const int lane = threadIdx.x & 63;
    const int t = __builtin_amdgcn_readfirstlane(blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6));
    if (t >= T) return;
    constexpr float none = -__builtin_inff();
    float z[PER];
    double s[PER];
    Choice c[PER];
    bool stands[PER];
    float b[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * 64 + lane;
        stands[i] = e < E;
        z[i] = stands[i] ? logit_at<LDT>(logits, (int64_t)t * E + e) : none;
        if (BIAS) b[i] = stands[i] ? bias[e] : 0.f;
    }
    float top = none;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        z[i] = z[i] != z[i] ? none : z[i];                       // (a logit that is no number: as good as -inf)
        top = fmaxf(top, z[i]);
    }
    const bool all_scores = BIAS || groups > 1 || (score == 0 && !renormalise);
    if (score == 0) top = wave_max(top);
    if (all_scores) {
        if (score == 0) {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < PER; i++) sum += s[i] = term(z[i], top);
            sum = wave_sum(sum);
            const double r = 1.0 / sum;
#pragma unroll
            for (int i = 0; i < PER; i++) s[i] = sum > 0.0 ? s[i] * r : 0.0;
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) s[i] = sigmoid(z[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if constexpr (BIAS) c[i] = b[i] != b[i] ? kNone : s[i] + (double)b[i];
        else c[i] = z[i];
    }
    if (groups > 1) {
        const int size = E / groups;
        // 64 / groups lanes (a power of two) to a group: its scores, laid out in LDS, among them, then the lanes' best two
        double* const all = group_lds + (threadIdx.x >> 6) * E;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (stands[i]) all[i * 64 + lane] = BIAS ? (double)c[i] : s[i];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int steps = 31 - __builtin_clz(64 / groups), g = lane >> steps;
        double first = kNone, second = kNone;
        if (g < groups)
            for (int e = lane & ((1 << steps) - 1); e < size; e += 1 << steps) {
                const double v = all[g * size + e];
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
        best_two(first, second, steps);
        double mine = group_best == 2 && size > 1 ? first + second : first;
        if (mine != mine) mine = kNone;                          // (+inf and -inf among the biases)
        mine = __shfl(mine, (lane << steps) & 63);               // lane g: the score of group g
        int better = 0;
        for (int g = 0; g < groups; g++) {
            const double v = lane_value(mine, g);
            better += v > mine || (v == mine && g < lane);
        }
        const uint64_t kept = __ballot(lane < groups && better < top_groups);
#pragma unroll
        for (int i = 0; i < PER; i++) stands[i] = stands[i] && (kept >> ((i * 64 + lane) / size)) & 1;
    }
    int32_t id = 0;
    float chosen = 0.f;                                          // lane j: choice j, its logit, its score
    double w = 0.0;
    for (int j = 0; j < top_k; j++) {
        // c rounded to fp32 keeps its order: the largest is among those of the largest fp32 number, nearly always that one alone
        float best = none;
#pragma unroll
        for (int i = 0; i < PER; i++) best = fmaxf(best, stands[i] ? (float)c[i] : none);
        best = wave_max(best);
        uint64_t holds[PER];
        int holders = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            holds[i] = __ballot(stands[i] && (float)c[i] == best);
            holders += __popcll(holds[i]);
        }
        if (BIAS && holders > 1) {
            Choice exact = (Choice)kNone;
#pragma unroll
            for (int i = 0; i < PER; i++) exact = larger(exact, (holds[i] >> lane) & 1 ? c[i] : (Choice)kNone);
            exact = wave_max(exact);
#pragma unroll
            for (int i = 0; i < PER; i++) holds[i] = __ballot(((holds[i] >> lane) & 1) && c[i] == exact);
        }
        bool found = false;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const uint64_t at = holds[i];
            if (!found && at) {
                found = true;
                const int who = __builtin_ctzll(at);
                const float its = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, z[i]), who));
                const double score_ = all_scores ? lane_value(s[i], who) : 0.0;
                if (lane == j) {
                    id = i * 64 + who;
                    chosen = its;
                    w = score_;
                }
                if (lane == who) stands[i] = false;
            }
        }
    }
    if (!all_scores && lane < top_k) w = score == 0 ? term(chosen, top) : sigmoid(chosen);
    if (renormalise) {
        const double sum = wave_sum(lane < top_k ? w : 0.0);
        w = sum > 0.0 ? w / sum : 0.0;
    }
    if (lane < top_k) {
        ids[(int64_t)t * top_k + lane] = id;
        weights[(int64_t)t * top_k + lane] = (float)(w * (double)scale);
    }
}

}  // namespace

hipError_t launch_route(const void* logits, int ldt, int64_t T, int E, int top_k, int score, const float* bias, int groups, int top_groups,
                        int group_best, bool renormalise, float scale, int32_t* ids, float* weights, hipStream_t st)
{
    const int waves = T <= 256 ? 1 : 4;                          // few tokens: a CU each
    const dim3 grid((unsigned)((T + waves - 1) / waves)), block(waves * 64);
    const int per = (E + 63) / 64;
    auto go = [&](auto kernel) {
        kernel<<<grid, block, groups > 1 ? (size_t)waves * E * 8 : 0, st>>>(logits, (int)T, E, top_k, score, bias, groups, top_groups, group_best, renormalise ? 1 : 0, scale, ids, weights);
    };
    auto with = [&](auto bias_, auto ldt_) {
        constexpr bool B = decltype(bias_)::value;
        constexpr int L = decltype(ldt_)::value;
        if (per <= 1) go(route_kernel<1, B, L>);
        else if (per <= 2) go(route_kernel<2, B, L>);
        else if (per <= 4) go(route_kernel<4, B, L>);
        else if (per <= 8) go(route_kernel<8, B, L>);
        else go(route_kernel<16, B, L>);
    };
    auto with_bias = [&](auto ldt_) { bias ? with(std::true_type{}, ldt_) : with(std::false_type{}, ldt_); };
    if (ldt == kF32) with_bias(std::integral_constant<int, kF32>{});
    else if (ldt == kF16) with_bias(std::integral_constant<int, kF16>{});
    else with_bias(std::integral_constant<int, kBF16>{});
    return hipGetLastError();
}

}  // namespace cybq
