// route.hip - the router of a mixture of experts: scores of a token's E logits, the choice of its top_k experts, their weights.
//
//   s = softmax(z) or 1 / (1 + exp(-z));   c = s + bias (no bias: the order of z, which is that of s without its rounding)
//   a group's score = its largest c, or the sum of its two largest; the experts of the top_groups best groups stand for choice
//   ids = the top_k largest c among them, ties to the lowest index;   weights = s[ids] (/ their sum) * scale
//
// One wave per token: lane l holds experts l, l + 64, ..  Everything up to the weights' last rounding is fp64: which of two experts is
// chosen, and with it a whole row of the products behind it, hangs on the last bits of c, and 256 numbers per token are no work.
// A round of the choice is a wave maximum (a butterfly) and one ballot per 64 experts, which finds the lowest index that holds it.
#include "cybq_internal.h"

namespace cybq {

namespace {

constexpr double kNone = -__builtin_inf();

__device__ __forceinline__ float logit_at(const void* z, int dt, int64_t i)
{
    if (dt == kF32) return static_cast<const float*>(z)[i];
    if (dt == kF16) return (float)static_cast<const _Float16*>(z)[i];
    return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(z)[i] << 16);
}

__device__ __forceinline__ double wave_max(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = fmax(v, __shfl_xor(v, d));
    return v;
}

__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// PER: experts per lane
template <int PER>
__global__ __launch_bounds__(256) void route_kernel(const void* __restrict__ logits, int ldt, int T, int E, int top_k, int score,
                                                    const float* __restrict__ bias, int groups, int top_groups, int group_best, int renormalise,
                                                    float scale, int32_t* __restrict__ ids, float* __restrict__ weights)
{
    const int lane = threadIdx.x & 63;
    const int t = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
    if (t >= T) return;
    double s[PER], c[PER];
    bool stands[PER];
    double top = kNone;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = i * 64 + lane;
        stands[i] = e < E;
        const float z = stands[i] ? logit_at(logits, ldt, (int64_t)t * E + e) : 0.f;
        c[i] = !stands[i] || z != z ? kNone : (double)z;         // (a logit that is no number: as good as -inf)
        top = fmax(top, c[i]);
    }
    if (score == 0) {
        top = wave_max(top);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            // all logits -inf: every score is zero; some +inf: they share the whole
            s[i] = c[i] == kNone ? 0.0 : top == -kNone ? (c[i] == top ? 1.0 : 0.0) : exp(c[i] - top);
            sum += s[i];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int i = 0; i < PER; i++) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++) s[i] = 1.0 / (1.0 + exp(-c[i]));
    }
    if (bias) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const double b = stands[i] ? (double)bias[i * 64 + lane] : 0.0;
            c[i] = b != b ? kNone : s[i] + b;
        }
    }
    if (groups > 1) {
        const int size = E / groups;
        double mine = kNone;                                     // lane g: the score of group g
        for (int g = 0; g < groups; g++) {
            double a = kNone, b = kNone;                         // the two largest so far
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int e = i * 64 + lane;
                const double v = e >= g * size && e < (g + 1) * size ? (bias ? c[i] : s[i]) : kNone;
                b = fmax(b, fmin(a, v));
                a = fmax(a, v);
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double a2 = __shfl_xor(a, d), b2 = __shfl_xor(b, d);
                b = fmax(fmax(b, b2), fmin(a, a2));
                a = fmax(a, a2);
            }
            double v = group_best == 2 && size > 1 ? a + b : a;
            if (v != v) v = kNone;                               // (+inf and -inf among the biases)
            if (lane == g) mine = v;
        }
        int better = 0;
        for (int g = 0; g < groups; g++) {
            const double v = __shfl(mine, g);
            better += v > mine || (v == mine && g < lane);
        }
        const uint64_t kept = __ballot(lane < groups && better < top_groups);
#pragma unroll
        for (int i = 0; i < PER; i++) stands[i] = stands[i] && (kept >> ((i * 64 + lane) / size)) & 1;
    }
    int32_t id = 0;
    double w = 0.0;                                              // lane j: choice j
    for (int j = 0; j < top_k; j++) {
        double best = kNone;
#pragma unroll
        for (int i = 0; i < PER; i++) best = fmax(best, stands[i] ? c[i] : kNone);
        best = wave_max(best);
        bool found = false;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const uint64_t at = __ballot(stands[i] && c[i] == best);
            if (!found && at) {
                found = true;
                const int who = __builtin_ctzll(at);
                const double v = __shfl(s[i], who);
                if (lane == j) {
                    id = i * 64 + who;
                    w = v;
                }
                if (lane == who) stands[i] = false;
            }
        }
    }
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
        kernel<<<grid, block, 0, st>>>(logits, ldt, (int)T, E, top_k, score, bias, groups, top_groups, group_best, renormalise ? 1 : 0, scale, ids, weights);
    };
    if (per <= 1) go(route_kernel<1>);
    else if (per <= 2) go(route_kernel<2>);
    else if (per <= 4) go(route_kernel<4>);
    else if (per <= 8) go(route_kernel<8>);
    else go(route_kernel<16>);
    return hipGetLastError();
}

}  // namespace cybq
