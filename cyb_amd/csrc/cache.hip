// cache.hip - new tokens into the paged cache (rotary embedding, quantisation) and back out of it.
//
//   x0' = x0 c - x1 s, x1' = x1 c + x0 s      (products exact and their sum rounded in fp64, then to fp32)
//   Q8, Q4, per 32 dimensions: d = f16(absmax / qmax), q = clamp(round_half_away(x / d))
//
// The rotation is in fp64 because integers come out of it: which of two a key becomes hangs on its last bits, and two programs that
// rotate in fp32 with and without fused multiplications disagree in one key of a few ten thousand.
//
// A workgroup takes the rows of one sequence that fall into one block of 32 positions, and one kv head with the query heads that share
// it; a thread takes eight dimensions of a row.  Bound by memory: rows in, rows and blocks out.
#include "cache_parts.h"
#include "cybq_internal.h"

namespace cybq {

namespace {

constexpr int kThreads = 256;

// workgroup `u` of the grid -> sequence and block of positions; false: none
__device__ __forceinline__ bool find_block(const BatchView& t, int u, int* b, Seq* s, int* block)
{
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < t.seqs; base += 64) {
        Seq mine = {0, 0, 0};
        if (base + lane < t.seqs) mine = seq_of(t, base + lane);
        const int count = row_blocks(mine), upto = wave_prefix(count);
        const int total = __builtin_amdgcn_readlane(upto, 63);
        if (u < total) {
            const int l = __builtin_ctzll(__ballot(upto > u));
            *b = base + l;
            s->row0 = __builtin_amdgcn_readlane(mine.row0, l);
            s->n = __builtin_amdgcn_readlane(mine.n, l);
            s->len = __builtin_amdgcn_readlane(mine.len, l);
            *block = ((s->len - s->n) >> 5) + u - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(count, l));
            return true;
        }
        u -= total;
    }
    return false;
}

// block `block` of sequence b and this head, nullptr: it has no page
__device__ __forceinline__ uint8_t* block_at(const CacheView& c, const BatchView& t, int b, int block, int head, int block_bytes)
{
    const int at = block >> c.page_shift;
    if (block < 0 || at >= t.table_pages) return nullptr;
    const int page = t.tables[(int64_t)b * t.table_pages + at];
    if ((unsigned)page >= (unsigned)c.pages) return nullptr;
    return c.base + page * c.page_bytes + (int64_t)((head << c.page_shift) + (block & ((1 << c.page_shift) - 1))) * block_bytes;
}

template <int DT>
__device__ __forceinline__ void load8(const void* x, int64_t at, float out[8])
{
    if constexpr (DT == kF32) {
        const float4_t* p = reinterpret_cast<const float4_t*>(static_cast<const float*>(x) + at);
        const float4_t a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] = a[i], out[4 + i] = b[i];
    } else {
        const u32x4_t v = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(x) + at);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == kF16) out[2 * i] = f16_bits_to_f32(v[i] & 0xffffu), out[2 * i + 1] = f16_bits_to_f32(v[i] >> 16);
            else out[2 * i] = __builtin_bit_cast(float, v[i] << 16), out[2 * i + 1] = __builtin_bit_cast(float, v[i] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi)
{
    const half2_t v = {(_Float16)lo, (_Float16)hi};
    return as_u32(v);
}

__device__ __forceinline__ u32x4_t pack8(int dt, const float v[8])
{
    u32x4_t out;
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = dt == kF16 ? pack_f16x2(v[2 * i], v[2 * i + 1]) : pack_bf16x2(v[2 * i], v[2 * i + 1]);
    return out;
}

__device__ __forceinline__ void store8(void* y, int dt, int64_t at, const float v[8])
{
    if (dt == kF32) {
        float4_t* p = reinterpret_cast<float4_t*>(static_cast<float*>(y) + at);
        p[0] = float4_t{v[0], v[1], v[2], v[3]};
        p[1] = float4_t{v[4], v[5], v[6], v[7]};
    } else {
        *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(y) + at) = pack8(dt, v);
    }
}

// eight dimensions from 8 c on of the row at x[at], turned; the partner's dimensions are read next to them
template <int DT>
__device__ __forceinline__ void load_turned(const void* x, int64_t at, int c, const float* rope, int rot, bool halves, float out[8])
{
    load8<DT>(x, at + 8 * c, out);
    const int d = 8 * c, half = rot >> 1;
    if (!rope || d >= rot) return;
    if (halves) {
        const bool upper = d >= half;
        float other[8];
        load8<DT>(x, at + (upper ? d - half : d + half), other);
        const float4_t* cs = reinterpret_cast<const float4_t*>(rope + 2 * (upper ? d - half : d));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4_t p = cs[i];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const double co = p[2 * j], si = upper ? p[2 * j + 1] : -p[2 * j + 1];
                out[2 * i + j] = (float)__builtin_fma((double)out[2 * i + j], co, (double)other[2 * i + j] * si);
            }
        }
    } else {
        const float4_t* cs = reinterpret_cast<const float4_t*>(rope + d);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float4_t p = cs[i];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const double a = out[4 * i + 2 * j], b = out[4 * i + 2 * j + 1], co = p[2 * j], si = p[2 * j + 1];
                out[4 * i + 2 * j] = (float)__builtin_fma(a, co, -(b * si));
                out[4 * i + 2 * j + 1] = (float)__builtin_fma(b, co, a * si);
            }
        }
    }
}

// round_half_away(x / d) for the correctly rounded quotient, |x / d| <= 128: far from a half-integer the product with the
// reciprocal decides (it is within 3 units in the last place), near one the lane divides
__device__ __forceinline__ float quotient_rounded(float x, float d, float rd)
{
    const float h = fabsf(x * rd) + 0.5f;
    const float f = truncf(h);
    const float away = fminf(h - f, f + 1.0f - h);
    float res = f;
    if (!(away > h * (1.0f / 1048576.0f))) res = truncf(fabsf(roundf(x / d)));
    return copysignf(res, x);
}

// what a cache can hold: NaN as 0, the rest within its range (so that nothing read back is ever infinite, and a masked value times a
// probability of 0 is 0)
__device__ __forceinline__ float limited(float x, float limit) { return x != x ? 0.f : fminf(fmaxf(x, -limit), limit); }

template <int KIND, int G, int DT>
__global__ __launch_bounds__(kThreads) void append_kernel(CacheView c, BatchView t, const void* __restrict__ q, int64_t q_stride, int group,
                                                          const void* __restrict__ k, int64_t k_stride, const void* __restrict__ v, int64_t v_stride,
                                                          const float* __restrict__ rope, int rot, int halves, void* __restrict__ q_out, int qdt)
{
    constexpr int DIM = 32 * G, CH = DIM / 8, BLOCK = cache_block_bytes(KIND, DIM), HALF = cache_half_bytes(KIND, DIM), DATA = cache_data_bytes(KIND, DIM);
    constexpr float LIMIT = KIND == kCacheF16 ? 65504.0f : KIND == kCacheBF16 ? 3.3895313892515355e38f : 57344.0f;
    constexpr float QMAX = KIND == kCacheQ4 ? 7.0f : 127.0f;
    int b, block;
    Seq s;
    if (!find_block(t, blockIdx.x, &b, &s, &block)) return;
    const int head = blockIdx.y, p0 = s.len - s.n;
    const int from = max(p0, block * kBlockTokens), rows = min(s.len, (block + 1) * kBlockTokens) - from;
    uint8_t* const to = block_at(c, t, b, block, head, BLOCK);
    const int64_t capacity = (int64_t)t.table_pages << (c.page_shift + 5);
    const int heads = q ? group : 0;                       // (query heads of a row that this workgroup turns)
    const int items = rows * (heads + 2) * CH;
    for (int it = threadIdx.x; it < items; it += kThreads) {
        const int ch = it % CH, hr = it / CH, which = hr % (heads + 2), i = hr / (heads + 2);
        const int p = from + i;
        const int64_t row = s.row0 + (p - p0);
        const bool there = p >= 0 && p < capacity;
        const float* turn = rope && there ? rope + (int64_t)p * rot : nullptr;
        float x[8];
        if (which < heads) {
            const int h = head * group + which;
            load_turned<DT>(q, row * q_stride + h * DIM, ch, turn, rot, halves, x);
            if (!there) {
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = 0.f;
            }
            store8(q_out, qdt, (row * c.kv_heads * group + h) * DIM + 8 * ch, x);
            continue;
        }
        const bool value = which == heads + 1;             // (the four threads of a group are in it together)
        if (!to) continue;
        if (value) load8<DT>(v, row * v_stride + head * DIM + 8 * ch, x);
        else load_turned<DT>(k, row * k_stride + head * DIM, ch, turn, rot, halves, x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = limited(x[e], LIMIT);
        const int tok = p & 31, g = ch >> 2, q4 = ch & 3;
        uint8_t* const half = to + (value ? HALF : 0);
        if constexpr (!cache_quantised(KIND)) {
            const u32x4_t w = pack8(KIND == kCacheF16 ? kF16 : kBF16, x);
            if (!value) *reinterpret_cast<u32x4_t*>(half + key_place<KIND, G>(tok, g, q4)) = w;
            else {
#pragma unroll
                for (int e = 0; e < 8; e++) *reinterpret_cast<uint16_t*>(half + value_place<KIND, G>(tok, 8 * ch + e)) = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            }
        } else {
            float amax = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[e]));
            amax = fmaxf(amax, __shfl_xor(amax, 1));
            amax = fmaxf(amax, __shfl_xor(amax, 2));
            const _Float16 dh = (_Float16)(amax / QMAX);
            const float d = (float)dh, rd = __builtin_amdgcn_rcpf(d);
            uint32_t u[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float r = d != 0.f ? quotient_rounded(x[e], d, rd) : 0.f;
                u[e] = (uint32_t)((int)fminf(fmaxf(r, -QMAX), QMAX) + (KIND == kCacheQ4 ? 8 : 128));
            }
            if (q4 == 0) *reinterpret_cast<uint16_t*>(half + DATA + scale_place(tok, g)) = __builtin_bit_cast(uint16_t, dh);
            if constexpr (KIND == kCacheQ8) {
                if (!value) {
                    u32x2_t w = {u[0] | u[1] << 8 | u[2] << 16 | u[3] << 24, u[4] | u[5] << 8 | u[6] << 16 | u[7] << 24};
                    *reinterpret_cast<u32x2_t*>(half + key_place<KIND, G>(tok, g, q4)) = w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) half[value_place<KIND, G>(tok, 8 * ch + e)] = (uint8_t)u[e];
                }
            } else {
                if (!value) {
                    uint32_t w = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++) w |= u[e] << (16 * (e & 1) + 4 * (e >> 1 & 1) + 8 * (e >> 2));
                    *reinterpret_cast<uint32_t*>(half + key_place<KIND, G>(tok, g, q4)) = w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const uint32_t upper = __shfl_xor((int)u[e], 2);       // dimension + 16: two threads on
                        if (q4 < 2) half[value_place<KIND, G>(tok, 8 * ch + e)] = (uint8_t)(u[e] | upper << 4);
                    }
                }
            }
        }
    }
}

// eight integers of a key (dimensions 8 ch .. of a token) or of a value
template <int KIND, int G>
__device__ __forceinline__ void held8(const uint8_t* half, bool value, int tok, int ch, float x[8])
{
    const int g = ch >> 2, q4 = ch & 3;
    if constexpr (!cache_quantised(KIND)) {
        uint32_t w[8];
        if (!value) {
            const u32x4_t p = *reinterpret_cast<const u32x4_t*>(half + key_place<KIND, G>(tok, g, q4));
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = p[e >> 1] >> (16 * (e & 1)) & 0xffffu;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = *reinterpret_cast<const uint16_t*>(half + value_place<KIND, G>(tok, 8 * ch + e));
        }
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = KIND == kCacheF16 ? f16_bits_to_f32(w[e]) : __builtin_bit_cast(float, w[e] << 16);
    } else {
        const float d = f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(half + cache_data_bytes(KIND, 32 * G) + scale_place(tok, g)));
        int u[8];
        if (value) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int dim = 8 * ch + e;
                const int byte = half[value_place<KIND, G>(tok, KIND == kCacheQ4 ? dim & ~16 : dim)];
                u[e] = KIND == kCacheQ4 ? (byte >> (dim & 16 ? 4 : 0)) & 15 : byte;
            }
        } else if constexpr (KIND == kCacheQ8) {
            const u32x2_t w = *reinterpret_cast<const u32x2_t*>(half + key_place<KIND, G>(tok, g, q4));
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] = (int)(w[e >> 2] >> (8 * (e & 3)) & 255u);
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(half + key_place<KIND, G>(tok, g, q4));
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] = (int)(w >> (16 * (e & 1) + 4 * (e >> 1 & 1) + 8 * (e >> 2)) & 15u);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)(u[e] - (KIND == kCacheQ4 ? 8 : 128)) * d;
    }
}

template <int KIND, int G>
__global__ __launch_bounds__(kThreads) void read_kernel(CacheView c, BatchView t, void* __restrict__ k, void* __restrict__ v, int dt)
{
    constexpr int DIM = 32 * G, CH = DIM / 8, BLOCK = cache_block_bytes(KIND, DIM), HALF = cache_half_bytes(KIND, DIM);
    int b, block;
    Seq s;
    if (!find_block(t, blockIdx.x, &b, &s, &block)) return;
    const int head = blockIdx.y, p0 = s.len - s.n;
    const int from = max(p0, block * kBlockTokens), rows = min(s.len, (block + 1) * kBlockTokens) - from;
    const uint8_t* const src = block_at(c, t, b, block, head, BLOCK);
    const int items = rows * 2 * CH;
    for (int it = threadIdx.x; it < items; it += kThreads) {
        const int ch = it % CH, hr = it / CH, i = hr >> 1;
        const bool value = hr & 1;
        const int p = from + i;
        float x[8] = {};
        if (src) held8<KIND, G>(src + (value ? HALF : 0), value, p & 31, ch, x);
        store8(value ? v : k, dt, ((int64_t)(s.row0 + (p - p0)) * c.kv_heads + head) * DIM + 8 * ch, x);
    }
}

template <int KIND, int G>
hipError_t append_as(const CacheView& c, const BatchView& t, dim3 grid, const void* q, int64_t q_stride, int group, const void* k, int64_t k_stride,
                     const void* v, int64_t v_stride, int dt, const float* rope, int rot, int halves, void* q_out, int qdt, hipStream_t st)
{
    auto kernel = dt == kF32 ? append_kernel<KIND, G, kF32> : dt == kF16 ? append_kernel<KIND, G, kF16> : append_kernel<KIND, G, kBF16>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, c, t, q, q_stride, group, k, k_stride, v, v_stride, rope, rot, halves, q_out, qdt);
    return hipGetLastError();
}

template <int KIND, int G>
hipError_t read_as(const CacheView& c, const BatchView& t, dim3 grid, void* k, void* v, int dt, hipStream_t st)
{
    hipLaunchKernelGGL((read_kernel<KIND, G>), grid, dim3(kThreads), 0, st, c, t, k, v, dt);
    return hipGetLastError();
}

#define CYBQ_BY_DIM(F, KIND, ...)                     \
    switch (c.dim) {                                  \
        case 64: return F<KIND, 2>(__VA_ARGS__);      \
        case 96: return F<KIND, 3>(__VA_ARGS__);      \
        case 128: return F<KIND, 4>(__VA_ARGS__);     \
        default: return F<KIND, 8>(__VA_ARGS__);      \
    }
#define CYBQ_BY_KIND(F, ...)                                        \
    switch (c.kind) {                                               \
        case kCacheF16: CYBQ_BY_DIM(F, kCacheF16, __VA_ARGS__)      \
        case kCacheBF16: CYBQ_BY_DIM(F, kCacheBF16, __VA_ARGS__)    \
        case kCacheQ4: CYBQ_BY_DIM(F, kCacheQ4, __VA_ARGS__)        \
        default: CYBQ_BY_DIM(F, kCacheQ8, __VA_ARGS__)              \
    }

// rows that follow each other touch at most (n + 62) / 32 blocks of a sequence, and a block that is touched has a row
dim3 grid_of(const CacheView& c, const BatchView& t)
{
    const int64_t blocks = (int64_t)t.rows / kBlockTokens + 2 * (int64_t)t.seqs;
    return dim3((unsigned)(blocks < t.rows ? blocks : t.rows), (unsigned)c.kv_heads);
}

}  // namespace

hipError_t launch_cache_append(const CacheView& c, const BatchView& t, const void* q, int64_t q_stride, int group, const void* k, int64_t k_stride,
                               const void* v, int64_t v_stride, int dt, const float* rope, int rot, bool halves, void* q_out, int qdt, hipStream_t st)
{
    const dim3 grid = grid_of(c, t);
    CYBQ_BY_KIND(append_as, c, t, grid, q, q_stride, group, k, k_stride, v, v_stride, dt, rope, rot, halves ? 1 : 0, q_out, qdt, st)
}

hipError_t launch_cache_read(const CacheView& c, const BatchView& t, void* k, void* v, int dt, hipStream_t st)
{
    const dim3 grid = grid_of(c, t);
    CYBQ_BY_KIND(read_as, c, t, grid, k, v, dt, st)
}

}  // namespace cybq
