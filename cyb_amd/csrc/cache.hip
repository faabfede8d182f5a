// cache.hip - new tokens into the paged cache (rotary embedding, quantisation) and back out of it.
//
//   x0' = x0 c - x1 s, x1' = x1 c + x0 s      (products exact and their sum rounded in fp64, then to fp32)
//   Q8, Q4, per 32 dimensions: d = f16(absmax / qmax), q = clamp(round_half_away(x / d))
//
// The rotation is in fp64 because integers come out of it: which of two a key becomes hangs on its last bits, and two programs that
// rotate in fp32 with and without fused multiplications disagree in one key of a few ten thousand.
//
// A workgroup takes the rows of one sequence that fall into one block of 32 positions, and one kv head.  Bound by memory: rows in, rows and
// blocks out.  Fewer than 32 new rows of a sequence: one launch for keys, values and queries, bytes written one by one (one token, or 48 of one
// each: 3.6 us, most of it the way from the lengths to the table to the page).  More: queries in a launch of their own (4096 tokens, 32 heads of
// 128, 67 MB: 16 - 20 us = 3.4 - 4.1 TB/s), whose registers then cost the other kernel no waves, and a block's keys and values by waves that have
// what lies side by side in it - a key's dimensions of two tokens, eight dimensions of the eight tokens of a value's 8 or 16 bytes -, written
// 8 and 16 bytes at a time (4096 tokens, 8 heads of 128, bf16 to Q8, 26 MB: 12.4 - 14 us = 1.8 - 2.1 TB/s: of its five waves the one that has the values
// has 64 of them to a lane, the others 16, so that a workgroup has that one's time).  Reading back: a block's bytes come once and rows go out 16
// bytes to a lane (80000 tokens, 8 heads of 128, Q8 to bf16, 359 MB: 68 - 79 us = 4.5 - 5.3 TB/s).
#include "cache_parts.h"
#include "cybq_internal.h"

namespace cybq {

namespace {

constexpr int kTurnThreads = 256;

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

// eight elements of a row, as they come from memory
template <int DT>
struct Eight {
    u32x4_t v[DT == kF32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* x, int64_t at)
    {
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(static_cast<const char*>(x) + at * (DT == kF32 ? 4 : 2));
        v[0] = p[0];
        if constexpr (DT == kF32) v[1] = p[1];
    }
    __device__ __forceinline__ float operator[](int e) const
    {
        if constexpr (DT == kF32) {
            const uint32_t w = v[e >> 2][e & 3];              // (a copy: of an element named in place the compiler casts the first)
            return __builtin_bit_cast(float, w);
        } else if constexpr (DT == kF16) return f16_bits_to_f32(v[0][e >> 1] >> (16 * (e & 1)) & 0xffffu);
        else return __builtin_bit_cast(float, e & 1 ? v[0][e >> 1] & 0xffff0000u : v[0][e >> 1] << 16);
    }
};

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

// x0 c - x1 s and x1 c + x0 s
__device__ __forceinline__ void turn(float x0, float x1, float c, float s, float* y0, float* y1)
{
    const double a = x0, b = x1, cd = c, sd = s;
    *y0 = (float)__builtin_fma(a, cd, -(b * sd));
    *y1 = (float)__builtin_fma(b, cd, a * sd);
}

// eight dimensions from 8 ch on of the row at x[at], turned (turn: the position's angles, or nullptr); the partner's are read next to them
template <int DT>
__device__ __forceinline__ void load_turned(const void* x, int64_t at, int ch, const float* angles, int rot, bool halves, float out[8])
{
    Eight<DT> own;
    own.load(x, at + 8 * ch);
#pragma unroll
    for (int e = 0; e < 8; e++) out[e] = own[e];
    const int d = 8 * ch, half = rot >> 1;
    if (!angles || d >= rot) return;
    if (halves) {
        const bool upper = d >= half;
        Eight<DT> other;
        other.load(x, at + (upper ? d - half : d + half));
        const float4_t* cs = reinterpret_cast<const float4_t*>(angles + 2 * (upper ? d - half : d));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4_t p = cs[i];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int e = 2 * i + j;
                float unused;
                turn(own[e], other[e], p[2 * j], upper ? -p[2 * j + 1] : p[2 * j + 1], &out[e], &unused);
            }
        }
    } else {
        const float4_t* cs = reinterpret_cast<const float4_t*>(angles + d);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float4_t p = cs[i];
#pragma unroll
            for (int j = 0; j < 2; j++) turn(own[4 * i + 2 * j], own[4 * i + 2 * j + 1], p[2 * j], p[2 * j + 1], &out[4 * i + 2 * j], &out[4 * i + 2 * j + 1]);
        }
    }
}

// Sixteen dimensions of a query row that turn together, or lie side by side; their angles serve all heads.
struct Angles {
    float4_t cs[4];
    int c0, c1;                                               // eighths of the row
    bool turns;
    __device__ __forceinline__ Angles(int j, const float* angles, int rot, bool halves)
    {
        const int turning = rot >> 4;
        c0 = 2 * j;
        c1 = 2 * j + 1;
        if (halves && j < turning) c0 = j, c1 = j + turning;
        turns = angles && j < turning;
        const float4_t* p = reinterpret_cast<const float4_t*>(angles + 16 * j);
#pragma unroll
        for (int i = 0; i < 4; i++) cs[i] = turns ? p[i] : float4_t{1.f, 0.f, 1.f, 0.f};
    }
    template <int DT>
    __device__ __forceinline__ void turned(const Eight<DT>& a, const Eight<DT>& b, bool halves, float x[8], float y[8]) const
    {
        if (!turns) {                                         // (not by an angle of 0: infinity times its sine is NaN, and -0 + 0 is 0)
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = a[e], y[e] = b[e];
        } else if (halves) {
#pragma unroll
            for (int e = 0; e < 8; e++) turn(a[e], b[e], cs[e >> 1][2 * (e & 1)], cs[e >> 1][2 * (e & 1) + 1], &x[e], &y[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                turn(a[2 * e], a[2 * e + 1], cs[e >> 1][2 * (e & 1)], cs[e >> 1][2 * (e & 1) + 1], &x[2 * e], &x[2 * e + 1]);
                turn(b[2 * e], b[2 * e + 1], cs[2 + (e >> 1)][2 * (e & 1)], cs[2 + (e >> 1)][2 * (e & 1) + 1], &y[2 * e], &y[2 * e + 1]);
            }
        }
    }
};

// what a cache can hold: NaN as 0, the rest within its range (so that nothing read back is ever infinite, and a masked value times a
// probability of 0 is 0)
__device__ __forceinline__ float limited(float x, float limit) { return x != x ? 0.f : fminf(fmaxf(x, -limit), limit); }

template <int KIND>
constexpr float kLimit = KIND == kCacheF16 ? 65504.0f : KIND == kCacheBF16 ? 3.3895313892515355e38f : 57344.0f;

template <int KIND>
__device__ __forceinline__ void limit8(float x[8])
{
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = limited(x[e], kLimit<KIND>);
}

// v of the lane one or two places from this one in its four
template <int STEP>
__device__ __forceinline__ uint32_t other_of_quad(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, STEP == 1 ? 0xB1 : 0x4E, 0xf, 0xf, true);        // quad permutations [1 0 3 2], [2 3 0 1]
}
template <int STEP>
__device__ __forceinline__ float other_of_quad(float v) { return __builtin_bit_cast(float, other_of_quad<STEP>(__builtin_bit_cast(uint32_t, v))); }

// Eight dimensions as a cache holds them: f[e] = q + 8 or q + 128 and their group's scale; the four lanes of a group call together.
// round_half_away of the quotient x / d rounded to fp32, d of 11 bits, without dividing and without a branch: such a quotient that is below a
// half-integer h stays below it when it is rounded (x would have to be nearer to h d than fp32 numbers lie), so the answer is the f with
// (f - 1/2) d <= |x| < (f + 1/2) d, and these products are exact.  The product with the reciprocal, made a little too large (2^-21: its own error
// is 3 units in the last place), finds f or f + 1.  12 instructions per value; with a clamp of each and corrections both ways 40, which
// is what bounded the kernel (4096 tokens, 8 heads of 128: 16 us, 9.6 of a 16-bit cache).
template <int KIND>
__device__ __forceinline__ _Float16 quantise8(const float x[8], float f[8])
{
    constexpr float QMAX = KIND == kCacheQ4 ? 7.0f : 127.0f, ZERO = KIND == kCacheQ4 ? 8.0f : 128.0f;
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[e]));
    amax = fmaxf(amax, other_of_quad<1>(amax));
    amax = fmaxf(amax, other_of_quad<2>(amax));
    const _Float16 dh = (_Float16)(amax / QMAX);
    const float d = (float)dh;
    const float rd = d != 0.f ? __builtin_amdgcn_rcpf(d) * (1.0f + 1.0f / 2097152.0f) : 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float a = fabsf(x[e]);
        float w = truncf(__builtin_fmaf(a, rd, 0.5f));
        w -= __builtin_fmaf(0.5f - w, d, a) < 0.f ? 1.0f : 0.f;
        f[e] = ZERO + copysignf(fminf(w, QMAX), x[e]);
    }
    return dh;
}

// f as byte `at` of w
__device__ __forceinline__ uint32_t byte_in(uint32_t w, int at, float f) { return __builtin_amdgcn_cvt_pk_u8_f32(f, at, w); }
__device__ __forceinline__ uint32_t bytes4(const float f[4]) { return byte_in(byte_in(byte_in(byte_in(0u, 0, f[0]), 1, f[1]), 2, f[2]), 3, f[3]); }
__device__ __forceinline__ uint32_t nibbles8(const float f[8])
{
    const float lo[4] = {f[0], f[4], f[1], f[5]}, hi[4] = {f[2], f[6], f[3], f[7]};
    return bytes4(lo) | bytes4(hi) << 4;
}

// a token's key or value, as bytes of its own
template <int KIND, int G>
__device__ __forceinline__ void put_one(uint8_t* half, bool value, int tok, int ch, const float x[8])
{
    const int g = ch >> 2, q4 = ch & 3;
    if constexpr (!cache_quantised(KIND)) {
        const u32x4_t w = pack8(KIND == kCacheF16 ? kF16 : kBF16, x);
        if (!value) *reinterpret_cast<u32x4_t*>(half + key_place<KIND, G>(tok, g, q4)) = w;
        else {
#pragma unroll
            for (int e = 0; e < 8; e++) *reinterpret_cast<uint16_t*>(half + value_place<KIND, G>(tok, 8 * ch + e)) = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        }
    } else {
        float f[8];
        const _Float16 dh = quantise8<KIND>(x, f);
        if (q4 == 0) *reinterpret_cast<uint16_t*>(half + cache_data_bytes(KIND, 32 * G) + scale_place(tok, g)) = __builtin_bit_cast(uint16_t, dh);
        if (!value) {
            if constexpr (KIND == kCacheQ8) *reinterpret_cast<u32x2_t*>(half + key_place<KIND, G>(tok, g, q4)) = u32x2_t{bytes4(f), bytes4(f + 4)};
            else *reinterpret_cast<uint32_t*>(half + key_place<KIND, G>(tok, g, q4)) = nibbles8(f);
        } else {
            uint32_t w[2] = {bytes4(f), bytes4(f + 4)};
            if constexpr (KIND == kCacheQ4) {                     // dimensions + 16: two lanes on
#pragma unroll
                for (int e = 0; e < 2; e++) w[e] |= other_of_quad<2>(w[e]) << 4;
                if (q4 >= 2) return;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) half[value_place<KIND, G>(tok, 8 * ch + e)] = (uint8_t)(w[e >> 2] >> (8 * (e & 3)));
        }
    }
}

// token of a block: slot s of quarter q4
__device__ __forceinline__ int token_of(int q4, int s) { return (q4 >> 1) << 4 | (s >> 2) << 3 | (q4 & 1) << 2 | (s & 3); }

// the rows of a workgroup
struct Rows {
    int b, block, from, rows;             // positions from .. from + rows, of block `block`
    int64_t row0;                         // row of `from`
    __device__ __forceinline__ bool find(const BatchView& t, int u)
    {
        Seq s;
        if (!find_block(t, u, &b, &s, &block)) return false;
        const int p0 = s.len - s.n;
        from = max(p0, block * kBlockTokens);
        rows = min(s.len, (block + 1) * kBlockTokens) - from;
        row0 = s.row0 + (from - p0);
        return true;
    }
};

// query heads head * group .. of the rows, sixteen dimensions of a row per lane, of all its heads (AHEAD of them on their way at once) or of
// one; rows at no position become zeros
template <int G, int DT, int AHEAD>
__device__ __forceinline__ void turn_queries(const Rows& r, int64_t capacity, int thread, int threads, const void* q, int64_t q_stride, int head, int group,
                                             int kv_heads, const float* rope, int rot, bool halves, void* q_out, int qdt)
{
    constexpr int DIM = 32 * G, N = DIM / 16;
    const int each = AHEAD == 1 ? 1 : group, runs = AHEAD == 1 ? group : 1;
    for (int it = thread; it < r.rows * runs * N; it += threads) {
        const int run = it / N % runs, i = it / N / runs, p = r.from + i;
        const bool there = p >= 0 && p < capacity;
        const Angles angles(it % N, rope && there ? rope + (int64_t)p * rot : nullptr, rot, halves);
        const int64_t from = (r.row0 + i) * q_stride + head * group * DIM, to = ((r.row0 + i) * kv_heads + head) * group * DIM;
        for (int h = run * each; h < run * each + each; h += AHEAD) {
            Eight<DT> a[AHEAD], b[AHEAD];
#pragma unroll
            for (int e = 0; e < AHEAD; e++) {
                const int at = min(h + e, group - 1) * DIM;
                a[e].load(q, from + at + 8 * angles.c0);
                b[e].load(q, from + at + 8 * angles.c1);
            }
#pragma unroll
            for (int e = 0; e < AHEAD; e++) {
                if (h + e >= group) break;
                float x[8], y[8];
                angles.turned(a[e], b[e], halves, x, y);
                if (!there) {
#pragma unroll
                    for (int d = 0; d < 8; d++) x[d] = y[d] = 0.f;
                }
                store8(q_out, qdt, to + (h + e) * DIM + 8 * angles.c0, x);
                store8(q_out, qdt, to + (h + e) * DIM + 8 * angles.c1, y);
            }
        }
    }
}

template <int G, int DT>
__global__ __launch_bounds__(kTurnThreads) void turn_kernel(CacheView c, BatchView t, const void* __restrict__ q, int64_t q_stride, int group,
                                                            const float* __restrict__ rope, int rot, int halves, void* __restrict__ q_out, int qdt)
{
    Rows r;
    if (!r.find(t, blockIdx.x)) return;
    turn_queries<G, DT, 4>(r, (int64_t)t.table_pages << (c.page_shift + 5), threadIdx.x, kTurnThreads, q, q_stride, blockIdx.y, group, c.kv_heads, rope, rot, halves,
                        q_out, qdt);
}

// Keys and values one token at a time: wave `wave` of `waves`
template <int KIND, int G, int DT>
__device__ __forceinline__ void put_rows(const Rows& r, uint8_t* to, bool value, int wave, int waves, const void* x, int64_t stride, int head, const float* rope,
                                         int rot, bool halves)
{
    constexpr int DIM = 32 * G, CH = DIM / 8;
    for (int it = wave * 64 + (threadIdx.x & 63); it < r.rows * CH; it += 64 * waves) {        // (the four lanes of a group are in it together)
        const int ch = it % CH, i = it / CH, p = r.from + i;
        float w[8];
        load_turned<DT>(x, (r.row0 + i) * stride + head * DIM, ch, rope && !value ? rope + (int64_t)p * rot : nullptr, rot, halves, w);
        limit8<KIND>(w);
        put_one<KIND, G>(to + (value ? cache_half_bytes(KIND, DIM) : 0), value, p & 31, ch, w);
    }
}

// Fewer than 32 rows of a sequence, which fill no block: one launch, a wave for the keys, one for the values, two for the queries
template <int KIND, int G, int DT>
__global__ __launch_bounds__(256) void append_few_kernel(CacheView c, BatchView t, const void* __restrict__ q, int64_t q_stride, int group,
                                                         const void* __restrict__ k, int64_t k_stride, const void* __restrict__ v, int64_t v_stride,
                                                         const float* __restrict__ rope, int rot, int halves, void* __restrict__ q_out, int qdt)
{
    Rows r;
    if (!r.find(t, blockIdx.x)) return;
    const int head = blockIdx.y, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave >= 2) {
        turn_queries<G, DT, 1>(r, (int64_t)t.table_pages << (c.page_shift + 5), threadIdx.x - 128, 128, q, q_stride, head, group, c.kv_heads, rope, rot, halves,
                               q_out, qdt);
        return;
    }
    uint8_t* const to = block_at(c, t, r.b, r.block, head, cache_block_bytes(KIND, 32 * G));
    if (to) put_rows<KIND, G, DT>(r, to, wave == 1, 0, 1, wave == 1 ? v : k, wave == 1 ? v_stride : k_stride, head, rope, rot, halves);
}

// Whole blocks: a wave has 64 of the keys' pairs of eight dimensions, or of the values' eights of eight
template <int G>
struct AppendShape {
    static constexpr int kKeyWaves = G, kValueWaves = (G + 3) / 4, kWaves = kKeyWaves + kValueWaves;
};

template <int KIND, int G, int DT>
__global__ __launch_bounds__(64 * AppendShape<G>::kWaves, 6) void append_kernel(CacheView c, BatchView t, const void* __restrict__ k, int64_t k_stride,
                                                                             const void* __restrict__ v, int64_t v_stride, const float* __restrict__ rope,
                                                                             int rot, int halves)
{
    typedef AppendShape<G> T;
    constexpr int DIM = 32 * G, CH = DIM / 8, BLOCK = cache_block_bytes(KIND, DIM), HALF = cache_half_bytes(KIND, DIM), DATA = cache_data_bytes(KIND, DIM);
    Rows r;
    if (!r.find(t, blockIdx.x)) return;
    const int head = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint8_t* const to = block_at(c, t, r.b, r.block, head, BLOCK);
    if (!to) return;
    const bool value = wave >= T::kKeyWaves;
    if (r.rows < kBlockTokens) {
        put_rows<KIND, G, DT>(r, to, false, wave, T::kWaves, k, k_stride, head, rope, rot, halves);
        put_rows<KIND, G, DT>(r, to, true, wave, T::kWaves, v, v_stride, head, rope, rot, halves);
        return;
    }
    const int64_t row0 = r.row0;
    const int from = r.from;
    if (!value) {                                                     // tokens m and m + 8 of every 16: their 16 bytes, or 8
        const int it = wave * 64 + lane;
        const int ch = it % CH, m = it / CH, g = ch >> 2, q4 = ch & 3, tok = (m >> 3) << 4 | (m & 7);
        float x[2][8];
#pragma unroll
        for (int w = 0; w < 2; w++) {
            const int i = tok + 8 * w;
            load_turned<DT>(k, (row0 + i) * k_stride + head * DIM, ch, rope ? rope + (int64_t)(from + i) * rot : nullptr, rot, halves, x[w]);
            limit8<KIND>(x[w]);
        }
        if constexpr (!cache_quantised(KIND)) {
#pragma unroll
            for (int w = 0; w < 2; w++) *reinterpret_cast<u32x4_t*>(to + key_place<KIND, G>(tok + 8 * w, g, q4)) = pack8(KIND == kCacheF16 ? kF16 : kBF16, x[w]);
        } else {
            float u[2][8];
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const _Float16 dh = quantise8<KIND>(x[w], u[w]);
                if (q4 == 0) *reinterpret_cast<uint16_t*>(to + DATA + scale_place(tok + 8 * w, g)) = __builtin_bit_cast(uint16_t, dh);
            }
            if constexpr (KIND == kCacheQ8)
                *reinterpret_cast<u32x4_t*>(to + key_place<KIND, G>(tok, g, q4)) = u32x4_t{bytes4(u[0]), bytes4(u[0] + 4), bytes4(u[1]), bytes4(u[1] + 4)};
            else *reinterpret_cast<u32x2_t*>(to + key_place<KIND, G>(tok, g, q4)) = u32x2_t{nibbles8(u[0]), nibbles8(u[1])};
        }
        return;
    }
    // Values: eight dimensions of the eight tokens of a quarter.  A lane's bytes of one dimension lie 16 apart from those of the next: they meet
    // in LDS, whence the wave writes whole lines (straight to memory every 512 bytes were 64 lines touched).
    constexpr int CHUNKS = CH < 16 ? CH : 16, GROUP = DATA / G;               // eights of a wave; bytes of 32 dimensions
    __shared__ u32x4_t lds[DATA / 16];
    uint8_t* const image = reinterpret_cast<uint8_t*>(lds);
    uint8_t* const half = to + HALF;
    const int vw = wave - T::kKeyWaves, ch = vw * 16 + lane % CHUNKS, q4 = min(lane / CHUNKS, 3), g = ch >> 2;
    const bool mine = lane < 4 * CHUNKS;
    Eight<DT> w[8];
#pragma unroll
    for (int j = 0; j < 8; j++) w[j].load(v, (row0 + token_of(q4, j)) * v_stride + head * DIM + 8 * ch);
    auto row = [&](int j, float (&x)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = w[j][e];
        limit8<KIND>(x);
    };
    if constexpr (!cache_quantised(KIND)) {
        u32x4_t out[8];                                           // dimension e: eight tokens of 16 bits
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float x[8];
            row(j, x);
            const u32x4_t p = pack8(KIND == kCacheF16 ? kF16 : kBF16, x);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t one = p[e >> 1] >> (16 * (e & 1)) & 0xffffu;
                out[e][j >> 1] = j & 1 ? out[e][j >> 1] | one << 16 : one;
            }
        }
        if (mine) {
#pragma unroll
            for (int e = 0; e < 8; e++) *reinterpret_cast<u32x4_t*>(image + value_place<KIND, G>(token_of(q4, 0), 8 * ch + e)) = out[e];
        }
    } else {
        u32x2_t out[8];                                           // dimension e (Q4: and e + 16): a byte of each token
        u32x4_t scales;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float x[8], u[8];
            row(j, x);
            const uint32_t dh = __builtin_bit_cast(uint16_t, quantise8<KIND>(x, u));
            scales[j >> 1] = j & 1 ? scales[j >> 1] | dh << 16 : dh;
            constexpr int order[4] = {0, 2, 1, 3};
            const int byte = KIND == kCacheQ4 ? order[j & 3] : j & 3;
#pragma unroll
            for (int e = 0; e < 8; e++) out[e][j >> 2] = byte_in(j & 3 ? out[e][j >> 2] : 0u, byte, u[e]);
        }
        if constexpr (KIND == kCacheQ4) {                             // (of use in the lower lanes of a group)
#pragma unroll
            for (int e = 0; e < 8; e++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t own = out[e][j];
                    out[e][j] = own | other_of_quad<2>(own) << 4;
                }
        }
        if (mine && (KIND == kCacheQ8 || (ch & 3) < 2)) {
#pragma unroll
            for (int e = 0; e < 8; e++) *reinterpret_cast<u32x2_t*>(image + value_place<KIND, G>(token_of(q4, 0), 8 * ch + e)) = out[e];
        }
        if (mine && (ch & 3) == 0) *reinterpret_cast<u32x4_t*>(half + DATA + scale_place(token_of(q4, 0), g)) = scales;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int first = vw * 4 * GROUP, bytes = CHUNKS / 4 * GROUP;             // the wave's part of the block
    for (int at = 16 * lane; at < bytes; at += 1024) *reinterpret_cast<u32x4_t*>(half + first + at) = *reinterpret_cast<const u32x4_t*>(image + first + at);
}

__device__ __forceinline__ float held_bits(int kind, uint32_t w) { return kind == kCacheF16 ? f16_bits_to_f32(w & 0xffffu) : __builtin_bit_cast(float, w << 16); }

// A wave reads a block's keys, one its values: whole bytes of all tokens, rows of those that are asked for.
template <int KIND, int G>
__global__ __launch_bounds__(128) void read_kernel(CacheView c, BatchView t, void* __restrict__ k, void* __restrict__ v, int dt)
{
    constexpr int DIM = 32 * G, CH = DIM / 8, BLOCK = cache_block_bytes(KIND, DIM), HALF = cache_half_bytes(KIND, DIM), DATA = cache_data_bytes(KIND, DIM);
    constexpr float ZERO = KIND == kCacheQ4 ? 8.0f : 128.0f;
    int b, block;
    Seq s;
    if (!find_block(t, blockIdx.x, &b, &s, &block)) return;
    const int head = blockIdx.y, p0 = s.len - s.n, lane = threadIdx.x & 63;
    const int from = max(p0, block * kBlockTokens), rows = min(s.len, (block + 1) * kBlockTokens) - from;
    const uint8_t* const src = block_at(c, t, b, block, head, BLOCK);
    const int before = from - block * kBlockTokens;                       // token i of the block is row i - before of `rows`
    const int64_t row0 = s.row0 + (from - p0);
    auto put = [&](void* to, int tok, int ch, const float x[8]) __attribute__((always_inline)) {
        const int i = tok - before;
        if (i >= 0 && i < rows) store8(to, dt, ((row0 + i) * c.kv_heads + head) * DIM + 8 * ch, x);
    };
    if (!src) {
        const float zeros[8] = {};
        for (int it = threadIdx.x; it < 64 * CH; it += 128) put(it < 32 * CH ? k : v, it / CH & 31, it % CH, zeros);
        return;
    }
    if (threadIdx.x < 64) {
#pragma unroll 4
        for (int it = lane; it < 16 * CH; it += 64) {
            const int ch = it % CH, m = it / CH, g = ch >> 2, q4 = ch & 3, tok = (m >> 3) << 4 | (m & 7);
            float x[2][8];
            if constexpr (!cache_quantised(KIND)) {
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const u32x4_t p = *reinterpret_cast<const u32x4_t*>(src + key_place<KIND, G>(tok + 8 * w, g, q4));
#pragma unroll
                    for (int e = 0; e < 8; e++) x[w][e] = held_bits(KIND, p[e >> 1] >> (16 * (e & 1)));
                }
            } else {
                const uint16_t* const sc = reinterpret_cast<const uint16_t*>(src + DATA + scale_place(tok, g));
                const float d[2] = {f16_bits_to_f32(sc[0]), f16_bits_to_f32(sc[4])};
                if constexpr (KIND == kCacheQ8) {
                    const u32x4_t p = *reinterpret_cast<const u32x4_t*>(src + key_place<KIND, G>(tok, g, q4));
#pragma unroll
                    for (int e = 0; e < 16; e++) x[e >> 3][e & 7] = ((float)(p[e >> 2] >> (8 * (e & 3)) & 255u) - ZERO) * d[e >> 3];
                } else {
                    const u32x2_t p = *reinterpret_cast<const u32x2_t*>(src + key_place<KIND, G>(tok, g, q4));
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        x[e >> 3][e & 7] = ((float)(p[e >> 3] >> (16 * (e & 1) + 4 * (e >> 1 & 1) + 8 * (e >> 2 & 1)) & 15u) - ZERO) * d[e >> 3];
                }
            }
#pragma unroll
            for (int w = 0; w < 2; w++) put(k, tok + 8 * w, ch, x[w]);
        }
        return;
    }
    for (int it = lane; it < 4 * CH; it += 64) {
        const int ch = it % CH, q4 = it / CH;
        const uint8_t* const half = src + HALF;
        u32x4_t p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int d = 8 * ch + e;
            const uint8_t* const at = half + value_place<KIND, G>(token_of(q4, 0), KIND == kCacheQ4 ? d & ~16 : d);
            if constexpr (!cache_quantised(KIND)) p[e] = *reinterpret_cast<const u32x4_t*>(at);
            else {
                const u32x2_t w = *reinterpret_cast<const u32x2_t*>(at);
                p[e] = u32x4_t{w[0], w[1], 0u, 0u};
            }
        }
        u32x4_t scales = {0u, 0u, 0u, 0u};
        if constexpr (cache_quantised(KIND)) scales = *reinterpret_cast<const u32x4_t*>(half + DATA + scale_place(token_of(q4, 0), ch >> 2));
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float x[8];
            const float d = f16_bits_to_f32(scales[j >> 1] >> (16 * (j & 1)) & 0xffffu);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if constexpr (!cache_quantised(KIND)) x[e] = held_bits(KIND, p[e][j >> 1] >> (16 * (j & 1)));
                else if constexpr (KIND == kCacheQ8) x[e] = ((float)(p[e][j >> 2] >> (8 * (j & 3)) & 255u) - ZERO) * d;
                else {
                    constexpr int order[4] = {0, 2, 1, 3};
                    x[e] = ((float)(p[e][j >> 2] >> (8 * order[j & 3] + (ch & 2 ? 4 : 0)) & 15u) - ZERO) * d;
                }
            }
            put(v, token_of(q4, j), ch, x);
        }
    }
}

template <int KIND, int G, int DT>
hipError_t append_of(const CacheView& c, const BatchView& t, dim3 grid, const void* q, int64_t q_stride, int group, const void* k, int64_t k_stride,
                     const void* v, int64_t v_stride, const float* rope, int rot, int halves, void* q_out, int qdt, hipStream_t st)
{
    if (t.max_new < kBlockTokens) {
        hipLaunchKernelGGL((append_few_kernel<KIND, G, DT>), grid, dim3(q ? 256 : 128), 0, st, c, t, q, q_stride, group, k, k_stride, v, v_stride, rope, rot, halves,
                           q_out, qdt);
        return hipGetLastError();
    }
    if (q) {
        hipLaunchKernelGGL((turn_kernel<G, DT>), grid, dim3(kTurnThreads), 0, st, c, t, q, q_stride, group, rope, rot, halves, q_out, qdt);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((append_kernel<KIND, G, DT>), grid, dim3(64 * AppendShape<G>::kWaves), 0, st, c, t, k, k_stride, v, v_stride, rope, rot, halves);
    return hipGetLastError();
}

template <int KIND, int G>
hipError_t append_as(const CacheView& c, const BatchView& t, dim3 grid, const void* q, int64_t q_stride, int group, const void* k, int64_t k_stride,
                     const void* v, int64_t v_stride, int dt, const float* rope, int rot, int halves, void* q_out, int qdt, hipStream_t st)
{
    auto call = dt == kF32 ? append_of<KIND, G, kF32> : dt == kF16 ? append_of<KIND, G, kF16> : append_of<KIND, G, kBF16>;
    return call(c, t, grid, q, q_stride, group, k, k_stride, v, v_stride, rope, rot, halves, q_out, qdt, st);
}

template <int KIND, int G>
hipError_t read_as(const CacheView& c, const BatchView& t, dim3 grid, void* k, void* v, int dt, hipStream_t st)
{
    hipLaunchKernelGGL((read_kernel<KIND, G>), grid, dim3(128), 0, st, c, t, k, v, dt);
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
