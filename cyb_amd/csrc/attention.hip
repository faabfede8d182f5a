// attention.hip - attention of new tokens over the paged cache (cache_parts.h).
//
//   s_j = scale q . k_j,  max(0, p - window + 1) <= j <= p,  in a page;     y = sum_j softmax(s)_j v_j;  nothing to see: y = 0
//
// One pass with a running maximum and sum per row, fp32.  Rows of one kv head - its `group` query heads of one new token after
// another - stand side by side as columns of S^T = K Q^T, so a lane holds scores of one row only: maxima and sums meet other lanes
// twice, and the scores are, as they lie, the operand of Y^T = V^T P^T.
//
// Operands.  16-bit caches: their own type, P of bf16 as two numbers (its 8 bits alone would be the result's error).  Q8, Q4: f16.  Keys are
// the exact integers, their scales come in fp32 on each group's products; values are round_f16(scale q), 2^-12, and P is two numbers, so that this
// rounding stands alone (48 conversations: 3.5e-4 off with one number, 2.9e-4 with two, 2.1e-4 of them y's own; no slower, memory is what such
// calls wait for); rows of bf16 become f16 behind a power of two.
#include <algorithm>
#include <type_traits>

#include "cache_parts.h"
#include "cybq_internal.h"

namespace cybq {

namespace {

// Work is shared out on the device: lengths are known there only, and a captured call meets longer ones every time.  A unit is one tile
// of rows of one sequence and kv head, and a part of the blocks that it sees; parts are as long as makes `target` units of all.
struct AttnArgs {
    CacheView c;
    BatchView t;
    const void* q;
    void* y;
    int64_t q_stride;
    float* slabs;
    unsigned* tickets;
    int group, qdt, window, target;              // target: workgroups of a round of the tiles kernel
    int few;                                     // > 0: sequences of up to so many rows per kv head are the rows kernel's, others not
    float scale;                                 // times log2 e
};

constexpr int kMaxUnits = 1 << 24;               // of a call
// Probabilities are 2^((s - m) c + kShift): a row's m is its largest score, or near it, and may lag behind the scores by kLagF16 (in exponents) before sums
// are scaled anew: every scaling is a detour of a wave that all others of its workgroup wait for (with a lag of 3 one step in seven, 512 rows of a Q8
// cache after 15872 tokens took 216 us; with 11: 198).
// P of f16 stays at 2^15 or below; it is exact to its bits from 2^-14 on and to 2^-25 below, of a row's largest 2^-18 and 2^-29 for many rows.  The rows
// kernel's waves wait for nobody: m is put kRowsBelow below the largest, so that 2^-26 and 2^-37 of it are left (8 drafts of 5 tokens 16.5 -> 16.6 us).
// P of bf16 has fp32's range: m is put kAhead above the largest, and sums of p |v| are never more than those of |v|, which may be anything that fp32 holds.
constexpr float kShiftF16 = 4.f, kLagF16 = 11.f, kRowsBelow = 8.f;
constexpr float kAhead = 16.f;
constexpr float kFar = 4096.f;                   // up to here a product of a score and its factor is off by at most 2^-13

// Workgroups of a round of the rows kernel (two to a CU), and how many parts there may be beyond one of each tile: twice as many.  Grids, slabs and
// tickets are made for these.  Rows kernel: a part is work / extra blocks or more, extra at most kRounds target, so that the tiles' blocks make that many
// parts at most.  Tiles kernel: a part is work / target blocks or more, and work counts at least half of the blocks of each tile.  Parts that need a slab are
// those of tiles with two or more: at most twice the parts beyond one of each.
constexpr int kTarget = 512, kMostExtra = 2 * kTarget;
constexpr float kRounds = 2.f;                   // (rows kernel)
constexpr int kLeast = 4, kTileLeast = 8;        // blocks of a part
// Tiles kernel.  A tile is cut where that makes it kJoinBlocks shorter: storing the parts, waiting for the last and adding them takes about that long
// (prompts of one sequence, 28, 40 blocks: 1800 tokens of heads of 128 76, 54 us, 2000 85, 60, 2000 of heads of 64 48, 33; 16: 1000 tokens 40, 34), into
// up to sqrt(kJoin * its blocks) parts: each adds 1.5 us to what the last of them has to do (96 rows of 4000 tokens 0.1, 0.2, 0.4: 51, 45, 45 us, with
// no limit 64).  Measured on F16 of 128 and BF16 of 64; a block of larger heads or of Q8 and Q4 takes longer, and there the same numbers cut less than
// might pay.
constexpr int kJoinBlocks = 40;
constexpr float kJoin = 0.2f;

// Rows of a sequence and kv head (new tokens times group) that the rows kernel takes.  Where there are few in all, many too: the other kernel's
// tiles, each of 256 rows, would be fewer than there are CUs, their parts many and long to join (heads of 128, 4 query heads to each of 8 kv heads;
// us, rows kernel and tiles kernel.  F16: 128 rows of 1000 tokens 11 and 34, 16 x 24 of 3000 73 and 81, 8 x 64 60 and 59, 32 x 32 166 and 115;
// Q4: 2 x 128 55 and 52, 8 x 64 80 and 62, 32 x 16 of 4000 106 and 127; other heads go by the same numbers, which were not measured on them).
constexpr int kFewRows = 64, kFewAlone = 512;
constexpr int few_in_all(int kind) { return cache_quantised(kind) ? 1 << 13 : 1 << 14; }

struct Unit {
    Seq s;
    int b, tile, head, split, splits, slab, ticket;
};

// first and last block that rows r0 .. r1 (positions p0 ..) see
__device__ __forceinline__ void seen(const AttnArgs& a, int p_first, int p_last, int64_t capacity, int* lo, int* hi)
{
    const int64_t end = min((int64_t)p_last, capacity - 1);
    const int first = a.window && p_first >= a.window ? p_first - a.window + 1 : 0;
    *lo = first >> 5;
    *hi = end < first ? *lo : (int)(end >> 5) + 1;
}

// tiles of a sequence, 0: the other kernel's
template <int ROWS, bool MANY>
__device__ __forceinline__ int tiles_of(const AttnArgs& a, const Seq& s)
{
    const int rows = s.n * a.group;
    return a.few && (rows > a.few) != MANY ? 0 : (rows + ROWS - 1) / ROWS;
}

// sum over the wave, the same on every lane
__device__ __forceinline__ float wave_total(float v)
{
    auto step = [&](int moved) { v += __builtin_bit_cast(float, moved); };
    step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x111, 0xf, 0xf, true));       // as in wave_prefix
    step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x112, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x114, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x118, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x142, 0xa, 0xf, false));
    step(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x143, 0xc, 0xf, false));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// what a lane knows of its sequence: its tiles, the blocks of the one that sees the most, and of one on average (at least half of that)
struct Share {
    Seq s;
    int tiles, blocks;
    float mean;
};
template <int ROWS, bool MANY>
__device__ __forceinline__ Share share_of(const AttnArgs& a, int b, int64_t capacity)
{
    Share x = {{0, 0, 0}, 0, 0, 0.f};
    if (b < a.t.seqs) {
        x.s = seq_of(a.t, b);
        int lo, hi;
        seen(a, x.s.len - x.s.n, x.s.len - 1, capacity, &lo, &hi);
        x.tiles = tiles_of<ROWS, MANY>(a, x.s);
        x.blocks = hi - lo;
        if (MANY && a.window) x.blocks = min(x.blocks, (int)(((int64_t)a.window + ROWS / a.group + 2) >> 5) + 2);
        x.mean = (float)x.blocks;
        if (MANY && !a.window) x.mean -= fminf((float)(x.s.n >> 6), 0.5f * x.mean);
    }
    return x;
}

template <int ROWS, bool MANY>
__device__ __forceinline__ bool find_unit(const AttnArgs& a, int u, Unit* out)
{
    const int lane = threadIdx.x & 63;
    const int64_t capacity = (int64_t)a.t.table_pages << (a.c.page_shift + 5);
    const int heads = a.c.kv_heads;
    Share x = share_of<ROWS, MANY>(a, lane, capacity);
    float work = (float)x.tiles * x.mean, tiles = (float)x.tiles;
    for (int base = 64; base < a.t.seqs; base += 64) {
        const Share more = share_of<ROWS, MANY>(a, base + lane, capacity);
        work += (float)more.tiles * more.mean;
        tiles += (float)more.tiles;
    }
    work = wave_total(work) * (float)heads;
    tiles = wave_total(tiles) * (float)heads;
    int part;
    if constexpr (!MANY) {
        // Every tile begins a part of its own, so what is to be had in one round of workgroups are `target` less the tiles; where that is less than half
        // of a round, rounds follow each other anyway and parts are made for their balance (48 conversations of up to 8192 tokens: 1, 2, 4, 8 rounds 111,
        // 103, 108, 120 us).  (A little more, so that what is rounded never makes more parts than the slabs hold.)
        const float more = (float)kTarget - tiles, extra = more >= 0.5f * (float)kTarget ? more : kRounds * (float)kTarget;
        part = max(kLeast, (int)fminf(work / extra * 1.0001f + 1.0f, 1.0e9f));
    } else {
        // Only what is longer than a workgroup's share by kJoinBlocks is cut; where the tiles are one round, into the shortest parts that still are.
        const float share = work / (float)a.target;
        part = max(kTileLeast, (int)fminf(share * 1.0001f + (float)(kJoinBlocks + 1), 1.0e9f));
        if (a.t.seqs <= 64 && tiles <= (float)a.target && __ballot((float)x.blocks - share >= (float)kJoinBlocks)) {
            for (int k = 0; k < 5; k++) {
                const int shorter = max(kTileLeast, (int)(share * (1.0f + 0.1f * (float)k)) + 1);
                const float all = wave_total((float)(x.tiles * heads) * __builtin_ceilf((float)x.blocks * __builtin_amdgcn_rcpf((float)shorter)));
                if (all <= (float)a.target) {
                    part = min(part, shorter);
                    break;
                }
            }
        }
    }
    int64_t units = 0;
    int slabs = 0, tickets = 0;
    bool found = false;
    for (int base = 0; base < a.t.seqs; base += 64) {
        if (base) x = share_of<ROWS, MANY>(a, base + lane, capacity);
        int splits = x.tiles ? max(1, (x.blocks + part - 1) / part) : 0;
        if (MANY) {
            splits = min(splits, max(1, (int)__builtin_sqrtf(kJoin * (float)x.blocks)));
            if (splits > 1 && x.blocks - x.blocks / splits < kJoinBlocks) splits = 1;
        }
        // (a batch whose starts make no sense may add up to anything: what cannot be right stays above every grid)
        const int rows = min(x.tiles * heads, kMaxUnits + 1), mine = (int)min((int64_t)rows * splits, (int64_t)kMaxUnits + 1);
        const int upto = wave_prefix(mine), slab_upto = wave_prefix(splits > 1 ? mine : 0), ticket_upto = wave_prefix(splits > 1 ? rows : 0);
        const int total = __builtin_amdgcn_readlane(upto, 63);
        // All in one round, two workgroups to a CU: next to the one that sees the most goes the one that sees the least
        if (MANY && a.t.seqs <= 64 && total <= a.target && u < total) {
            const int half = a.target / 2 / heads * heads;
            if (u >= half) u = total - heads - (u - half) / heads * heads + (u - half) % heads;
        }
        if (!found && u < units + total) {
            found = true;
            const int l = __builtin_ctzll(__ballot((int)units + upto > u));
            out->s.row0 = __builtin_amdgcn_readlane(x.s.row0, l);
            out->s.n = __builtin_amdgcn_readlane(x.s.n, l);
            out->s.len = __builtin_amdgcn_readlane(x.s.len, l);
            out->b = base + l;
            out->splits = __builtin_amdgcn_readlane(splits, l);
            const int at = u - (int)units - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l));
            // heads first: workgroups of one head, which read the same blocks, go to the same XCDs where there are 2, 4 or 8 of them; the last
            // tiles first, which see the most
            const int behind = at / heads, of_tile = behind / out->splits;
            out->head = at - behind * heads;
            out->split = behind - of_tile * out->splits;
            out->tile = __builtin_amdgcn_readlane(x.tiles, l) - 1 - of_tile;
            const int rest = out->tile * heads + out->head;
            out->slab = slabs + __builtin_amdgcn_readlane(slab_upto, l) - __builtin_amdgcn_readlane(mine, l) + rest * out->splits + out->split;
            out->ticket = tickets + __builtin_amdgcn_readlane(ticket_upto, l) - __builtin_amdgcn_readlane(rows, l) + rest;
        }
        units += total;
        slabs += __builtin_amdgcn_readlane(slab_upto, 63);
        tickets += __builtin_amdgcn_readlane(ticket_upto, 63);
    }
    // more units than workgroups: the starts rise and fall.  Nobody begins what nobody could finish.
    return found && units <= (int64_t)gridDim.x;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <int STEP>
__device__ __forceinline__ float other_quarter(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = STEP == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (uint32_t)(threadIdx.x & STEP ? r[0] : r[1]));
}

template <int KIND>
__device__ __forceinline__ float4_t mfma16(Frag16 a, Frag16 b, float4_t c)
{
    if constexpr (KIND == kCacheBF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, b.b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi)
{
    const half2_t v = {(_Float16)lo, (_Float16)hi};
    return as_u32(v);
}

// A score's factor is a normal number: of 0 a hidden score would be NaN, of infinity one of 0.  (Scores that are not 0 are multiples of 2^-48 on
// quantised caches: where the largest factor takes the place of a larger one, one token has it all either way.)
constexpr float kLeastFactor = 0x1p-126f, kMostFactor = 0x1.fffffep127f;

// rows of bf16 as f16: the power of two that brings the row's largest to 2^14 .. 2^15; *c, the scores' factor, takes it off again
__device__ __forceinline__ float row_power(float top, float* c)
{
    const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
    const int up = e == 0 || e == 255 ? 0 : max(-126, min(126, 141 - e));           // 2^up, and 2^-up, are normal numbers
    *c = fminf(fmaxf(*c * __builtin_bit_cast(float, (uint32_t)(127 - up) << 23), kLeastFactor), kMostFactor);
    return __builtin_bit_cast(float, (uint32_t)(127 + up) << 23);
}

// a block's keys or values and their scales, as a lane has them from memory
template <int KIND, int G>
struct Half {
    static constexpr int N = KIND == kCacheQ8 ? G : KIND == kCacheQ4 ? (G + 1) / 2 : 2 * G;
    u32x4_t d[N];
    u32x4_t s[cache_quantised(KIND) ? G : 1];
    __device__ __forceinline__ void load(const uint8_t* p, int lane)
    {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (KIND == kCacheQ4 && (G & 1) && i == N - 1) {
                const u32x2_t v = *reinterpret_cast<const u32x2_t*>(p + i * 1024 + lane * 8);
                d[i] = u32x4_t{v[0], v[1], 0u, 0u};
            } else {
                d[i] = *reinterpret_cast<const u32x4_t*>(p + i * 1024 + lane * 16);
            }
        }
        if constexpr (cache_quantised(KIND)) {
#pragma unroll
            for (int g = 0; g < G; g++) s[g] = *reinterpret_cast<const u32x4_t*>(p + cache_data_bytes(KIND, 32 * G) + (g * 4 + (lane >> 4)) * 16);
        }
    }
};

// eight nibbles (bit 16 (s & 1) + 4 (s >> 1 & 1) + 8 (s >> 2)) -> exact f16 integers
__device__ __forceinline__ void nibbles_f16(uint32_t w, uint32_t magic, uint32_t out[4])
{
    const half2_t sub = {(_Float16)-1032.0f, (_Float16)-1032.0f}, mul = {(_Float16)0.0625f, (_Float16)0.0625f}, add = {(_Float16)-72.0f, (_Float16)-72.0f};
    const uint32_t h = w >> 8;
    out[0] = as_u32(as_h2((w & 0x000F000Fu) | magic) + sub);
    out[1] = as_u32(as_h2((w & 0x00F000F0u) | magic) * mul + add);
    out[2] = as_u32(as_h2((h & 0x000F000Fu) | magic) + sub);
    out[3] = as_u32(as_h2((h & 0x00F000F0u) | magic) * mul + add);
}

// keys of tile t16 and group g as operand: exact integers, or the values themselves
template <int KIND, int G>
__device__ __forceinline__ Frag16 key_operand(const Half<KIND, G>& k, int t16, int g, uint32_t magic)
{
    Frag16 f;
    if constexpr (KIND == kCacheQ8) {
        uint32_t o[4];
        unpack_q8_f16(k.d[g][2 * t16], k.d[g][2 * t16 + 1], o);
        f.u = u32x4_t{o[0], o[1], o[2], o[3]};
    } else if constexpr (KIND == kCacheQ4) {
        uint32_t o[4];
        nibbles_f16(k.d[g >> 1][(g & 1) * 2 + t16], magic, o);
        f.u = u32x4_t{o[0], o[1], o[2], o[3]};
    } else {
        f.u = k.d[t16 * G + g];
    }
    return f;
}

// values of dimensions 16 dt .. as operand, scales on them
template <int KIND, int G>
__device__ __forceinline__ Frag16 value_operand(const Half<KIND, G>& v, int dt, uint32_t magic)
{
    Frag16 f;
    if constexpr (cache_quantised(KIND)) {
        const int g = dt >> 1;
        uint32_t o[4];
        if constexpr (KIND == kCacheQ8) {
            unpack_q8_f16(v.d[g][2 * (dt & 1)], v.d[g][2 * (dt & 1) + 1], o);
        } else {
            const half2_t sub = {(_Float16)-1032.0f, (_Float16)-1032.0f}, mul = {(_Float16)0.0625f, (_Float16)0.0625f},
                          add = {(_Float16)-72.0f, (_Float16)-72.0f};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t w = v.d[g >> 1][(g & 1) * 2 + (i >> 1)] >> (8 * (i & 1));
                o[i] = dt & 1 ? as_u32(as_h2((w & 0x00F000F0u) | magic) * mul + add) : as_u32(as_h2((w & 0x000F000Fu) | magic) + sub);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) f.u[i] = as_u32(as_h2(o[i]) * as_h2(v.s[g][i]));
    } else {
        f.u = v.d[dt];
    }
    return f;
}

// Rows on an F16 cache are means of f16 values: what the rounding of their probabilities lifts past the largest of them is that number (NaN
// stays).  (Q8 and Q4 hold nothing near it, and fp32 sums of bf16 values none.)
__device__ __forceinline__ float within_f16(float x) { return x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x; }

template <int KIND>
__device__ __forceinline__ void store_row4(void* y, int dt, int64_t at, float4_t v)
{
    u32x2_t w;
    if constexpr (KIND == kCacheF16) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = within_f16(v[e]);
    }
    if (KIND == kCacheF16 || dt == kF16) w = u32x2_t{pack_half2(v[0], v[1]), pack_half2(v[2], v[3])};
    else w = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(y) + at) = w;
}

// Parts travel past the caches: stores and loads at system scope, nothing flushed, nothing invalidated.
__device__ __forceinline__ void put_float2(float* to, float x, float y)
{
    __hip_atomic_store(reinterpret_cast<uint64_t*>(to), __builtin_bit_cast(uint64_t, f32x2_t{x, y}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}
__device__ __forceinline__ void put_float4(float* to, float4_t v)
{
    put_float2(to, v[0], v[1]);
    put_float2(to + 2, v[2], v[3]);
}
__device__ __forceinline__ f32x2_t get_float2(const float* from)
{
    return __builtin_bit_cast(f32x2_t, __hip_atomic_load(reinterpret_cast<const uint64_t*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM));
}
__device__ __forceinline__ float4_t get_float4(const float* from)
{
    const f32x2_t a = get_float2(from), b = get_float2(from + 2);
    return float4_t{a[0], a[1], b[0], b[1]};
}

// The workgroup's part has been stored: whether it is the tile's last, and all of them are there.  The ticket is left at zero for the next call;
// parts are added in their order whoever arrives when.
__device__ __forceinline__ bool last_part(const AttnArgs& a, const Unit& u, unsigned* flag)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                  // mine has reached memory
    __syncthreads();                                                  // (and everybody is done reading LDS)
    if (threadIdx.x == 0) {
        const unsigned old = __hip_atomic_fetch_add(a.tickets + u.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool end = old + 1u == (unsigned)u.splits;
        if (end) __hip_atomic_store(a.tickets + u.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = end ? 1u : 0u;
    }
    __syncthreads();
    const bool end = *flag != 0u;
    __syncthreads();
    return end;
}

// Few rows: tiles of 16, four waves that take a part's blocks in turn, each with the next of its blocks on its way while it
// works on one.  Waves meet in LDS, the parts of a tile in slabs in memory: the part that is last adds them in order.  Bound by HBM where the
// context is long: 100001 tokens of a Q8 cache, 8 heads of 128, 218 MB: 45 - 51 us = 4.3 - 4.9 TB/s (three waves to a SIMD with one block each: 75), of
// F16 84, BF16 86, Q4 36; 48 conversations of up to 8192 tokens, Q8, 452 MB: 98 us = 4.6 TB/s, F16 158 = 5.4, BF16 165 = 5.2, Q4 74 = 3.2 (unpacking
// counts there); 4 heads of 256 F16 and BF16 159, Q8 123, Q4 97 (one wave to a SIMD, sums that move between the two halves of its registers).  Short
// contexts wait for one thing after another (1000 tokens: 8.1 - 8.9 us): lengths 1.5, products 1.3, the rest the table, the block and the way of the
// parts through memory.  Two tiles of rows to a workgroup, so that what a block needs is done once for 32 rows, have registers for one block at a
// time only: 8 drafts of 5 tokens with 7 heads each 24 us instead of 19.  (16.7 as it is: 35 rows are three tiles, and each unpacks every block.)
constexpr int kRows = 16;
template <int G>
struct RowsShape {
    static constexpr int kWaves = 4;
    static constexpr int kLds = kWaves * 2 * G * 64 * 16 + kWaves * 32 * 4;
    static constexpr int kSlab = kRows * 32 * G + 2 * kRows;                  // floats of a part: its rows, and their maxima and sums in pairs
};

template <int KIND, int G>
__device__ __forceinline__ void rows_part(const AttnArgs& a, float4_t* lds)       // lds: [waves][DT][64], then [waves][16] maxima and sums
{
    constexpr int kWaves = RowsShape<G>::kWaves;
    constexpr int DIM = 32 * G, BLOCK = cache_block_bytes(KIND, DIM), HALF = cache_half_bytes(KIND, DIM), DT = 2 * G;
    constexpr bool BF = KIND == kCacheBF16, SPLIT_P = KIND != kCacheF16;
    constexpr float kShift = BF ? 0.f : kShiftF16;
    float* const stats = reinterpret_cast<float*>(lds + kWaves * DT * 64);
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q4 = lane >> 4, r = lane & 15;
    const uint32_t magic = q4_magic_vgpr();
    Unit u;
    if (!find_unit<kRows, false>(a, blockIdx.x, &u)) return;
    const int64_t capacity = (int64_t)a.t.table_pages << (a.c.page_shift + 5);
    const int r0 = u.tile * kRows, rows = min(kRows, u.s.n * a.group - r0);
    const int p0 = u.s.len - u.s.n, i_first = r0 / a.group, i_last = (r0 + rows - 1) / a.group;
    int lo, hi;
    seen(a, p0 + i_first, p0 + i_last, capacity, &lo, &hi);
    const int each = (hi - lo) / u.splits, more = (hi - lo) % u.splits;
    const int first = lo + u.split * each + min(u.split, more), last = first + each + (u.split < more ? 1 : 0);
    // my row
    const bool real = r < rows;
    const int i = (r0 + (real ? r : 0)) / a.group, in_group = (r0 + (real ? r : 0)) - i * a.group;
    const int p = p0 + i;
    const int row_hi = real ? (int)min((int64_t)p, capacity - 1) : -1;
    const int row_lo = a.window && p >= a.window ? p - a.window + 1 : 0;
    const int all_hi = (int)min((int64_t)(p0 + i_first), capacity - 1);                       // every real row sees all of all_lo .. all_hi
    const int all_lo = a.window && p0 + i_last >= a.window ? p0 + i_last - a.window + 1 : 0;
    const int head = u.head * a.group + in_group;
    Frag16 qf[G];
    float c = a.scale;
    {
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)(u.s.row0 + i) * a.q_stride + head * DIM + 8 * q4;
#pragma unroll
        for (int g = 0; g < G; g++) qf[g].u = real ? *reinterpret_cast<const u32x4_t*>(q + 32 * g) : u32x4_t{0u, 0u, 0u, 0u};
        if (cache_quantised(KIND) && a.qdt == kBF16) {                // to f16: the row's largest at 2^14 .. 2^15
            float x[8 * G], top = 0.f;
#pragma unroll
            for (int e = 0; e < 8 * G; e++) {
                const uint32_t w = qf[e >> 3].u[(e & 7) >> 1];
                x[e] = __builtin_bit_cast(float, e & 1 ? w & 0xffff0000u : w << 16);
                top = fmaxf(top, fabsf(x[e]));
            }
            top = fmaxf(top, other_quarter<16>(top));
            top = fmaxf(top, other_quarter<32>(top));
            const float f = row_power(top, &c);
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int j = 0; j < 4; j++) qf[g].u[j] = pack_half2(x[8 * g + 2 * j] * f, x[8 * g + 2 * j + 1] * f);
        }
    }
    const float lag = fminf((BF ? kAhead : kLagF16) / c, 1e30f);
    // my blocks are first + wv + kWaves i; a lane asks for the page of one of 64 of them, those that have one are worked on
    const int32_t* const table = a.t.tables + (int64_t)u.b * a.t.table_pages;
    const int in_page = (1 << a.c.page_shift) - 1;
    int base = first + wv, page = -1;
    uint64_t there = 0;
    auto look_up = [&]() {
        for (; base < last; base += 64 * kWaves) {
            const int blk = base + lane * kWaves;
            page = blk < last ? table[blk >> a.c.page_shift] : -1;
            there = __ballot((unsigned)page < (unsigned)a.c.pages);
            if (there) return;
        }
    };
    auto next_block = [&](int* blk) -> const uint8_t* {
        if (!there) {
            base += 64 * kWaves;
            look_up();
            if (!there) return nullptr;
        }
        const int l = __builtin_ctzll(there);
        there &= there - 1;
        *blk = base + l * kWaves;
        const int id = __builtin_amdgcn_readlane(page, l);
        return a.c.base + id * a.c.page_bytes + (int64_t)((u.head << a.c.page_shift) + (*blk & in_page)) * BLOCK;
    };
    float4_t y[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) y[d] = float4_t{0.f, 0.f, 0.f, 0.f};
    const float none = -__builtin_inff();
    float m = none, l = 0.f;                                          // m: of scores without their factor
    Half<KIND, G> k0, v0, k1, v1;
    int blk = 0;
    look_up();
    const uint8_t* at = there ? next_block(&blk) : nullptr;
    if (at) {
        k0.load(at, lane);
        v0.load(at + HALF, lane);
    }
    // one block; the next one's keys and values go to nk, nv
    auto work = [&](const Half<KIND, G>& k, const Half<KIND, G>& v, Half<KIND, G>& nk, Half<KIND, G>& nv) __attribute__((always_inline)) {
        int next_blk = 0;
        const uint8_t* const next = next_block(&next_blk);
        if (next) {
            nk.load(next, lane);
            nv.load(next + HALF, lane);
        }
        float4_t s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < G; g++) {
                const Frag16 kf = key_operand<KIND, G>(k, t, g, magic);
                if constexpr (cache_quantised(KIND)) {
                    const float4_t part = mfma16<KIND>(kf, qf[g], float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const half2_t sc = as_h2(k.s[g][2 * t + (e >> 1)]);
                        s[t][e] = __builtin_fmaf((float)sc[e & 1], part[e], s[t][e]);
                    }
                } else {
                    s[t] = mfma16<KIND>(kf, qf[g], s[t]);
                }
            }
        }
        const int tok = blk * kBlockTokens + 16 * (q4 >> 1) + 4 * (q4 & 1);
        if (blk * kBlockTokens < all_lo || blk * kBlockTokens + 31 > all_hi) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int j = tok + 8 * t + e;
                    if (j < row_lo || j > row_hi) s[t][e] = none;
                }
        }
        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        top = fmaxf(top, other_quarter<16>(top));
        top = fmaxf(top, other_quarter<32>(top));
        if (__ballot(top > (BF ? m : m + lag))) {
            float to = BF ? top + lag : __builtin_fmaf(lag, -kRowsBelow / kLagF16, top);
            if (!BF && top - to > lag) to = top;                      // (where fp32 scores are that far from each other)
            const float now = top > (BF ? m : m + lag) ? to : m;
            const float f = m == none ? 0.f : exp2_fast((m - now) * c);
            m = now;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; d++) y[d] *= f;
        }
        const float least = m == none ? 0.f : m;                      // (taken off before the factor comes in: m c may be known to no more than its 24 bits)
        Frag16 ph, pl;
        float pr[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            pr[e] = exp2_fast(__builtin_fmaf(s[e >> 2][e & 3] - least, c, kShift));
            l += pr[e];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (BF) {
                ph.u[j] = pack_bf16x2(pr[2 * j], pr[2 * j + 1]);
                pl.u[j] = pack_bf16x2(pr[2 * j] - __builtin_bit_cast(float, ph.u[j] << 16), pr[2 * j + 1] - __builtin_bit_cast(float, ph.u[j] & 0xffff0000u));
            } else {
                ph.u[j] = pack_half2(pr[2 * j], pr[2 * j + 1]);
                if constexpr (SPLIT_P) pl.u[j] = pack_half2(pr[2 * j] - (float)as_h2(ph.u[j])[0], pr[2 * j + 1] - (float)as_h2(ph.u[j])[1]);
            }
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const Frag16 vf = value_operand<KIND, G>(v, d, magic);
            y[d] = mfma16<KIND>(vf, ph, y[d]);
            if constexpr (SPLIT_P) y[d] = mfma16<KIND>(vf, pl, y[d]);
        }
        at = next;
        blk = next_blk;
    };
    while (at) {
        work(k0, v0, k1, v1);
        if (!at) break;
        work(k1, v1, k0, v0);
    }
    l += other_quarter<16>(l);
    l += other_quarter<32>(l);
    // waves meet
    if (lane < 16) {
        stats[wv * 16 + lane] = m * c;
        stats[kWaves * 16 + wv * 16 + lane] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; d++) lds[(wv * DT + d) * 64 + lane] = y[d];
    __syncthreads();
    float top = none, sum = 0.f, f[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; w++) top = fmaxf(top, stats[w * 16 + r]);
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        const float mw = stats[w * 16 + r];
        f[w] = mw == none ? 0.f : exp2_fast(mw - top);
        sum += f[w] * stats[kWaves * 16 + w * 16 + r];                // (a row of NaN has a sum of NaN and no maximum)
    }
    const int64_t row_at = ((int64_t)(u.s.row0 + i) * a.c.kv_heads * a.group + head) * DIM + 4 * q4;
    constexpr int SLAB = RowsShape<G>::kSlab;
    float* const slab = a.slabs + (size_t)u.slab * SLAB;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    for (int d = wv; d < DT; d += kWaves) {
        float4_t o = lds[d * 64 + lane] * f[0];                       // (sums of a wave without a maximum are zeros, or its row is NaN)
#pragma unroll
        for (int w = 1; w < kWaves; w++) o += lds[(w * DT + d) * 64 + lane] * f[w];
        if (!real) continue;
        if (u.splits == 1) store_row4<KIND>(a.y, a.qdt, row_at + 16 * d, o * inv);
        else put_float4(slab + r * DIM + 16 * d + 4 * q4, o);
    }
    if (u.splits == 1) return;
    if (threadIdx.x < 16) put_float2(slab + kRows * DIM + 2 * r, top, sum);
    if (!last_part(a, u, reinterpret_cast<unsigned*>(lds))) return;
    // The rows of all parts: threads share out the rows' float4s, and the parts where there are more threads; everything is asked for at once (of
    // more than 8 rows of 128 two float4s to a thread and six parts: a second round would wait for memory again, 1.3 us).
    constexpr int THREADS = 64 * kWaves, QUADS = DIM / 4;
    const int items = rows * QUADS, runs = max(1, THREADS / items);
    const float* const of_tile = slab - (size_t)u.split * SLAB;
    auto join = [&](auto at_once, auto parts_ahead) __attribute__((always_inline)) {
        constexpr int N = decltype(at_once)::value, AHEAD = decltype(parts_ahead)::value;
        for (int it0 = 0; it0 < items; it0 += N * THREADS) {
            const int run = N > 1 || runs == 1 ? 0 : threadIdx.x / items;
            bool mine[N];
            int row[N], quad[N];
            float m2[N], l2[N];
            float4_t o[N];
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int it = it0 + n * THREADS + threadIdx.x - run * items;
                mine[n] = it < items && run < runs;
                row[n] = mine[n] ? it / QUADS : 0;
                quad[n] = mine[n] ? it - row[n] * QUADS : 0;
                m2[n] = none;
                l2[n] = 0.f;
                o[n] = float4_t{0.f, 0.f, 0.f, 0.f};
            }
            for (int e0 = run; e0 < u.splits && mine[0]; e0 += AHEAD * runs) {
                float4_t part[N][AHEAD];
                f32x2_t of[N][AHEAD];
#pragma unroll
                for (int e = 0; e < AHEAD; e++) {
                    const float* const from = of_tile + (size_t)min(e0 + e * runs, u.splits - 1) * SLAB;
#pragma unroll
                    for (int n = 0; n < N; n++) {
                        part[n][e] = get_float4(from + row[n] * DIM + 4 * quad[n]);
                        of[n][e] = get_float2(from + kRows * DIM + 2 * row[n]);
                    }
                }
#pragma unroll
                for (int n = 0; n < N; n++) {
                    float now = m2[n];
#pragma unroll
                    for (int e = 0; e < AHEAD; e++) now = fmaxf(now, of[n][e][0]);
                    const float old = m2[n] == none ? 0.f : exp2_fast(m2[n] - now);
                    o[n] *= old;
                    l2[n] *= old;
                    m2[n] = now;
#pragma unroll
                    for (int e = 0; e < AHEAD; e++) {
                        const float fe = of[n][e][0] == none || e0 + e * runs >= u.splits ? 0.f : exp2_fast(of[n][e][0] - now);
                        o[n] += part[n][e] * fe;
                        l2[n] += e0 + e * runs >= u.splits ? 0.f : of[n][e][1] * fe;
                    }
                }
            }
            if (N == 1 && runs > 1) {                                // (all in one round)
                float* const pairs = reinterpret_cast<float*>(lds + THREADS);
                lds[threadIdx.x] = o[0];
                pairs[2 * threadIdx.x] = m2[0];
                pairs[2 * threadIdx.x + 1] = l2[0];
                __syncthreads();
                if (run) return;
                for (int e = 1; e < runs; e++) {
                    const int at = threadIdx.x + e * items;
                    const float me = pairs[2 * at], now = fmaxf(m2[0], me);
                    const float fo = m2[0] == none ? 0.f : exp2_fast(m2[0] - now), fe = me == none ? 0.f : exp2_fast(me - now);
                    o[0] = o[0] * fo + lds[at] * fe;
                    l2[0] = l2[0] * fo + pairs[2 * at + 1] * fe;
                    m2[0] = now;
                }
            }
#pragma unroll
            for (int n = 0; n < N; n++) {
                if (!mine[n]) continue;
                const int at = r0 + row[n], of_token = at / a.group;
                const float by = l2[n] == 0.f ? 0.f : 1.0f / l2[n];
                store_row4<KIND>(a.y, a.qdt, (((int64_t)u.s.row0 + of_token) * a.c.kv_heads * a.group + u.head * a.group + at - of_token * a.group) * DIM + 4 * quad[n],
                           o[n] * by);
            }
        }
    };
    if (items > THREADS) join(std::integral_constant<int, 2>{}, std::integral_constant<int, 6>{});
    else join(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
}

template <int KIND, int G>
__global__ __launch_bounds__(64 * RowsShape<G>::kWaves, G <= 4 ? 2 : 1) void attention_rows_kernel(AttnArgs a)
{
    extern __shared__ float4_t lds[];
    rows_part<KIND, G>(a, lds);
}

// ---- many rows ------------------------------------------------------------------------------------------------

typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <int KIND>
__device__ __forceinline__ f32x16_t mfma32(Frag16 a, Frag16 b, f32x16_t c)
{
    if constexpr (KIND == kCacheBF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.b, b.b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
}

// 16 bytes per lane from base + off (the lane's own) to LDS bytes lds_off + 16 * lane, past the registers
__device__ __forceinline__ void copy_to_lds(uint32_t lds_off, const void* base, uint32_t off)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds_off)), "v"(off), "s"(base));
}

template <int KIND, int G>
struct TileShape {
    static constexpr int kBlocks = G <= 4 ? 2 : 1;            // blocks of a step
    // Waves, each with 32 rows: eight where they share the work of unpacking (Q8, Q4: 216 us instead of 308 for 512 rows after 15872 tokens) or where
    // three steps of copies fit a CU once only (heads of 128: 2040 us instead of 2150 for 4096 rows after 28672 tokens); else four, in more workgroups
    // (heads of 64: 62 us instead of 69 for 2000 rows)
    static constexpr int kWaves = cache_quantised(KIND) ? (G <= 4 ? 8 : 4) : (G == 4 ? 8 : 4);
    static constexpr int kRows = 32 * kWaves;
    // Steps of keys, and of values, that LDS holds: three, so that copies have two steps to arrive in; quantised bytes wait in registers instead
    static constexpr int kRing = cache_quantised(KIND) ? 2 : 3;
    static constexpr int kPerCu = G > 4 || kWaves == 8 ? 1 : 2;              // workgroups
    static constexpr int kTarget = 256 * kPerCu, kMostExtra = 2 * kTarget;
    static constexpr int kHalf = kBlocks * kBlockTokens * 32 * G * 2;         // bytes of a step's keys, or values
    static constexpr int kLds = std::max(2 * kRing * kHalf, RowsShape<G>::kLds);         // (a single sequence of few rows)
    static constexpr int kSlab = kRows * 32 * G + 2 * kRows;  // floats of a part
};

// A step's keys or values on their way to LDS in the order of 32 x 32 x 16 operands: [block][dimensions 16 step ..][half of 8][32 tokens] 16 B,
// [block][dimensions 32 dtile ..][16 tokens j][half][32 dimensions] 16 B.  16-bit caches: copied there, a lane's 16 B each from its place.
// Q8, Q4: asked for in registers, and turned into f16 (scales on them, rounded once) when the step ahead is done.
template <int KIND, int G>
struct Stage {
    typedef TileShape<KIND, G> T;
    static constexpr bool kQuant = cache_quantised(KIND);
    static constexpr int N = kQuant ? Half<KIND, G>::N : 2 * G;                          // 1 KiB pieces of a block's half
    static constexpr int PER = (T::kBlocks * N + T::kWaves - 1) / T::kWaves;             // pieces per wave
    static_assert(kQuant || T::kBlocks * N % T::kWaves == 0, "every wave has as many copies in flight as its waits count");
    struct Piece {
        u32x4_t d, s[2];
    };
    Piece raw[kQuant ? PER : 1];

    // pieces from .. to of that half (VALUES: the values); where: LDS byte offset
    template <bool VALUES>
    __device__ __forceinline__ void ask(const uint8_t* const (&block)[T::kBlocks], uint32_t where, int wv, int lane, int from_piece = 0, int to_piece = PER)
    {
#pragma unroll
        for (int e = from_piece; e < to_piece; e++) {
            const int p = wv + e * T::kWaves;
            if (T::kBlocks * N % T::kWaves && p >= T::kBlocks * N) break;
            const int bl = T::kBlocks == 1 ? 0 : p / N, i = p - bl * N;
            const uint8_t* const from = T::kBlocks == 1 || bl == 0 ? block[0] : block[T::kBlocks - 1];
            if constexpr (!kQuant) {
                // (a lane's place in a piece is the same in all of them: one register for the keys' offsets, one for the values')
                const uint32_t off = VALUES ? (lane >> 4 & 1) * 1024 + (lane & 15) * 16 + (lane >> 5) * 256
                                            : ((lane >> 3 & 1) * G * 64 + ((lane & 31) >> 4 << 3 | (lane & 7)) + (lane >> 5) * 16) * 16;
                const uint8_t* const piece = from + (VALUES ? cache_half_bytes(KIND, 32 * G) + (i >> 1) * 2048 : (i >> 1) * 1024) + (i & 1) * 512;
                copy_to_lds(where + p * 1024, piece, off);
            } else {
                const uint8_t* const src = from + (VALUES ? cache_half_bytes(KIND, 32 * G) : 0);
                const uint8_t* const sc = src + cache_data_bytes(KIND, 32 * G);
                Piece& r = raw[e];
                if (KIND == kCacheQ4 && (G & 1) && i == N - 1) {
                    const u32x2_t v = *reinterpret_cast<const u32x2_t*>(src + i * 1024 + lane * 8);
                    r.d = u32x4_t{v[0], v[1], 0u, 0u};
                } else {
                    r.d = *reinterpret_cast<const u32x4_t*>(src + i * 1024 + lane * 16);
                }
                constexpr int GROUPS = KIND == kCacheQ4 ? 2 : 1;
#pragma unroll
                for (int gg = 0; gg < GROUPS; gg++) {
                    const int g = min(GROUPS * i + gg, G - 1);
                    if (VALUES) r.s[gg] = *reinterpret_cast<const u32x4_t*>(sc + (g * 4 + (lane >> 4)) * 16);
                    else {
                        const uint16_t* at = reinterpret_cast<const uint16_t*>(sc) + (g * 4 + ((lane & 15) >> 2)) * 8 + (lane & 3);
                        r.s[0][2 * gg] = at[0] * 0x10001u;
                        r.s[0][2 * gg + 1] = at[4] * 0x10001u;
                    }
                }
            }
        }
    }
    template <bool VALUES>
    __device__ __forceinline__ void put(uint8_t* lds, uint32_t where, int wv, int lane, uint32_t magic)
    {
        if constexpr (kQuant) {
            const int m = lane & 15, q4 = lane >> 4;
#pragma unroll
            for (int e = 0; e < PER; e++) {
                const int p = wv + e * T::kWaves;
                if (T::kBlocks * N % T::kWaves && p >= T::kBlocks * N) break;
                const int bl = T::kBlocks == 1 ? 0 : p / N, i = p - bl * N;
                const Piece& r = raw[e];
                constexpr int GROUPS = KIND == kCacheQ4 ? 2 : 1;
#pragma unroll
                for (int gg = 0; gg < GROUPS; gg++) {
                    const int g = GROUPS * i + gg;
                    if (GROUPS * N != G && g >= G) break;
#pragma unroll
                    for (int t = 0; t < 2; t++) {             // keys: tile of 16 tokens; values: tile of 16 dimensions
                        uint32_t o[4];
                        if constexpr (KIND == kCacheQ8) unpack_q8_f16(r.d[2 * t], r.d[2 * t + 1], o);
                        else if (!VALUES) nibbles_f16(r.d[2 * gg + t], magic, o);
                        else {
                            const half2_t sub = {(_Float16)-1032.0f, (_Float16)-1032.0f}, mul = {(_Float16)0.0625f, (_Float16)0.0625f},
                                          add = {(_Float16)-72.0f, (_Float16)-72.0f};
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const uint32_t w = r.d[2 * gg + (k >> 1)] >> (8 * (k & 1));
                                o[k] = t ? as_u32(as_h2((w & 0x00F000F0u) | magic) * mul + add) : as_u32(as_h2((w & 0x000F000Fu) | magic) + sub);
                            }
                        }
                        u32x4_t v;
#pragma unroll
                        for (int k = 0; k < 4; k++) v[k] = as_u32(as_h2(o[k]) * as_h2(VALUES ? r.s[gg][k] : r.s[0][2 * gg + t]));
                        const int at = VALUES ? ((bl * G + g) * 2 + (q4 >> 1)) * 64 + t * 16 + m + (q4 & 1) * 32
                                              : (bl * 2 * G + 2 * g + (q4 >> 1)) * 64 + ((m >> 3) << 4 | t << 3 | (m & 7)) + (q4 & 1) * 32;
                        *reinterpret_cast<u32x4_t*>(lds + where + at * 16) = v;
                    }
                }
            }
        }
    }
};

// Many rows: a workgroup's waves have 32 rows each and go through the same blocks, 64 tokens (a head of 256: 32) a step.  While P of a step
// is formed the scores of the next are multiplied: its keys are in LDS one step earlier than its values.  Bound by issue: matrix instructions
// are 57 % of a SIMD's cycles, vector instructions 50, and the card clocks down to 1.64 GHz under them (4096 rows, 32 heads of 128, after 28672 tokens of F16:
// 1850 - 1975 us = 1.04 - 1.11 PFLOP/s; the library's product of 8192 x 8192 x 8192 1.27).  512 rows of 16384 tokens: F16 154 us, BF16 146, Q8 164 = 0.83
// PFLOP/s, Q4 161 (heads of 64: 99, 95, 104, 106; 96: 128, 123, 139, 141; 4 of 256: 167, 160, 204, 200).  Q8 and Q4: each value is also unpacked, once for 128 or
// 256 rows, and their loads are flat ones - a block's address comes from two lane reads, and the compiler cannot tell that it is global memory -: they
// count with the LDS reads, so that the operands fetched ahead are waited for to the last one five to ten times a step.  Short prompts are as long as the tile that sees the most (2000 rows, heads of 64: 34 us, 25 of them
// that tile's 32 steps).
template <int KIND, int G>
__global__ __launch_bounds__((64 * TileShape<KIND, G>::kWaves), (TileShape<KIND, G>::kWaves * TileShape<KIND, G>::kPerCu / 4)) void attention_tiles_kernel(AttnArgs a)
{
    typedef TileShape<KIND, G> T;
    constexpr int DIM = 32 * G, BLOCK = cache_block_bytes(KIND, DIM), ROWS = T::kRows, BL = T::kBlocks;
    constexpr bool BF = KIND == kCacheBF16;
    constexpr float kShift = BF ? 0.f : kShiftF16;
    extern __shared__ float4_t lds[];                                 // keys of kRing steps, values of as many
    uint8_t* const bytes = reinterpret_cast<uint8_t*>(lds);
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, r = lane & 31;
    const uint32_t magic = q4_magic_vgpr();
    Unit u;
    if (!find_unit<ROWS, true>(a, blockIdx.x, &u)) {
        // A single sequence is launched once: that it has few rows only the device knows (a launch of the rows kernel beside this one: 2000 rows of
        // heads of 64 33.8 -> 36.8 us)
        if (a.t.seqs == 1 && wv < RowsShape<G>::kWaves && seq_of(a.t, 0).n * a.group <= a.few) rows_part<KIND, G>(a, lds);
        return;
    }
    const int64_t capacity = (int64_t)a.t.table_pages << (a.c.page_shift + 5);
    const int all_rows = u.s.n * a.group, p0 = u.s.len - u.s.n;
    const int w0 = u.tile * ROWS, wg_rows = min(ROWS, all_rows - w0);
    int lo, hi;
    seen(a, p0 + w0 / a.group, p0 + (w0 + wg_rows - 1) / a.group, capacity, &lo, &hi);
    const int each = (hi - lo) / u.splits, more = (hi - lo) % u.splits;
    const int first = lo + u.split * each + min(u.split, more), last = first + each + (u.split < more ? 1 : 0);
    const int steps = (last - first + BL - 1) / BL;
    // my row, and what all of this wave's rows see
    const int r0 = w0 + wv * 32, rows = max(0, min(32, all_rows - r0));
    const bool real = r < rows;
    const int i = (real ? r0 + r : w0) / a.group, in_group = (real ? r0 + r : w0) - i * a.group;
    const int p = p0 + i;
    const int row_hi = real ? (int)min((int64_t)p, capacity - 1) : -1;
    const int row_lo = a.window && p >= a.window ? p - a.window + 1 : 0;
    int all_hi = 0x7fffffff, all_lo = 0;                             // every row sees all_lo .. all_hi (a wave without rows: nobody looks at what it sees)
    if (rows) {
        const int pf = p0 + r0 / a.group, pl = p0 + (r0 + rows - 1) / a.group;
        all_hi = (int)min((int64_t)pf, capacity - 1);
        all_lo = a.window && pl >= a.window ? pl - a.window + 1 : 0;
    }
    const int head = u.head * a.group + in_group;
    Frag16 qf[2 * G];
    float c = a.scale;
    {
        const uint16_t* q = static_cast<const uint16_t*>(a.q) + (int64_t)(u.s.row0 + i) * a.q_stride + head * DIM + 8 * h;
#pragma unroll
        for (int k = 0; k < 2 * G; k++) qf[k].u = real ? *reinterpret_cast<const u32x4_t*>(q + 16 * k) : u32x4_t{0u, 0u, 0u, 0u};
        if (cache_quantised(KIND) && a.qdt == kBF16) {
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * G; k++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    top = fmaxf(top, fmaxf(fabsf(__builtin_bit_cast(float, qf[k].u[j] << 16)), fabsf(__builtin_bit_cast(float, qf[k].u[j] & 0xffff0000u))));
            top = fmaxf(top, other_quarter<32>(top));
            const float f = row_power(top, &c);
#pragma unroll
            for (int k = 0; k < 2 * G; k++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    qf[k].u[j] = pack_half2(__builtin_bit_cast(float, qf[k].u[j] << 16) * f, __builtin_bit_cast(float, qf[k].u[j] & 0xffff0000u) * f);
        }
    }
    const float lag = fminf((BF ? kAhead : kLagF16) / c, 1e30f);
    const int32_t* const table = a.t.tables + (int64_t)u.b * a.t.table_pages;
    const int in_page = (1 << a.c.page_shift) - 1;
    // Where the part's blocks lie, a lane for each of 64 from `from_block` on, counted from the part's first (a block that is not there is
    // read from page 0: finite numbers, which nobody sees), and the pages of the 64 behind them.  Scalar arithmetic of 64 bits for every step and
    // wave, in its place, took a fifth of a step of heads of 64.
    auto pages_from = [&](int i) {
        const int blk = first + i + lane;
        return blk < last ? table[blk >> a.c.page_shift] : -1;
    };
    int from_block = 0, far_ids = pages_from(64);
    uint32_t at_lo, at_hi;
    uint64_t there;
    auto look_up = [&](int id) {
        const bool real_page = (unsigned)id < (unsigned)a.c.pages;
        there = __ballot(real_page);
        const uint64_t at = reinterpret_cast<uint64_t>(a.c.base) + (uint64_t)(real_page ? id : 0) * (uint64_t)a.c.page_bytes +
                            (uint64_t)((u.head << a.c.page_shift) + ((first + from_block + lane) & in_page)) * (uint64_t)BLOCK;
        at_lo = (uint32_t)at;
        at_hi = (uint32_t)(at >> 32);
    };
    look_up(pages_from(0));
    // of a step within those 64
    auto blocks_of = [&](int step, const uint8_t* (&at)[BL]) {
#pragma unroll
        for (int b = 0; b < BL; b++) {
            const int i = step * BL + b - from_block;
            at[b] = reinterpret_cast<const uint8_t*>((uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, i) << 32 | (uint32_t)__builtin_amdgcn_readlane(at_lo, i));
        }
    };
    f32x16_t y[G];
#pragma unroll
    for (int d = 0; d < G; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) y[d][e] = 0.f;
    const float none = -__builtin_inff();
    float m = none, l = 0.f;
    auto key_at = [&](uint32_t where, int k, int b) __attribute__((always_inline)) {
        Frag16 f;
        f.u = *reinterpret_cast<const u32x4_t*>(bytes + where + (b * 2 * G + k) * 1024 + lane * 16);
        return f;
    };
    auto value_at = [&](uint32_t where, int k, int d) __attribute__((always_inline)) {
        Frag16 f;
        f.u = *reinterpret_cast<const u32x4_t*>(bytes + where + (((k >> 1) * G + d) * 2 + (k & 1)) * 1024 + lane * 16);
        return f;
    };
    const f32x16_t zeros = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    constexpr bool QUANT = cache_quantised(KIND);
    constexpr int R = T::kRing;
    constexpr uint32_t K0 = 0, V0 = R * T::kHalf;
    constexpr int N = 2 * G * BL;                                    // matrix instructions of a step's scores, and of its values
    Stage<KIND, G> ks, vs;
    constexpr int AHEAD = QUANT ? 3 : R;                             // keys of step t + AHEAD are asked for in step t, values of t + AHEAD - 2
    const uint8_t* at[BL];
    const uint8_t* queue[3][BL];                                     // blocks of steps t + AHEAD - 2 ..
    uint32_t present;                                                // BL bits for each step from t on: whether its blocks are in a page
    f32x16_t s[BL];                                                  // scores of step t
    Frag16 pf[2 * BL];                                               // P of step t - 1, not yet on the sums
#pragma unroll
    for (int k = 0; k < 2 * BL; k++) pf[k].u = u32x4_t{0u, 0u, 0u, 0u};
    // Keys of step t + 1 and values of step t - 1 are in LDS when step t begins: step j in place j of R, counted round.
    auto fill = [&](bool values, int step, int place) __attribute__((always_inline)) {
        blocks_of(step, at);
        const uint32_t where = (values ? V0 : K0) + place * T::kHalf;
        if (values) vs.template ask<true>(at, where, wv, lane), vs.template put<true>(bytes, where, wv, lane, magic);
        else ks.template ask<false>(at, where, wv, lane), ks.template put<false>(bytes, where, wv, lane, magic);
    };
    if (steps) {
#pragma unroll
        for (int j = 0; j < R; j++) fill(false, j, j);
        fill(true, 0, R - 1);                                        // (values of "step -1", for a P of zeros: any finite ones)
        if constexpr (R == 3) fill(true, 0, 0);
        if constexpr (QUANT) {                                       // (turned and put into LDS in step 0)
            blocks_of(2, at);
            ks.template ask<false>(at, 0, wv, lane);
            blocks_of(0, at);
            vs.template ask<true>(at, 0, wv, lane);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int b = 0; b < BL; b++)
#pragma unroll
            for (int k = 0; k < 2 * G; k++) s[b] = mfma32<KIND>(key_at(K0, k, b), qf[k], k ? s[b] : zeros);
        __syncthreads();                                             // (keys of step R go where those of step 0 were)
    }
    blocks_of(AHEAD - 2, queue[0]);
    blocks_of(AHEAD - 1, queue[1]);
    present = (uint32_t)there & ((1u << AHEAD * BL) - 1u);
    uint32_t ring[R];                                                // places of steps t, t + 1, .. (and t - 1, the last)
#pragma unroll
    for (int j = 0; j < R; j++) ring[j] = j * T::kHalf;
    float top = none;
    constexpr uint32_t ALL = (1u << BL) - 1u;
    // The exponent is s c - m c in one instruction.  Where m c is so large that its rounding counts (far), m is taken off the scores first, and every
    // step begins outside of the inner loop.
    float off = kShift;
    bool far = false;
    // whether some row does not see all of step t's tokens
    auto hides = [&](int t) {
        const int tok = (first + t * BL) * kBlockTokens;
        return (present & ALL) != ALL || tok < all_lo || tok + BL * kBlockTokens - 1 > all_hi;
    };
    // Steps whose rows see everything and whose maxima have grown by less than the lag follow each other in the inner loop; at any other its scores
    // are masked, P that waits is added and the sums are scaled outside of it.  (In a branch of the loop the sums had two homes, 64
    // registers and as many moves.)
    for (int t = 0; t < steps;) {
        if (hides(t)) {
            const int tok = (first + t * BL) * kBlockTokens;
#pragma unroll
            for (int b = 0; b < BL; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int j = tok + b * kBlockTokens + 8 * (e >> 2) + 4 * h + (e & 3);
                    if (j < row_lo || j > row_hi || !(present >> b & 1)) s[b][e] = none;
                }
        }
        top = s[0][0];
#pragma unroll
        for (int b = 0; b < BL; b++)
#pragma unroll
            for (int e = b ? 0 : 1; e < 16; e++) top = fmaxf(top, s[b][e]);
        top = fmaxf(top, other_quarter<32>(top));
        const uint32_t before = V0 + ring[R - 1];
#pragma unroll
        for (int i = 0; i < N; i++) y[i % G] = mfma32<KIND>(value_at(before, i / G, i % G), pf[i / G], y[i % G]);
#pragma unroll
        for (int k = 0; k < 2 * BL; k++) pf[k].u = u32x4_t{0u, 0u, 0u, 0u};
        const float up = top > (BF ? m : m + lag) ? (BF ? top + lag : top) : m;
        const float f = m == none ? 0.f : exp2_fast((m - up) * c);
        m = up;
        l *= f;
#pragma unroll
        for (int d = 0; d < G; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) y[d][e] *= f;
        const float largest = m == none ? 0.f : m;
        far = __ballot(fabsf(largest * c) > kFar);
        off = kShift - (far ? 0.f : largest * c);
        if (far) {
#pragma unroll
            for (int b = 0; b < BL; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[b][e] -= largest;
        }
        do {
            // P of step t while the values of step t - 1 are multiplied, and behind that the first scores of step t + 1 (of none: of what is in LDS,
            // and nobody looks at them).  A wave issues in order, and a 32 x 32 instruction takes as long as eight others: the order below puts
            // about a pair's exponentials behind each.
            // Copies for steps to come (past the end they are read from page 0 and nobody looks at them), spread over the step: a CU takes 64 bytes a cycle
            // from its L1, and asked for in a row they held the waves up for 1000 of a step's 2500 cycles.
            blocks_of(t + AHEAD, queue[2]);
            present |= (uint32_t)(there >> ((t + AHEAD) * BL - from_block) & ALL) << AHEAD * BL;
            constexpr int SLOTS = 2 * N, PER = Stage<KIND, G>::PER;
            auto copies = [&](int i) __attribute__((always_inline)) {
                if constexpr (QUANT) {                               // what was asked for a step ago, and the next of it
                    if (i == N / 4) {
                        ks.template put<false>(bytes, K0 + ring[0], wv, lane, magic);
                        ks.template ask<false>(queue[2], 0, wv, lane);
                    }
                    if (i == 3 * N / 4) {
                        vs.template put<true>(bytes, V0 + ring[0], wv, lane, magic);
                        vs.template ask<true>(queue[0], 0, wv, lane);
                    }
                } else {
                    const int from = i * 2 * PER / SLOTS, to = (i + 1) * 2 * PER / SLOTS;
                    if (from < PER) ks.template ask<false>(queue[2], K0 + ring[0], wv, lane, from, to < PER ? to : PER);
                    if (to > PER) vs.template ask<true>(queue[0], V0 + ring[R - 2], wv, lane, from > PER ? from - PER : 0, to - PER);
                }
            };
            const uint32_t values_at = V0 + ring[R - 1], keys_at = K0 + ring[1];
            constexpr int PAIRS = 8 * BL, EARLY = BL == 2 ? 11 : PAIRS, LOOK = 6;
            Frag16 frag[2 * N], pn[2 * BL];
            // operands in the order of their use: values, then keys of the first block and of the second
            auto fetch = [&](int i) __attribute__((always_inline)) {
                if (i < N) frag[i] = value_at(values_at, i / G, i % G);
                else if (i < 2 * N) frag[i] = key_at(keys_at, (i - N) % (2 * G), (i - N) / (2 * G));
            };
            float sums[4] = {0.f, 0.f, 0.f, 0.f};
            auto pairs = [&](int from, int to) __attribute__((always_inline)) {
#pragma unroll
                for (int i = from; i < to; i++) {
                    const int b = i >> 3, e = 2 * (i & 7);
                    const float x0 = exp2_fast(__builtin_fmaf(s[b][e], c, off)), x1 = exp2_fast(__builtin_fmaf(s[b][e + 1], c, off));
                    sums[i & 3] += x0 + x1;
                    uint32_t w = KIND == kCacheBF16 ? pack_bf16x2(x0, x1) : pack_half2(x0, x1);
                    asm volatile("" : "+v"(w));                      // (here, and not where the next step needs it)
                    pn[i >> 2].u[i & 3] = w;
                }
            };
#pragma unroll
            for (int i = 0; i < LOOK; i++) fetch(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < N; i++) {
                fetch(i + LOOK);
                y[i % G] = mfma32<KIND>(frag[i], pf[i / G], y[i % G]);
                pairs(i * EARLY / N, (i + 1) * EARLY / N);
                copies(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            // scores: all of the first block, then of the second
            f32x16_t sn[BL];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int k = i % (2 * G), b = i / (2 * G);
                fetch(N + i + LOOK);
                sn[b] = mfma32<KIND>(frag[N + i], qf[k], k ? sn[b] : zeros);
                if (b == 0) pairs(EARLY + k * (PAIRS - EARLY) / (2 * G), EARLY + (k + 1) * (PAIRS - EARLY) / (2 * G));
                copies(N + i);
                __builtin_amdgcn_sched_barrier(0);
            }
            l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
            top = sn[0][0];
#pragma unroll
            for (int b = 0; b < BL; b++)
#pragma unroll
                for (int e = b ? 0 : 1; e < 16; e++) top = fmaxf(top, sn[b][e]);
            top = fmaxf(top, other_quarter<32>(top));
#pragma unroll
            for (int b = 0; b < BL; b++) s[b] = sn[b];
#pragma unroll
            for (int k = 0; k < 2 * BL; k++) pf[k] = pn[k];
            // what was asked for before this step is there (Q8, Q4: compiler's loads, and it waits for them)
            if constexpr (!QUANT) asm volatile("s_waitcnt vmcnt(%0)" ::"i"((R - 2) * 2 * Stage<KIND, G>::PER) : "memory");
            __syncthreads();
            const uint32_t first_place = ring[0];
#pragma unroll
            for (int j = 0; j + 1 < R; j++) ring[j] = ring[j + 1];
            ring[R - 1] = first_place;
            t++;
            present >>= BL;
#pragma unroll
            for (int b = 0; b < BL; b++) {
                queue[0][b] = queue[1][b];
                queue[1][b] = queue[2][b];
            }
            if ((t + AHEAD) * BL - from_block >= 64) {
                from_block += 64;
                look_up(far_ids);
                far_ids = pages_from(from_block + 64);
            }
        } while (t < steps && !far && !hides(t) && !__ballot(top > (BF ? m : m + lag)));
    }
    if (steps) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // (copies that nobody waited for do not outlive the workgroup's use of LDS)
#pragma unroll
        for (int i = 0; i < N; i++) y[i % G] = mfma32<KIND>(value_at(V0 + ring[R - 1], i / G, i % G), pf[i / G], y[i % G]);
    }
    l += other_quarter<32>(l);
    m = m == none ? none : m * c;
    const int64_t row_at = ((int64_t)(u.s.row0 + i) * a.c.kv_heads * a.group + head) * DIM + 4 * h;
    if (u.splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        if (real) {
#pragma unroll
            for (int d = 0; d < G; d++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    store_row4<KIND>(a.y, a.qdt, row_at + 32 * d + 8 * e, float4_t{y[d][4 * e] * inv, y[d][4 * e + 1] * inv, y[d][4 * e + 2] * inv, y[d][4 * e + 3] * inv});
        }
        return;
    }
    // a part: its sums, then maxima and sums of probabilities of its rows
    constexpr int SLAB = T::kSlab;
    float* const slab = a.slabs + (size_t)u.slab * SLAB;
    float* const stats = slab + ROWS * DIM + 2 * (wv * 32 + r);
#pragma unroll
    for (int d = 0; d < G; d++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            put_float4(slab + (((wv * G + d) * 4 + e) * 64 + lane) * 4, float4_t{y[d][4 * e], y[d][4 * e + 1], y[d][4 * e + 2], y[d][4 * e + 3]});
    if (h == 0) put_float2(stats, m, l);
    if (!last_part(a, u, reinterpret_cast<unsigned*>(lds))) return;
    const float* const of_tile = slab - (size_t)u.split * SLAB;
    auto part_of = [&](int e) { return get_float2(of_tile + (size_t)e * SLAB + ROWS * DIM + 2 * (wv * 32 + r)); };        // maximum and sum of my row
    top = none;
    float sum = 0.f;
    for (int e = 0; e < u.splits; e += 4) {
        f32x2_t of[4];
#pragma unroll
        for (int k = 0; k < 4; k++) of[k] = part_of(min(e + k, u.splits - 1));
#pragma unroll
        for (int k = 0; k < 4; k++) top = fmaxf(top, of[k][0]);
    }
#pragma unroll
    for (int d = 0; d < G; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) y[d][e] = 0.f;
    for (int e = 0; e < u.splits; e++) {
        const f32x2_t me = part_of(e);
        const float* const from = of_tile + (size_t)e * SLAB + (wv * G * 4 * 64 + lane) * 4;
        float4_t part[4 * G];                                        // asked for at once: past the caches a load takes a microsecond or two
#pragma unroll
        for (int k = 0; k < 4 * G; k++) part[k] = get_float4(from + k * 256);
        const float f = me[0] == none ? 0.f : exp2_fast(me[0] - top);
        sum += f * me[1];
#pragma unroll
        for (int k = 0; k < 4 * G; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) y[k / 4][4 * (k % 4) + j] += part[k][j] * f;
    }
    if (!real) return;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
    for (int d = 0; d < G; d++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            store_row4<KIND>(a.y, a.qdt, row_at + 32 * d + 8 * e, float4_t{y[d][4 * e] * inv, y[d][4 * e + 1] * inv, y[d][4 * e + 2] * inv, y[d][4 * e + 3] * inv});
}

template <int KIND, int G>
hipError_t rows_as(const AttnArgs& a, unsigned grid, hipStream_t st)
{
    (void)LdsRequest<&attention_rows_kernel<KIND, G>, RowsShape<G>::kLds>::registered;
    hipLaunchKernelGGL((attention_rows_kernel<KIND, G>), dim3(grid), dim3(64 * RowsShape<G>::kWaves), RowsShape<G>::kLds, st, a);
    return hipGetLastError();
}

template <int KIND, int G>
hipError_t tiles_as(const AttnArgs& a, unsigned grid, hipStream_t st)
{
    typedef TileShape<KIND, G> T;
    (void)LdsRequest<&attention_tiles_kernel<KIND, G>, T::kLds>::registered;
    hipLaunchKernelGGL((attention_tiles_kernel<KIND, G>), dim3(grid), dim3(64 * T::kWaves), T::kLds, st, a);
    return hipGetLastError();
}

template <int KIND, int G>
hipError_t attention_as(AttnArgs a, bool exact, hipStream_t st)
{
    // (max_new and rows bound a sequence's rows, no more: one token of a padded call, or of one that was captured for prompts, is the rows kernel's)
    const int64_t most = (int64_t)std::min(a.t.max_new, a.t.rows) * a.group;
    const int few = (int64_t)a.t.rows * a.group * a.c.kv_heads <= few_in_all(KIND) ? kFewAlone : kFewRows;
    const bool many = !exact && most > few;
    a.few = many ? few : 0;
    const int64_t rows = (int64_t)a.t.rows * a.group, blocks = (int64_t)a.t.table_pages << a.c.page_shift;
    // tiles of all, and the parts beyond one of each: what `target` makes of them, and no more than the table has blocks for
    auto grid = [&](int64_t tiles, int extra, int least) {
        return (unsigned)(tiles * a.c.kv_heads + std::min<int64_t>(extra, tiles * a.c.kv_heads * (blocks / least)));
    };
    // (a tile has a row, and a sequence of many rows more than `few`: a batch is mostly sequences without any, and each of a grid's workgroups looks
    // at all of them)
    const int64_t few_tiles = std::min({rows / kRows + a.t.seqs, many ? (int64_t)a.t.seqs * ((few + kRows - 1) / kRows) : rows, rows});
    const unsigned few_grid = grid(few_tiles, kMostExtra, kLeast);
    if (!many) return rows_as<KIND, G>(a, few_grid, st);
    a.target = TileShape<KIND, G>::kTarget;
    const int64_t many_tiles = rows / TileShape<KIND, G>::kRows + std::min<int64_t>(a.t.seqs, rows / (few + 1));
    const unsigned many_grid = grid(many_tiles, TileShape<KIND, G>::kMostExtra, kTileLeast);
    if (a.t.seqs == 1) return tiles_as<KIND, G>(a, std::max(few_grid, many_grid), st);
    const hipError_t e = rows_as<KIND, G>(a, few_grid, st);
    return e == hipSuccess ? tiles_as<KIND, G>(a, many_grid, st) : e;
}

}  // namespace

// A launch has fewer than 2^32 threads.  Rows kernel: 256 to a unit.  Tiles kernel, per kv head: rows / kRows tiles and one more for each sequence of more
// than kFewRows; rows of all heads are at most kRows kMaxUnits.
int64_t attention_max_units() { return kMaxUnits - 1; }
template <int KIND, int G>
constexpr bool kLaunches = ((int64_t)kRows * kMaxUnits / TileShape<KIND, G>::kRows + (int64_t)kRows * kMaxUnits / (kFewRows + 1) + TileShape<KIND, G>::kMostExtra) *
                               (64 * TileShape<KIND, G>::kWaves) < (int64_t)1 << 32;
static_assert(kLaunches<kCacheF16, 2> && kLaunches<kCacheF16, 4> && kLaunches<kCacheF16, 8> && kLaunches<kCacheQ8, 2> && kLaunches<kCacheQ8, 8>, "a grid's threads");
static_assert((int64_t)(kMaxUnits - 1) * 64 * RowsShape<2>::kWaves < (int64_t)1 << 32, "a grid's threads");

// Slabs: of parts of tiles that have more than one, at most twice those beyond one of each tile
size_t attention_scratch_bytes(int dim)
{
    const size_t rows = (size_t)2 * kMostExtra * kRows * (dim + 2);
    auto tiles = [](int extra, int slab) { return (size_t)2 * extra * slab; };
    size_t many;
    switch (dim) {                                                   // (the quantised kinds have as many, or half as many of twice the rows)
        case 64: many = tiles(TileShape<kCacheF16, 2>::kMostExtra, TileShape<kCacheF16, 2>::kSlab); break;
        case 96: many = tiles(TileShape<kCacheF16, 3>::kMostExtra, TileShape<kCacheF16, 3>::kSlab); break;
        case 128: many = tiles(TileShape<kCacheF16, 4>::kMostExtra, TileShape<kCacheF16, 4>::kSlab); break;
        default: many = tiles(TileShape<kCacheF16, 8>::kMostExtra, TileShape<kCacheF16, 8>::kSlab); break;
    }
    return std::max(rows, many) * sizeof(float);
}
template <int G>
constexpr bool kPartsFit = TileShape<kCacheQ8, G>::kMostExtra * TileShape<kCacheQ8, G>::kSlab <= TileShape<kCacheF16, G>::kMostExtra * TileShape<kCacheF16, G>::kSlab;
static_assert(kPartsFit<2> && kPartsFit<3> && kPartsFit<4> && kPartsFit<8>, "parts of all kinds fit the scratch");
static_assert(2 * std::max(kMostExtra, TileShape<kCacheF16, 2>::kMostExtra) * sizeof(unsigned) <= kAttnTicketBytes, "a ticket per tile");

int64_t attention_units_max(const BatchView& t, int kv_heads, int group)
{
    // tiles: (n * group + 15) / 16 of a sequence; parts: at most kMostExtra more than tiles
    return ((int64_t)t.rows * group / kRows + t.seqs) * kv_heads + std::max(kMostExtra, TileShape<kCacheF16, 2>::kMostExtra);
}

hipError_t launch_attention(const CacheView& c, const BatchView& t, const void* q, int64_t q_stride, int qdt, int group, float scale, int window, bool exact, void* y,
                            void* scratch, void* tickets, hipStream_t st)
{
    AttnArgs a;
    a.c = c;
    a.t = t;
    a.q = q;
    a.y = y;
    a.q_stride = q_stride;
    a.slabs = static_cast<float*>(scratch);
    a.tickets = static_cast<unsigned*>(tickets);
    a.group = group;
    a.qdt = qdt;
    a.window = window;
    a.scale = std::min(std::max(scale * 1.44269504088896340736f, kLeastFactor), kMostFactor);
#define CYBQ_ROWS(KIND)                                   \
    switch (c.dim) {                                      \
        case 64: return attention_as<KIND, 2>(a, exact, st); \
        case 96: return attention_as<KIND, 3>(a, exact, st); \
        case 128: return attention_as<KIND, 4>(a, exact, st);    \
        default: return attention_as<KIND, 8>(a, exact, st); \
    }
    switch (c.kind) {
        case kCacheF16: CYBQ_ROWS(kCacheF16)
        case kCacheBF16: CYBQ_ROWS(kCacheBF16)
        case kCacheQ4: CYBQ_ROWS(kCacheQ4)
        default: CYBQ_ROWS(kCacheQ8)
    }
#undef CYBQ_ROWS
}

}  // namespace cybq
