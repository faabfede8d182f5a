// experts.hip - products of rows with the block-quantised weights of the experts they were sent to.
//
// A stack of E experts is one weight of E * n rows (n a multiple of 16: expert e is the strips [e * n / 16, (e + 1) * n / 16)).
// A pair p = t * top_k + j is token t with its j-th expert ids[p]; an id outside 0 .. E - 1 is no expert.
//
//   out[p, :] = x[p / xdiv, :] W_ids[p]^T         xdiv = top_k: the tokens' rows; 1: a row of its own for every pair
//
// The kernels, by the number of rows that an expert has:
//   few   experts_few_kernel    one pass over each met expert's weights, HBM-bound; pieces of 1, 8, 16, 32 or 64 rows
//   many  experts_many_kernel   tiles of 64 or 128 rows, bound by what a CU's vector, matrix and memory pipes do between two barriers
//   back  experts_token_kernel  a few tokens, all their experts as one long K, no sums in memory; else few / many into fp32 sums [P, n] in the
//                               scratch and experts_sum_kernel
// Operands are exact - the integers q (bf16 and fp32 rows: biased, and a second product that takes the bias off), each group's sums times its
// scale in fp32, so scales that leave f16's range when multiplied with q do no harm - but for many rows and a y of bf16 in FAST mode, where they
// are round_f16(scale * q): 2e-4 relative L2 next to the 1.6e-3 of y's own rounding, and no FMAs behind the MFMAs.
//
// us per call, weights from HBM: 680 MB of others' and more are read in between (bytes: weights of the experts that the timed ids meet, rows and
// outputs; products without the bias'):
//   up, 8 of 128 experts of 2048 -> 2 x 768, Q4, one f16 token 7.2 (14 MB; 5.1 - 5.8 where the 256 MB cache has them); back 6.9 (7 MB; 6.4)
//                                                                                     the launch, three trips to memory, the stream
//   up, 2 of 8 of 4096 -> 2 x 14336, 16 bf16 tokens 97 (7.75 met: 513 MB, 5.3 TB/s); back, 32 f16 tokens 58 (267 MB, 4.6 TB/s; 46 - 57 with
//                                                                                     a part of them cached)                      HBM
//   up, 4 of 60 of 2592 -> 2 x 1040, Q8, 37 f16 tokens 69 (51 met: 293 MB, 4.2 TB/s; 55 - 69 partly cached)                        HBM
//   up, 8 of 128, 2048 bf16 tokens 155 - 173 (103 GFLOP: 0.60 - 0.67 PFLOP/s); back 156 - 167; 2 of 8 wide ones, 1024 tokens 508 - 541 (481 GFLOP:
//   0.89 - 0.95), each over runs on several machines
#include <algorithm>
#include <type_traits>

#include "gemv_parts.h"

namespace cybq {

namespace {

#include "gemm_parts.h"

// ---- which rows does an expert have: the lists ------------------------------------------------------------------
//
// int32 words: [0, E]: where expert e's pairs start in the order below, [E + 1]: number of row tiles, then (4-word aligned) the tiles
// {expert, first pair, pairs, number of the expert's tile << 16 | of tiles it has}, then the pairs in order of expert and, within one, of their number.

constexpr int kRowTile = 64;                                     // rows of a full tile, at least
__host__ __device__ inline int64_t lists_tiles_max(int64_t P, int E) { return P / kRowTile + (P < E ? P : E); }
__host__ __device__ inline int64_t lists_tiles_at(int E) { return (E + 2 + 3) / 4 * 4; }
__host__ __device__ inline int64_t lists_order_at(int64_t P, int E) { return lists_tiles_at(E) + 4 * lists_tiles_max(P, E); }

// sums of v over the threads ahead of this one, of all threads in `total`; two sums at a time.  wave_sums: [16]
__device__ __forceinline__ int2 block_exclusive_scan(int2 v, int2* wave_sums, int2* total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int2 s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int2 o = make_int2(__shfl_up(s.x, d), __shfl_up(s.y, d));
        if (lane >= d) s = make_int2(s.x + o.x, s.y + o.y);
    }
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    int2 before = {0, 0}, all = {0, 0};
    for (int i = 0; i < waves; i++) {
        const int2 w = wave_sums[i];
        if (i < wave) before = make_int2(before.x + w.x, before.y + w.y);
        all = make_int2(all.x + w.x, all.y + w.y);
    }
    *total = all;
    return make_int2(before.x + s.x - v.x, before.y + s.y - v.y);
}

// Every workgroup counts all pairs (per expert: all of them, and those ahead of its own share), scans the counts, and places its share:
// a histogram per wave, whose lanes with the same expert find each other by one ballot per bit of the id, so the order does not hang on
// atomics.  `block` of `blocks`, 1024 threads.  Launch and all, 16384 pairs 8.6 us, 2048 6.6 (with the ids asked for pass by pass and two
// scans 9.6 and 7.1; one workgroup alone placed 16384 in 12).
__device__ __forceinline__ void make_lists(const int32_t* __restrict__ ids, int P, int E, int bits, int row_tile, int block, int blocks, int32_t* __restrict__ out,
                                           int* lds)
{
    int *const total = lds, *const before = lds + E, *const hist = lds + 2 * E;      // hist: [16][E]
    int2* const wave_sums = reinterpret_cast<int2*>(lds + 18 * E);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int share = (P + blocks * 1024 - 1) / (blocks * 1024) * 64;         // pairs per wave, whole rounds of 64
    const int first = min(block * 16 * share, P), lo = min(first + wave * share, P), hi = min(lo + share, P);
    int* const my = hist + wave * E;
    int32_t id[16], own[16];
    auto request = [&](int32_t (&id)[16], int p0, int end, int step) {        // sixteen ids at a time: one trip to memory, not sixteen
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int p = p0 + i * step;
            id[i] = p < end ? ids[p] : -1;
        }
    };
    // the first of both passes on their way while LDS is cleared
    request(id, tid, P, 1024);
    request(own, lo + lane, hi, 64);
    for (int i = tid; i < 18 * E; i += 1024) lds[i] = 0;
    __syncthreads();
    for (int p0 = tid; p0 < P; p0 += 16384) {
        if (p0 >= 16384) request(id, p0, P, 1024);
#pragma unroll
        for (int i = 0; i < 16; i++)
            if ((unsigned)id[i] < (unsigned)E) {
                atomicAdd(&total[id[i]], 1);
                if (p0 + i * 1024 < first) atomicAdd(&before[id[i]], 1);
            }
    }
    for (int p0 = lo; p0 < hi; p0 += 1024) {
        if (p0 > lo) request(own, p0 + lane, hi, 64);
#pragma unroll
        for (int i = 0; i < 16; i++)
            if ((unsigned)own[i] < (unsigned)E) atomicAdd(&my[own[i]], 1);
    }
    __syncthreads();
    const int count = tid < E ? total[tid] : 0;
    const int n_tiles = (count + row_tile - 1) / row_tile;
    int2 all;
    const int2 ahead = block_exclusive_scan(make_int2(count, n_tiles), wave_sums, &all);
    const int start = ahead.x, tile0 = ahead.y;
    if (tid < E) {
        int at = start + before[tid], h[16];
#pragma unroll
        for (int w = 0; w < 16; w++) h[w] = hist[w * E + tid];
#pragma unroll
        for (int w = 0; w < 16; w++) {
            hist[w * E + tid] = at;
            at += h[w];
        }
        if (block == 0) {
            out[tid] = start;
            int4* const tiles = reinterpret_cast<int4*>(out + lists_tiles_at(E));
            // an expert's rows in tiles of like size, whole blocks of 16 rows
            const int rows = n_tiles ? ((count + n_tiles - 1) / n_tiles + 15) / 16 * 16 : 0;
            for (int i = 0; i < n_tiles; i++) tiles[tile0 + i] = make_int4(tid, start + i * rows, max(0, min(rows, count - i * rows)), i << 16 | n_tiles);
        }
    }
    if (block == 0 && tid == 0) {
        out[E] = all.x;
        out[E + 1] = all.y;
    }
    __syncthreads();
    int32_t* const order = out + lists_order_at(P, E);
    for (int p0 = lo; p0 < hi; p0 += 1024) {
        if (share > 1024) request(own, p0 + lane, hi, 64);       // (else they are still there)
        for (int i = 0; i < 16 && p0 + i * 64 < hi; i++) {
            const int e = own[0];
#pragma unroll
            for (int k = 0; k < 15; k++) own[k] = own[k + 1];
            const bool there = (unsigned)e < (unsigned)E;
            uint64_t same = __ballot(there);
            for (int b = 0; b < bits; b++) {
                const uint64_t set = __ballot((e >> b) & 1);
                same &= (e >> b) & 1 ? set : ~set;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1));
            int at = 0;
            if (there) at = my[e] + rank;
            __builtin_amdgcn_wave_barrier();
            if (there && rank == 0) my[e] = at + __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (there) order[at] = p0 + i * 64 + lane;
        }
    }
}

// bf16 rows -> f16 rows times a power of two each that brings the largest magnitude to 2^13 .. 2^14: exact but for elements below 2^-27 of it.
// One wave per row; rows without an expert (ids: of pairs, a row each) are left out.
__device__ __forceinline__ void stage_row(const uint16_t* __restrict__ x, const int32_t* __restrict__ ids, int E, int64_t rows, int K, int64_t row,
                                          uint16_t* __restrict__ out, float* __restrict__ unscale)
{
    const int lane = threadIdx.x & 63;
    if (row >= rows || (ids && (unsigned)ids[row] >= (unsigned)E)) return;
    const u32x4_t* const from = reinterpret_cast<const u32x4_t*>(x + row * K);
    u32x4_t* const to = reinterpret_cast<u32x4_t*>(out + row * K);
    const int n = K / 8;
    constexpr int HELD = 8;                                      // pieces of a lane that stay in registers (K up to 4096)
    u32x4_t held[HELD];
    uint32_t top = 0;                                            // bits of the largest magnitude (as integers they are in its order)
    auto magnitude = [&](const u32x4_t& v) {
#pragma unroll
        for (int k = 0; k < 4; k++) top = max(top, max((v[k] << 16) & 0x7fff0000u, v[k] & 0x7fff0000u));
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) held[i] = i * 64 + lane < n ? from[i * 64 + lane] : (u32x4_t){0u, 0u, 0u, 0u};
    for (int i = HELD * 64 + lane; i < n; i += 64) magnitude(from[i]);
#pragma unroll
    for (int i = 0; i < HELD; i++) magnitude(held[i]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    const int exponent = (int)(top >> 23) - 127;
    const int shift = top == 0 || exponent == 128 ? 0 : min(13 - exponent, 126);
    const float f = __builtin_bit_cast(float, (uint32_t)(127 + shift) << 23);
    auto scaled = [&](const u32x4_t& v) {
        u32x4_t o;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const half2_t h = {(_Float16)(__builtin_bit_cast(float, v[k] << 16) * f), (_Float16)(__builtin_bit_cast(float, v[k] & 0xffff0000u) * f)};
            o[k] = as_u32(h);
        }
        return o;
    };
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (i * 64 + lane < n) to[i * 64 + lane] = scaled(held[i]);
    for (int i = HELD * 64 + lane; i < n; i += 64) to[i] = scaled(from[i]);
    if (lane == 0) unscale[row] = __builtin_bit_cast(float, (uint32_t)(127 - shift) << 23);
}

// What the kernel for many rows needs beforehand, in one launch: the first list_blocks workgroups make the lists, the rest stage rows, a wave each.
__global__ __launch_bounds__(1024) void experts_prepare_kernel(const int32_t* __restrict__ ids, int P, int E, int bits, int row_tile, int list_blocks,
                                                               int32_t* __restrict__ lists, const uint16_t* __restrict__ x, int xdiv, int K,
                                                               uint16_t* __restrict__ staged, float* __restrict__ unscale)
{
    extern __shared__ int lists_lds[];                           // 18 * E, then 16 pairs of wave sums
    if ((int)blockIdx.x < list_blocks) make_lists(ids, P, E, bits, row_tile, blockIdx.x, list_blocks, lists, lists_lds);
    else stage_row(x, xdiv == 1 ? ids : nullptr, E, P / xdiv, K, (int64_t)((int)blockIdx.x - list_blocks) * 16 + (threadIdx.x >> 6), staged, unscale);
}

// ---- the multiply -------------------------------------------------------------------------------------------------
//
// Workgroup = 8 waves, COLS of them side by side, KH = 8 / COLS behind each other along K; a wave has two strips of one expert (a gate and its
// up strip) against up to 16 * RB of the expert's rows.  A step is KH K tiles: the rows of each are gathered into LDS once, whole 128-byte
// lines per eight lanes, pieces permuted so that the reads meet no bank conflicts; a wave's own weight tiles pass through LDS as well, only to
// be on their way without registers (global_load_lds).  D steps have a place in LDS, copies are counted by hand: they retire in order.
// (Weights and rows straight into registers, as operands: rows cost 64 separate accesses per load; 16 tokens on the wide experts 208 us
// against 101, 37 on 60 Q8 experts 124 against 46.)
struct ExpertsArgs {
    const uint8_t* w;
    const void* x;
    const int32_t* ids;
    const int32_t* lists;       // lists, or nullptr: an expert's pairs are found among the (at most kMaxDirect) ids
    int64_t P;
    int xdiv, K, KT, strips, E;
    int groups;                 // workgroups that share out an expert's strips
    int single;                 // one token: a pair has its expert to itself
    int by_pair;                // blockIdx.y is a pair (the first of its expert does the work), else an expert
    void* y;
    int ydt, n_out;
    const float* unscale;       // what the sums of a row of x are multiplied with (staged rows), or nullptr
};

constexpr int kMaxDirect = 512;
constexpr int kFewLds = 78 * 1024;                               // two workgroups to a CU

__device__ __forceinline__ void copy_lanes_to_lds(uint32_t lds_off, const void* base, uint32_t off, uint64_t lanes)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_mov_b64 exec, %3\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1" ::"s"(__builtin_amdgcn_readfirstlane(lds_off)), "v"(off), "s"(base), "s"(lanes));
}

// XB: blocks of eight rows
template <int BITS, int XM, int XB, int COLS, int BUDGET>
struct Shape {
    static constexpr int RB = (XB + 1) / 2, KH = 8 / COLS;
    static constexpr int PARTS = XM == XF32 ? 4 : 2;             // 128-byte lines of a row in a K tile
    static constexpr int BLOCKS = XB * PARTS;                    // 1-KB blocks of rows
    static constexpr int XTILE = BLOCKS * 1024;
    static constexpr int WQ = 1024 * (BITS / 4);
    static constexpr int WTILE = 2 * WQ + 256;                   // a wave's two strips
    static constexpr int STEP = KH * XTILE + 8 * WTILE;
    static constexpr int FIT = BUDGET / STEP;
    static constexpr int D = FIT > 6 ? 6 : FIT < 2 ? 2 : FIT;
    static constexpr int XC = (BLOCKS + COLS - 1) / COLS;        // copies per wave and step
    static constexpr int WC = 2 * (BITS / 4) + 1;
    static constexpr int LDS = D * STEP;
};

// eight fp32 values -> three bf16 operands that add up to them (24 significant bits: exact), the largest first.  Their bias products begin with
// the smallest, their products with the weights with the largest: one sum of each is as large as the bias makes it, not three
__device__ __forceinline__ void split_f32(const u32x4_t& lo, const u32x4_t& hi, Frag16 (&out)[3])
{
#pragma unroll
    for (int p = 0; p < 4; p++) {
        float v[2] = {__builtin_bit_cast(float, p < 2 ? lo[2 * p] : hi[2 * p - 4]), __builtin_bit_cast(float, p < 2 ? lo[2 * p + 1] : hi[2 * p - 3])};
#pragma unroll
        for (int part = 0; part < 3; part++) {
            uint32_t h[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                h[e] = __builtin_bit_cast(uint32_t, v[e]) & 0xffff0000u;              // cut: the rest keeps its sign and fits what follows
                v[e] = (h[e] & 0x7f800000u) == 0x7f800000u ? 0.f : v[e] - __builtin_bit_cast(float, h[e]);
            }
            out[part].u[p] = (h[0] >> 16) | h[1];
        }
    }
}

// bf16 operands: Q4 the numbers 16 + u (u = q + 8 in the upper four bits of the mantissa), Q8 the numbers u = q + 128; a product of the rows
// with the constant -24 (-128) takes the bias off in the same accumulation.  (128 + u, a bias of 136, costs an instruction less per eight
// weights and two more bits of the sums: 2.8e-6 relative L2 against float64 where this has 5e-7.)
constexpr uint32_t kNeg24x2 = 0xC1C0C1C0u;
__device__ __forceinline__ uint32_t magic16_vgpr()
{
    uint32_t mv;
    asm volatile("v_mov_b32 %0, 0x41804180" : "=v"(mv));
    return mv;
}
// slots 2k, 2k + 1 of group 2p + t from word pair p
__device__ __forceinline__ uint32_t q4_bf16_word(uint32_t wa, uint32_t wb, int t, int k, uint32_t magic)
{
    const uint32_t w = k >> 1 ? wb : wa;
    const uint32_t v = t ? (k & 1 ? w >> 9 : w >> 1) : (k & 1 ? w >> 5 : w << 3);
    return (v & 0x00780078u) | magic;
}

template <int BITS, int OPM>
__device__ __forceinline__ void expert_operands(const TileRegs<BITS>& t, uint32_t magic, Frag16 (&b)[4])
{
    if constexpr (BITS == 4 && OPM == XBF16) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int k = 0; k < 4; k++) b[j].u[k] = q4_bf16_word(t.q[0][2 * (j >> 1)], t.q[0][2 * (j >> 1) + 1], j & 1, k, magic);
    } else {
        tile_operands<BITS, OPM>(t, magic, b);
    }
}

// Strips strip0 + 2 col, + 1 of expert e against the pairs list[0 .. n), n <= 8 * XB.
template <int BITS, int XM, bool PAIR, int XB, int COLS, int BUDGET>
__device__ __forceinline__ void expert_tile(const ExpertsArgs& g, int e, const int32_t* list, int n, int strip0, uint8_t* smem)
{
    using S = Shape<BITS, XM, XB, COLS, BUDGET>;
    constexpr int D = S::D, RB = S::RB, KH = S::KH, OPM = XM == XF16 ? XF16 : XBF16;
    constexpr int GB = XM == XF32 ? 128 : 64;                    // bytes of a group of a row
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = wave % COLS, kh = wave / COLS;
    const int i16 = lane & 15, oct = lane >> 4;
    const int G = g.K / kGroup;
    const int steps = (g.KT + KH - 1) / KH;

    const int strip = min(strip0 + col * 2, g.strips - 2 + (g.strips & 1)), second = min(strip + 1, g.strips - 1);
    const uint8_t* const wsrc = g.w + ((int64_t)e * g.strips + strip) * g.KT * kTileBytes<BITS>;
    const uint32_t wstep = (uint32_t)(second - strip) * (uint32_t)(g.KT * kTileBytes<BITS>);
    const uint32_t sc_off = (lane >= 8 ? wstep : 0u) + (uint32_t)(kTileQBytes<BITS> + (lane & 7) * 16);
    auto copy_w = [&](int step, int buf) {
        const uint32_t src = (uint32_t)min(step * KH + kh, g.KT - 1) * (uint32_t)kTileBytes<BITS>;
        const uint32_t at = (uint32_t)(buf * S::STEP + KH * S::XTILE + wave * S::WTILE);
#pragma unroll
        for (int q = 0; q < BITS / 4; q++) {
            copy_to_lds(at + q * 1024, wsrc, src + q * 1024u + (uint32_t)lane * 16u);
            copy_to_lds(at + S::WQ + q * 1024, wsrc, wstep + src + q * 1024u + (uint32_t)lane * 16u);
        }
        copy_lanes_to_lds(at + 2 * S::WQ, wsrc, sc_off + src, 0xffffull);
    };
#pragma unroll
    for (int d = 0; d < D - 1; d++) copy_w(d, d);

    // block b = rows 8 * (b / PARTS) .. + 8, line b % PARTS of the K tile; copy c of a wave is block c * COLS + col of its kh's tile
    const int crow = lane >> 3, piece = (lane & 7) ^ crow;
    uint32_t xoff[S::XC];
    int xblk[S::XC];
    uint64_t xlanes[S::XC];
#pragma unroll
    for (int c = 0; c < S::XC; c++) {
        xblk[c] = min(c * COLS + col, S::BLOCKS - 1);
        const int row0 = xblk[c] / S::PARTS * 8;
        xoff[c] = (uint32_t)(list[min(row0 + crow, n - 1)] / g.xdiv) * (uint32_t)(g.K * (GB / 32));
        xlanes[c] = XB > 4 || n >= row0 + 8 ? ~0ull : (1ull << (8 * max(n - row0, 1))) - 1;
    }
    auto copy_x = [&](int step, int buf) {
        const int kt = min(step * KH + kh, g.KT - 1);
#pragma unroll
        for (int c = 0; c < S::XC; c++) {
            // (groups past the end of a row: its last one; they are not multiplied)
            const int part = xblk[c] % S::PARTS;
            const int grp = min(XM == XF32 ? kt * 4 + part : kt * 4 + part * 2 + (piece >> 2), G - 1);
            const uint32_t from = xoff[c] + (uint32_t)grp * GB + (uint32_t)(XM == XF32 ? piece : piece & 3) * 16u;
            const uint32_t to = (uint32_t)(buf * S::STEP + kh * S::XTILE + xblk[c] * 1024);
            if constexpr (XB > 4) copy_to_lds(to, g.x, from);
            else copy_lanes_to_lds(to, g.x, from, xlanes[c]);
        }
    };
#pragma unroll
    for (int d = 0; d < D - 1; d++) copy_x(d, d);

    float4_t acc[RB][2];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int s = 0; s < 2; s++) acc[i][s] = (float4_t){0.f, 0.f, 0.f, 0.f};
    const uint32_t magic = OPM == XF16 ? q4_magic_vgpr() : magic16_vgpr();
    const int hr = XB == 1 ? 0 : i16 >> 3;                       // (XB = 1: rows 8 .. 15 of the operand are rows 0 .. 7 again)
    const uint32_t raw = (uint32_t)(hr * (S::PARTS * 1024) + (i16 & 7) * 128 + (((XM == XF32 ? 2 * oct : oct) ^ (i16 & 7)) * 16));
    Frag16 off;
    const uint32_t offw = BITS == 4 ? kNeg24x2 : kBf16Neg128x2;
    off.u = (u32x4_t){offw, offw, offw, offw};

    auto multiply = [&](const uint8_t* at, int groups) {
        const uint8_t* const wp = at + KH * S::XTILE + wave * S::WTILE;
        const uint8_t* const xp = at + kh * S::XTILE;
        TileRegs<BITS> w[2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int q = 0; q < BITS / 4; q++) w[s].q[q] = *reinterpret_cast<const u32x4_t*>(wp + s * S::WQ + q * 1024 + lane * 16);
            w[s].s = *reinterpret_cast<const u32x2_t*>(wp + 2 * S::WQ + s * 128 + i16 * 8);
        }
        Frag16 b[2][4];
        expert_operands<BITS, OPM>(w[0], magic, b[0]);
        expert_operands<BITS, OPM>(w[1], magic, b[1]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j >= groups) break;
            float sc[2];
#pragma unroll
            for (int s = 0; s < 2; s++) {
                sc[s] = f16_bits_to_f32((j & 1) ? w[s].s[j >> 1] >> 16 : w[s].s[j >> 1] & 0xffffu);
            }
#pragma unroll
            for (int i = 0; i < RB; i++) {
                constexpr int NA = XM == XF32 ? 3 : 1;
                Frag16 a[3];
                if constexpr (XM == XF32) {
                    const uint8_t* const p = xp + i * (2 * S::PARTS * 1024) + j * 1024;
                    split_f32(*reinterpret_cast<const u32x4_t*>(p + raw), *reinterpret_cast<const u32x4_t*>(p + (raw ^ 16u)), a);
                } else {
                    a[0].u = *reinterpret_cast<const u32x4_t*>(xp + i * (2 * S::PARTS * 1024) + (j >> 1) * 1024 + ((j & 1) ? raw ^ 64u : raw));
                }
                float4_t c = {0.f, 0.f, 0.f, 0.f};
                if constexpr (OPM == XBF16) {
#pragma unroll
                    for (int k = NA - 1; k >= 0; k--) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[k].b, off.b, c, 0, 0, 0);
                }
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    float4_t d = c;
                    if constexpr (OPM == XBF16) {
#pragma unroll
                        for (int k = 0; k < NA; k++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[k].b, b[s][j].b, d, 0, 0, 0);
                    } else {
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0].h, b[s][j].h, d, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][s][r] = fmaf(sc[s], d[r], acc[i][s][r]);
                }
            }
        }
    };
    int buf = 0;
    auto enter = [&](int step) {
        // this step's copies are there - mine, and behind the barrier everybody's - and nobody reads the last one's place any more.  (The
        // rows of the first D - 1 steps were asked for behind all their weights.)
        if (step < D - 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((D - 2) * S::XC) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((D - 2) * (S::XC + S::WC)) : "memory");
        if constexpr (COLS > 1) asm volatile("s_barrier" ::: "memory");
        const int free = buf == 0 ? D - 1 : buf - 1;
        copy_x(step + D - 1, free);
        copy_w(step + D - 1, free);
    };
    // (steps of whole K tiles by themselves: a body that may end early costs a move of every sum per step)
    int step = 0;
    for (const int whole = G / 4 / KH; step < whole; step++) {
        enter(step);
        multiply(smem + buf * S::STEP, 4);
        buf = buf + 1 == D ? 0 : buf + 1;
    }
    for (; step < steps; step++) {
        enter(step);
        const int left = G - (step * KH + kh) * 4;
        if (left > 0) multiply(smem + buf * S::STEP, min(left, 4));
        buf = buf + 1 == D ? 0 : buf + 1;
    }
    // (no copy may land in LDS that holds something else by then)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    if constexpr (KH > 1) {
        // the sums of the waves along K meet in their order
        float4_t* const red = reinterpret_cast<float4_t*>(smem);
        __syncthreads();
        if (kh)
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int s = 0; s < 2; s++) red[((kh * COLS + col) * RB * 2 + i * 2 + s) * 64 + lane] = acc[i][s];
        __syncthreads();
        if (kh) return;
#pragma unroll
        for (int k = 1; k < KH; k++)
#pragma unroll
            for (int i = 0; i < RB; i++)
#pragma unroll
                for (int s = 0; s < 2; s++) acc[i][s] += red[((k * COLS + col) * RB * 2 + i * 2 + s) * 64 + lane];
    }
    const bool there = strip0 + col * 2 < g.strips, both = strip0 + col * 2 + 1 < g.strips;
    if (!there) return;
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int m = i * 16 + oct * 4 + r;
            if (m >= n) continue;
            const int64_t at = (int64_t)list[m] * g.n_out;
            if constexpr (PAIR) {
                store_out(g.y, g.ydt, at + (strip0 / 2 + col) * 16 + i16, silu_mul(acc[i][0][r], acc[i][1][r]));
            } else {
                store_out(g.y, g.ydt, at + (strip0 + col * 2) * 16 + i16, acc[i][0][r]);
                if (both) store_out(g.y, g.ydt, at + (strip0 + col * 2 + 1) * 16 + i16, acc[i][1][r]);
            }
        }
}

// ---- one row ------------------------------------------------------------------------------------------------------
//
// A wave by itself: two weight tiles per step (of a gate and its up strip, or of one strip) against one row each, all 16 rows of an operand
// the same one: every lane group of 16 has a tile's sums in its first register, so a group's scale is one fma, not four.  No barriers; D steps
// have a place in the wave's part of LDS, counted as above.  `at(step, slot)` names a tile.
struct RowTile {
    const uint8_t* w;           // the tile
    const char* x;              // its 128 elements of the row
    int groups;                 // of them that are there (0: the tile counts for nothing, but both addresses can be read)
    float factor;               // on the sums
};

template <int BITS, int XM, bool SHARED>
struct RowShape {
    static constexpr int XT = XM == XF32 ? 512 : 256;
    static constexpr int WQ = 1024 * (BITS / 4);
    static constexpr int XAT = 2 * WQ + 256;
    static constexpr int STEP = XAT + XT * (SHARED ? 1 : 2);
    static constexpr int FIT = kFewLds / (8 * STEP);
    static constexpr int D = FIT > 4 ? 4 : FIT < 2 ? 2 : FIT;
    static constexpr int COPIES = 2 * (BITS / 4) + (SHARED ? 2 : 3);
    static constexpr int LDS = 8 * D * STEP;
};

// SHARED: both tiles meet the same piece of the row
template <int BITS, int XM, bool SHARED, class At>
__device__ __forceinline__ void stream_row(int steps, At at, float (&acc)[2], uint8_t* smem)
{
    using S = RowShape<BITS, XM, SHARED>;
    constexpr int D = S::D, OPM = XM == XF16 ? XF16 : XBF16, NA = XM == XF32 ? 3 : 1;
    constexpr int XL = S::XT / 16;                               // lanes that copy 128 elements
    const int lane = threadIdx.x & 63, i16 = lane & 15, oct = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t mine = (uint32_t)(wave * D * S::STEP);
    auto copy = [&](int step, int buf) {
        const uint32_t to = mine + buf * S::STEP;
        const RowTile t0 = at(min(step, steps - 1), 0), t1 = at(min(step, steps - 1), 1);
#pragma unroll
        for (int q = 0; q < BITS / 4; q++) {
            copy_to_lds(to + q * 1024, t0.w, q * 1024u + (uint32_t)lane * 16u);
            copy_to_lds(to + S::WQ + q * 1024, t1.w, q * 1024u + (uint32_t)lane * 16u);
        }
        const uint32_t scales = (uint32_t)(kTileQBytes<BITS> + (lane & 7) * 16);
        if constexpr (SHARED) {                                  // (strips of one expert: less than 4 GiB apart)
            copy_lanes_to_lds(to + 2 * S::WQ, t0.w, (lane >= 8 ? (uint32_t)(t1.w - t0.w) : 0u) + scales, 0xffffull);
        } else {
            copy_lanes_to_lds(to + 2 * S::WQ, t0.w, scales, 0xffull);
            copy_lanes_to_lds(to + 2 * S::WQ + 128, t1.w, scales, 0xffull);
        }
        // (past the end of a row: its last piece; those groups are not multiplied)
        const uint32_t piece = (uint32_t)(lane % XL), last0 = (uint32_t)(max(t0.groups, 1) * XL / 4 - 1);
        if constexpr (SHARED) {
            copy_lanes_to_lds(to + S::XAT, t0.x, min(piece, last0) * 16u, (1ull << XL) - 1);
        } else {
            const uint32_t last1 = (uint32_t)(max(t1.groups, 1) * XL / 4 - 1), there = (uint32_t)(t1.x - t0.x);
            copy_lanes_to_lds(to + S::XAT, t0.x, lane < XL ? min(piece, last0) * 16u : there + min(piece, last1) * 16u, XL == 32 ? ~0ull : 0xffffffffull);
        }
    };
    for (int d = 0; d < D - 1; d++) copy(d, d);
    const uint32_t magic = OPM == XF16 ? q4_magic_vgpr() : magic16_vgpr();
    Frag16 off;
    const uint32_t offw = BITS == 4 ? kNeg24x2 : kBf16Neg128x2;
    off.u = (u32x4_t){offw, offw, offw, offw};
    acc[0] = acc[1] = 0.f;
    int buf = 0;
    for (int step = 0; step < steps; step++) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((D - 2) * S::COPIES) : "memory");
        copy(step + D - 1, buf == 0 ? D - 1 : buf - 1);
        const uint8_t* const from = smem + mine + buf * S::STEP;
        Frag16 a[4][NA];
        float4_t c[4];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const RowTile t = at(step, s);
            TileRegs<BITS> w;
#pragma unroll
            for (int q = 0; q < BITS / 4; q++) w.q[q] = *reinterpret_cast<const u32x4_t*>(from + s * S::WQ + q * 1024 + lane * 16);
            w.s = *reinterpret_cast<const u32x2_t*>(from + 2 * S::WQ + s * 128 + i16 * 8);
            Frag16 b[4];
            expert_operands<BITS, OPM>(w, magic, b);
            if (!SHARED || s == 0) {
                const uint8_t* const xp = from + S::XAT + (SHARED ? 0 : s * S::XT);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (XM == XF32) {
                        const u32x4_t* const p = reinterpret_cast<const u32x4_t*>(xp + j * 128 + oct * 32);
                        Frag16 three[3];
                        split_f32(p[0], p[1], three);
#pragma unroll
                        for (int k = 0; k < 3; k++) a[j][k] = three[k];
                    } else {
                        a[j][0].u = *reinterpret_cast<const u32x4_t*>(xp + j * 64 + oct * 16);
                    }
                    c[j] = (float4_t){0.f, 0.f, 0.f, 0.f};
                    if constexpr (OPM == XBF16) {
#pragma unroll
                        for (int k = NA - 1; k >= 0; k--) c[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][k].b, off.b, c[j], 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j >= t.groups) break;
                float4_t d = c[j];
                if constexpr (OPM == XBF16) {
#pragma unroll
                    for (int k = 0; k < NA; k++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][k].b, b[j].b, d, 0, 0, 0);
                } else {
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j][0].h, b[j].h, d, 0, 0, 0);
                }
                acc[s] = fmaf(f16_bits_to_f32((j & 1) ? w.s[j >> 1] >> 16 : w.s[j >> 1] & 0xffffu) * t.factor, d[0], acc[s]);
            }
        }
        buf = buf + 1 == D ? 0 : buf + 1;
    }
    // (no copy may land in LDS that holds something else by then)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}

// Strips strip0 + 2 col, + 1 of expert e against pair p.
template <int BITS, int XM, bool PAIR, int COLS>
__device__ __forceinline__ void expert_row(const ExpertsArgs& g, int e, int p, int strip0, uint8_t* smem)
{
    constexpr int KH = 8 / COLS, XS = XM == XF32 ? 4 : 2;
    const int lane = threadIdx.x & 63, i16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = wave % COLS, kh = wave / COLS, G = g.K / kGroup;
    const int strip = min(strip0 + col * 2, g.strips - 2 + (g.strips & 1)), second = min(strip + 1, g.strips - 1);
    const uint8_t* const wsrc = g.w + ((int64_t)e * g.strips + strip) * g.KT * kTileBytes<BITS>;
    const uint32_t wstep = (uint32_t)(second - strip) * (uint32_t)(g.KT * kTileBytes<BITS>);
    const char* const row = static_cast<const char*>(g.x) + (int64_t)(p / g.xdiv) * g.K * XS;
    float acc[2];
    stream_row<BITS, XM, true>((g.KT + KH - 1) / KH, [&](int step, int s) {
        const int kt = step * KH + kh, there = min(kt, g.KT - 1);
        return RowTile{wsrc + (s ? wstep : 0u) + (int64_t)there * kTileBytes<BITS>, row + (int64_t)there * (kTileK * XS), max(min(G - kt * 4, 4), 0), 1.0f};
    }, acc, smem);
    if constexpr (KH > 1) {
        float* const red = reinterpret_cast<float*>(smem);
        __syncthreads();
        if (kh && lane < 16) {
            red[(kh * COLS + col) * 32 + i16] = acc[0];
            red[(kh * COLS + col) * 32 + 16 + i16] = acc[1];
        }
        __syncthreads();
        if (kh) return;
#pragma unroll
        for (int k = 1; k < KH; k++) {
            acc[0] += red[(k * COLS + col) * 32 + i16];
            acc[1] += red[(k * COLS + col) * 32 + 16 + i16];
        }
    }
    if (lane >= 16 || strip0 + col * 2 >= g.strips) return;
    const int64_t at = (int64_t)p * g.n_out;
    if constexpr (PAIR) {
        store_out(g.y, g.ydt, at + (strip0 / 2 + col) * 16 + i16, silu_mul(acc[0], acc[1]));
    } else {
        store_out(g.y, g.ydt, at + (strip0 + col * 2) * 16 + i16, acc[0]);
        if (strip0 + col * 2 + 1 < g.strips) store_out(g.y, g.ydt, at + (strip0 + col * 2 + 1) * 16 + i16, acc[1]);
    }
}

// ---- many rows per expert -----------------------------------------------------------------------------------------
//
// The lists' row tiles.  Workgroup = a tile of up to 16 * RB rows x 16 strips: four waves side by side with four strips each, times two that
// share out every K tile, two groups of 32 each.  A weight operand is made once and meets all rows; rows are read from LDS by four waves, not
// eight.  Between two MFMAs stand two vector instructions that make the next group's operands, so a wave's MFMAs are hardly ever held up by them;
// clumps of them ahead of the MFMAs, and all copies at once behind the barrier, cost 7 %.  2 of 8 experts of 4096 -> 2 x 14336, 1024 bf16 tokens: 860 us
// with exact operands and two workgroups of 64 rows to a CU, 685 with rounded ones, 596 with one of 128 rows, 529 now; without its
// copies 411, without its MFMAs 412, so it is neither alone but what of both does not overlap: eight waves that meet at a barrier per K tile.
// Tried on that case, where a workgroup's start and end hardly count (32 K tiles): workgroups that stay and look the next item up behind the
// products (529 -> 550: tiles differ in length); K tiles started at different places by the workgroups that share rows (566 -> 692); row
// tiles outermost (566 -> 590).
//   OP 0 / 1  exact operands, f16 / bf16 rows: a strip and group starts from zero (bf16: from the product that takes the bias off, one
//             for four strips), its sums are scaled on their way into the fp32 accumulators, four FMAs per MFMA
//   OP 2      f16 rows (bf16 ones behind a power of two per row), operands round_f16(scale * q), one MFMA and no FMAs
template <int BITS, int RB>
struct ManyShape {
    static constexpr int XTILE = RB * 4096;
    static constexpr int WQ = 1024 * (BITS / 4);
    static constexpr int WTILE = 2 * WQ + 256;                   // two strips
    static constexpr int STEP = XTILE + 8 * WTILE;
    static constexpr int BUDGET = 156 * 1024;
    static constexpr int FIT = BUDGET / STEP;
    static constexpr int D = FIT > 5 ? 5 : FIT;
    static constexpr int XC = (RB + 1) / 2;
    static constexpr int WC = 2 * (BITS / 4) + 1;
    static_assert(D >= 3 && RB * 16384 <= BUDGET, "LDS");
};
constexpr int many_rows(int bits, int op) { return bits == 4 && op == 2 ? 128 : 64; }          // rows of a tile (Q8 words leave LDS for no more, exact operands registers)

template <int I, int N, class F>
__device__ __forceinline__ void static_for(F&& f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

template <int BITS, int OP, bool PAIR, int RB>
__device__ __forceinline__ void many_tile(const ExpertsArgs& g, int e, const int32_t* list, int n, int strip0, uint8_t* smem)
{
    using S = ManyShape<BITS, RB>;
    constexpr int D = S::D, CS = 4, OPM = OP == 1 ? XBF16 : XF16;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = wave >> 1, kh = wave & 1;
    const int i16 = lane & 15, oct = lane >> 4;
    const int G = g.K / kGroup;

    // the rows' pairs and factors, for the copies and - by then a trip to memory each - for the end
    int32_t* const row_pair = reinterpret_cast<int32_t*>(smem + S::BUDGET);
    float* const row_factor = reinterpret_cast<float*>(smem + S::BUDGET + 512);
    if (tid < n) {
        const int p = list[tid];
        row_pair[tid] = p;
        if (OP == 2) row_factor[tid] = g.unscale ? g.unscale[p / g.xdiv] : 1.0f;
    }

    // copies: a wave's share of the rows (block b = rows 8 * (b / 2) .. + 8, line b % 2 of the K tile), and strips 2 * wave, + 1
    const int crow = lane >> 3, piece = (lane & 7) ^ crow;
    uint32_t xoff[S::XC];
    int xblk[S::XC];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < S::XC; c++) {
        xblk[c] = min(c * 8 + wave, RB * 4 - 2 + (wave & 1));
        xoff[c] = (uint32_t)(row_pair[min((xblk[c] >> 1) * 8 + crow, n - 1)] / g.xdiv) * (uint32_t)(g.K * 2);
    }
    const int strip = min(strip0 + wave * 2, g.strips - 1), second = min(strip + 1, g.strips - 1);
    const uint8_t* const wsrc = g.w + ((int64_t)e * g.strips + strip) * g.KT * kTileBytes<BITS>;
    const uint32_t wstep = (uint32_t)(second - strip) * (uint32_t)(g.KT * kTileBytes<BITS>);
    const uint32_t q_off = (uint32_t)lane * 16u, sc_off = (lane >= 8 ? wstep : 0u) + (uint32_t)(kTileQBytes<BITS> + (lane & 7) * 16);
    const int whole = G / 4;
    // piece c of step `step`: the words, which come from further away, the scales, the rows' blocks
    constexpr int PIECES = S::XC + S::WC;
    auto copy_piece = [&](auto c_, int step, int buf) {
        constexpr int c = decltype(c_)::value;
        const int kt = min(step, g.KT - 1);
        const uint32_t at = (uint32_t)(buf * S::STEP), wat = at + S::XTILE + wave * S::WTILE;
        if constexpr (c + 1 < S::WC) {
            constexpr int q = c / 2, second_strip = c % 2;
            copy_to_lds(wat + second_strip * S::WQ + q * 1024, wsrc + (int64_t)kt * kTileBytes<BITS> + (second_strip ? wstep : 0u) + q * 1024, q_off);
        } else if constexpr (c < S::WC) {
            copy_lanes_to_lds(wat + 2 * S::WQ, wsrc + (int64_t)kt * kTileBytes<BITS>, sc_off, 0xffffull);
        } else {
            constexpr int block = c - S::WC;
            const uint32_t from = (uint32_t)min(kt * 4 + (wave & 1) * 2 + (piece >> 2), G - 1) * 64u + (uint32_t)(piece & 3) * 16u;   // (past the end of a row: its last group)
            copy_to_lds(at + xblk[block] * 1024, g.x, xoff[block] + from);
        }
    };
#pragma unroll
    for (int d = 0; d < D - 1; d++) static_for<0, PIECES>([&](auto c_) { copy_piece(c_, d, d); });

    float4_t acc[RB][CS];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int s = 0; s < CS; s++) acc[i][s] = (float4_t){0.f, 0.f, 0.f, 0.f};
    const uint32_t magic = OPM == XF16 ? q4_magic_vgpr() : magic16_vgpr();
    const uint32_t raw = (uint32_t)((i16 >> 3) * 2048 + kh * 1024 + (i16 & 7) * 128 + ((oct ^ (i16 & 7)) * 16));
    const uint32_t wread = (uint32_t)(S::XTILE + col * 2 * S::WTILE + (BITS == 4 ? lane * 16 + kh * 8 : kh * 1024 + lane * 16));
    const uint32_t sread = (uint32_t)(S::XTILE + col * 2 * S::WTILE + 2 * S::WQ + i16 * 8 + kh * 4);
    Frag16 off;
    const uint32_t offw = BITS == 4 ? kNeg24x2 : kBf16Neg128x2;
    off.u = (u32x4_t){offw, offw, offw, offw};

    // a wave's packed words and scales of a step, the operands of one of its two groups, and their products with all rows
    struct Words {
        uint32_t q[CS][BITS / 2], sc[CS];
    };
    auto read_words = [&](Words& w, const uint8_t* at) {
#pragma unroll
        for (int s = 0; s < CS; s++) {
            const uint8_t* const p = at + (s >> 1) * S::WTILE + (s & 1) * S::WQ + wread;
            if constexpr (BITS == 4) {
                const u32x2_t v = *reinterpret_cast<const u32x2_t*>(p);
                w.q[s][0] = v[0];
                w.q[s][1] = v[1];
            } else {
                const u32x4_t v = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
                for (int k = 0; k < 4; k++) w.q[s][k] = v[k];
            }
            w.sc[s] = *reinterpret_cast<const uint32_t*>(at + (s >> 1) * S::WTILE + (s & 1) * 128 + sread);
        }
    };
    // word k of strip s's operand of group j: two of a lane's eight weights
    auto operand_word = [&](Frag16& b, const Words& w, int s, int j, int k) {
        uint32_t v;
        if constexpr (BITS == 4) {
            const uint32_t src = w.q[s][k >> 1] >> (k & 1 ? 8 : 0);
            if constexpr (OPM == XBF16) {
                v = q4_bf16_word(w.q[s][0], w.q[s][1], j, k, magic);
            } else if (j == 0) {
                v = as_u32(as_h2((src & 0x000F000Fu) | magic) + (half2_t){(_Float16)-1032.0f, (_Float16)-1032.0f});
            } else {
                v = as_u32(as_h2((src & 0x00F000F0u) | magic) * (half2_t){(_Float16)0.0625f, (_Float16)0.0625f} + (half2_t){(_Float16)-72.0f, (_Float16)-72.0f});
            }
        } else {
            const uint32_t src = w.q[s][2 * j + (k >> 1)];
            if constexpr (OPM == XBF16) {
                const uint32_t h = k & 1 ? src >> 16 : src;
                v = pack_bf16x2((float)(h & 0xffu), (float)((h >> 8) & 0xffu));
            } else {
                v = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, src, k & 1 ? 0x04030402u : 0x04010400u)) + (half2_t){(_Float16)-1152.0f, (_Float16)-1152.0f});
            }
        }
        if constexpr (OP == 2) {
            const _Float16 f = __builtin_bit_cast(_Float16, (uint16_t)(j ? w.sc[s] >> 16 : w.sc[s] & 0xffffu));
            v = as_u32(as_h2(v) * (half2_t){f, f});
        }
        b.u[k] = v;
    };
    Words w[2];
    Frag16 b[2][CS], a[4];
    float4_t d[3], bias[2];                                      // exact operands: products on their way to the sums
    int buf = 0;
    auto read_a = [&](Frag16& f, const uint8_t* at, int i, int j) { f.u = *reinterpret_cast<const u32x4_t*>(at + i * 4096 + (j ? raw ^ 64u : raw)); };
    constexpr int MMAS = RB * CS;
    // Group J of a step's two: the products of the operands b[J] with all rows, in an order that is kept: between the MFMAs the rows' operands three
    // row blocks ahead, the words of the next group's operands (`next`: of this step's or the next one's words), a row block at a time.
    auto group = [&](auto j_, const uint8_t* at, const uint8_t* at_next, const Words& now, const Words& next, int copy_step, int free) {
        constexpr int J = decltype(j_)::value;
        auto scaled = [&](auto m_) {
            constexpr int m = decltype(m_)::value, i = m / CS, s = m % CS;
            const float f = f16_bits_to_f32(J ? now.sc[s] >> 16 : now.sc[s] & 0xffffu);
#pragma unroll
            for (int r = 0; r < 4; r++) acc[i][s][r] = fmaf(f, d[m % 3][r], acc[i][s][r]);
        };
        static_for<0, MMAS>([&](auto m_) {
            constexpr int m = decltype(m_)::value, i = m / CS, s = m % CS;
            if constexpr (s == 0) {
                if constexpr (i + 3 < RB) read_a(a[(i + 3) % 4], at, i + 3, J);
            }
            if constexpr (OP == 2) {
                acc[i][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % 4].h, b[J][s].h, acc[i][s], 0, 0, 0);
            } else if constexpr (OP == 0) {
                d[m % 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i % 4].h, b[J][s].h, (float4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            } else {
                if constexpr (s == 0 && i == 0) bias[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0].b, off.b, (float4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                d[m % 3] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i % 4].b, b[J][s].b, bias[i & 1], 0, 0, 0);
                if constexpr (s == 2 && i + 1 < RB)
                    bias[(i + 1) & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[(i + 1) % 4].b, off.b, (float4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            }
            if constexpr (OP != 2 && m >= 2) scaled(std::integral_constant<int, (m >= 2 ? m - 2 : 0)>{});
            // the next group's words: from LDS since the first row block, so behind it where there are more
            constexpr int skip = J == 1 && RB > 1 ? CS : 0, slots = MMAS - skip;
            if constexpr (m >= skip) {
                constexpr int lo = (m - skip) * 16 / slots, hi = (m - skip + 1) * 16 / slots;
#pragma unroll
                for (int k = lo; k < hi; k++) operand_word(b[1 - J][k >> 2], next, k >> 2, 1 - J, k & 3);
            }
            // the copies spread out: all at once behind the barrier they held up the MFMAs behind them until the address unit had taken
            // them in (1024 rows on 8 experts of 4096 -> 14336: 560 us)
            if constexpr (J == 1) static_for<m * PIECES / MMAS, (m + 1) * PIECES / MMAS>([&](auto c_) { copy_piece(c_, copy_step, free); });
            if constexpr (s == CS - 1) __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (OP != 2) {
            scaled(std::integral_constant<int, (MMAS >= 2 ? MMAS - 2 : 0)>{});
            scaled(std::integral_constant<int, MMAS - 1>{});
        }
        // the first three row blocks of what follows
        read_a(a[0], at_next, 0, 1 - J);
        if constexpr (RB > 1) read_a(a[1], at_next, 1, 1 - J);
        if constexpr (RB > 2) read_a(a[2], at_next, 2, 1 - J);
    };
    // One barrier per step, in its middle.  Ahead of it the first group's products, whose operands are there; behind it the next step's copies
    // are in LDS and the last step's place is free.
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((D - 2) * (S::XC + S::WC)) : "memory");
    read_words(w[0], smem);
    read_a(a[0], smem, 0, 0);
    if constexpr (RB > 1) read_a(a[1], smem, 1, 0);
    if constexpr (RB > 2) read_a(a[2], smem, 2, 0);
#pragma unroll
    for (int s = 0; s < CS; s++)
#pragma unroll
        for (int k = 0; k < 4; k++) operand_word(b[0][s], w[0], s, 0, k);
    auto step_ = [&](int step, const Words& now, Words& next, bool first, bool second) {
        const uint8_t* const at = smem + buf * S::STEP;
        const int free = buf == 0 ? D - 1 : buf - 1;
        buf = buf + 1 == D ? 0 : buf + 1;
        const uint8_t* const at_next = smem + buf * S::STEP;
        if (first) group(std::integral_constant<int, 0>{}, at, at, now, now, 0, 0);
        // (no wait for reads of LDS: those on their way are of this step's place, the last step's went into MFMAs ahead of here)
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((D - 3) * (S::XC + S::WC)) : "memory");
        read_words(next, at_next);
        if (second) group(std::integral_constant<int, 1>{}, at, at_next, now, next, step + D - 1, free);
    };
    // (whole K tiles by themselves: a body that may end early costs a move of every sum per step)
    int step = 0;
    for (; step + 2 <= whole; step += 2) {
        step_(step, w[0], w[1], true, true);
        step_(step + 1, w[1], w[0], true, true);
    }
    if (step < whole) {
        step_(step, w[0], w[1], true, true);
        w[0] = w[1];
        step++;
    }
    if (whole < g.KT) {
        const int mine = G - whole * 4 - kh * 2;
        step_(step, w[0], w[1], mine > 0, mine > 1);
    }
    // (no copy may land in LDS that holds something else by then)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    // the two halves of K meet: the first wave finishes row blocks 0 .. H - 1, the second the rest
    constexpr int H = (RB + 1) / 2;
    float4_t* const red = reinterpret_cast<float4_t*>(smem) + col * (RB * CS * 64) + lane;
#pragma unroll
    for (int i = 0; i < RB; i++)
        if ((i < H) == (kh == 1))
#pragma unroll
            for (int s = 0; s < CS; s++) red[(i * CS + s) * 64] = acc[i][s];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RB; i++) {
        if ((i < H) == (kh == 1)) continue;
        float4_t v[CS];
#pragma unroll
        for (int s = 0; s < CS; s++) v[s] = acc[i][s] + red[(i * CS + s) * 64];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int m = i * 16 + oct * 4 + r;
            if (m >= n) continue;
            const float f = OP == 2 ? row_factor[m] : 1.0f;
            const int64_t at = (int64_t)row_pair[m] * g.n_out;
#pragma unroll
            for (int s = 0; s < CS; s += PAIR ? 2 : 1) {
                const int st = strip0 + col * 4 + s;
                if (st >= g.strips) continue;
                if constexpr (PAIR) store_out(g.y, g.ydt, at + st * 8 + i16, silu_mul(v[s][r] * f, v[s + 1][r] * f));
                else store_out(g.y, g.ydt, at + st * 16 + i16, v[s][r] * f);
            }
        }
    }
}

template <int BITS, int OP, bool PAIR>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void experts_many_kernel(ExpertsArgs g)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int items = g.lists[g.E + 1] * g.groups;
    const int per_xcd = (items + 7) >> 3;
    const int item = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per_xcd || item >= items) return;
    // an expert's items one after the other, the row tiles of 16 strips together: they meet the same words in the XCD's L2, and all
    // of the expert's items its rows
    const int4* const tiles = reinterpret_cast<const int4*>(g.lists + lists_tiles_at(g.E));
    const int some = __builtin_amdgcn_readfirstlane(item / g.groups), packed = __builtin_amdgcn_readfirstlane(tiles[some].w);
    const int first = some - (packed >> 16), count = packed & 0xffff, rest = item - first * g.groups;
    const int tile_n = __builtin_amdgcn_readfirstlane(rest / count);
    const int4 t = tiles[first + rest - tile_n * count];
    const int e = __builtin_amdgcn_readfirstlane(t.x), n = __builtin_amdgcn_readfirstlane(t.z);
    const int32_t* const list = g.lists + lists_order_at(g.P, g.E) + __builtin_amdgcn_readfirstlane(t.y);
    if (n <= 0) return;
    auto go = [&](auto rb) { many_tile<BITS, OP, PAIR, decltype(rb)::value>(g, e, list, n, tile_n * 16, smem); };
    using std::integral_constant;
    const int rb = (n + 15) / 16;
    if (rb == 1) go(integral_constant<int, 1>{});
    else if (rb == 2) go(integral_constant<int, 2>{});
    else if (rb == 3) go(integral_constant<int, 3>{});
    else if (many_rows(BITS, OP) == 64 || rb == 4) go(integral_constant<int, 4>{});
    else if constexpr (many_rows(BITS, OP) == 128) {
        if (rb == 5) go(integral_constant<int, 5>{});
        else if (rb == 6) go(integral_constant<int, 6>{});
        else if (rb == 7) go(integral_constant<int, 7>{});
        else go(integral_constant<int, 8>{});
    }
}

// Few rows per expert: 8 or 16 at a time.  Two workgroups share a CU where their LDS allows it: one's start and end overlap the other's stream.
// the blocks of eight rows that a piece has at most, and the LDS of the largest of 1, 2, 4, 8
template <int XM, int COLS>
constexpr int few_rows()
{
    return XM == XF32 ? (COLS == 8 ? 4 : COLS == 4 ? 2 : 1) : COLS;
}

template <int BITS, int XM, int COLS, int XB = 1>
constexpr int few_ring()
{
    if constexpr (XB > few_rows<XM, COLS>()) return RowShape<BITS, XM, true>::LDS;
    else return std::max(Shape<BITS, XM, XB, COLS, kFewLds>::LDS, few_ring<BITS, XM, COLS, XB * 2>());
}

// f(XB) for XB = FIRST, 2 FIRST, .. LAST until one answers true
template <int XB, int LAST, class F>
__device__ __forceinline__ void static_for_rows(F&& f)
{
    if (f(std::integral_constant<int, XB>{})) return;
    if constexpr (XB < LAST) static_for_rows<XB * 2, LAST>(f);
}

template <int BITS, int XM, bool PAIR, int COLS>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(4, 4))) void experts_few_kernel(ExpertsArgs g)
{
    // (the copies count LDS addresses from zero: these kernels have no static LDS)
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    int32_t* const rows = reinterpret_cast<int32_t*>(smem + few_ring<BITS, XM, COLS>());          // the pairs of the expert, kMaxDirect at a time
    const int lane = threadIdx.x & 63, slot = blockIdx.y, strip0 = blockIdx.x * (2 * COLS);
    const int e = __builtin_amdgcn_readfirstlane(g.by_pair ? g.ids[slot] : slot);
    if ((unsigned)e >= (unsigned)g.E) return;
    auto all = [&](int n) {
        const int32_t* const list = rows;
        for (int r0 = 0; r0 < n;) {
            if (r0) __syncthreads();
            if (n - r0 == 1) {
                expert_row<BITS, XM, PAIR, COLS>(g, e, __builtin_amdgcn_readfirstlane(list[r0]), strip0, smem);
                r0 += 1;
                continue;
            }
            // (rows in one piece where it can be had: every piece reads the weights again)
            static_for_rows<1, few_rows<XM, COLS>()>([&](auto xb_) {
                constexpr int XB = decltype(xb_)::value;
                if (XB * 8 < n - r0 && XB < few_rows<XM, COLS>()) return false;
                expert_tile<BITS, XM, PAIR, XB, COLS, kFewLds>(g, e, list + r0, min(n - r0, XB * 8), strip0, smem);
                r0 += XB * 8;
                return true;
            });
        }
    };
    if (g.lists) {
        const int a = __builtin_amdgcn_readfirstlane(g.lists[e]), n = __builtin_amdgcn_readfirstlane(g.lists[e + 1]) - a;
        const int32_t* const order = g.lists + lists_order_at(g.P, g.E) + a;
        for (int r = 0; r < n; r += kMaxDirect) {
            if (r) __syncthreads();
            if (r + (int)threadIdx.x < n) rows[threadIdx.x] = order[r + threadIdx.x];
            __syncthreads();
            all(min(n - r, kMaxDirect));
        }
        return;
    }
    // the expert's pairs among the ids; every wave looks for itself
    int n = 0, first = -1;
    if (g.single) {
        n = 1;
        if (threadIdx.x == 0) rows[0] = slot;
    } else {
        for (int p0 = 0; p0 < (int)g.P; p0 += 64) {
            const bool mine = p0 + lane < (int)g.P && g.ids[p0 + lane] == e;
            const uint64_t who = __ballot(mine);
            if (mine && threadIdx.x < 64) rows[n + __popcll(who & ((1ull << lane) - 1))] = p0 + lane;
            if (who && first < 0) first = p0 + __builtin_ctzll(who);
            n += __popcll(who);
        }
        if (n == 0 || (g.by_pair && first != slot)) return;
    }
    __syncthreads();
    all(n);
}

// ---- few tokens, the way back: a token's experts one after the other as one long K, their weights on the groups' scales --------------
//
// y[t, n] = residual[t, n] + sum over the pairs and K: workgroup = a strip of 16 columns and a token, its eight waves share out the
// KT tiles of every pair that has an expert (a token's absent pairs cost nothing).  One launch and no sums in memory, but an expert's weights are
// read once per token.
struct TokenArgs {
    const uint8_t* w;
    const void* x;
    const int32_t* ids;
    const float* weights;
    const void* residual;
    int top_k, K, KT, strips, E;
    uint32_t per_kt;            // 2^32 / KT, rounded up: what a tile's number is multiplied with for its pair (exact below 2^32 / KT)
    void* y;
    int ydt;
};
constexpr int kTokenMaxKT = 4096;                                // 64 * KT tiles

template <int BITS, int XM>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(4, 4))) void experts_token_kernel(TokenArgs g)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    constexpr int XS = XM == XF32 ? 4 : 2;
    const int lane = threadIdx.x & 63, strip = blockIdx.x, t = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int N = g.strips * 16, n = strip * 16 + (lane & 15), G = g.K / kGroup;
    const int64_t p0 = (int64_t)t * g.top_k, at = (int64_t)t * N + n;
    int id = lane < g.top_k ? g.ids[p0 + lane] : -1, pair = lane;       // lane j: pair j's
    float weight = lane < g.top_k ? g.weights[p0 + lane] : 0.f;
    const float first = g.residual ? load_out(g.residual, g.ydt, at) : 0.f;
    const uint64_t with = __ballot((unsigned)id < (unsigned)g.E);
    const int pairs = __popcll(with);
    if (pairs != g.top_k) {
        // lane j: the j-th pair that has an expert, in their order; the rest behind them, and no tile is theirs
        const uint64_t below = (1ull << lane) - 1;
        const int to = 4 * ((with >> lane) & 1 ? __popcll(with & below) : pairs + __popcll(~with & below));
        id = __builtin_amdgcn_ds_permute(to, id);
        pair = __builtin_amdgcn_ds_permute(to, pair);
        weight = __builtin_bit_cast(float, __builtin_amdgcn_ds_permute(to, __builtin_bit_cast(int, weight)));
    }
    const int tiles = pairs * g.KT;
    float acc[2] = {0.f, 0.f};
    if (tiles) stream_row<BITS, XM, false>((tiles + 15) / 16, [&](int step, int s) {
        const int u = (step * 8 + wave) * 2 + s, v = min(u, tiles - 1);
        const int j = g.KT == 1 ? v : (int)__umulhi((uint32_t)v, g.per_kt), kt = v - j * g.KT;
        return RowTile{g.w + (((int64_t)__builtin_amdgcn_readlane(id, j) * g.strips + strip) * g.KT + kt) * kTileBytes<BITS>,
                       static_cast<const char*>(g.x) + (p0 + __builtin_amdgcn_readlane(pair, j)) * g.K * XS + (int64_t)kt * (kTileK * XS),
                       u < tiles ? min(G - kt * 4, 4) : 0, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), j))};
    }, acc, smem);
    float* const red = reinterpret_cast<float*>(smem);
    __syncthreads();
    if (lane < 16) red[wave * 16 + lane] = acc[0] + acc[1];
    __syncthreads();
    if (threadIdx.x >= 16) return;
    float v = first;
#pragma unroll
    for (int k = 0; k < 8; k++) v += red[k * 16 + lane];
    store_out(g.y, g.ydt, at, v);
}

// ---- y[t] = residual[t] + sum_j weights[t, j] z[t, j], in order of j, fp32 ----------------------------------------
__global__ __launch_bounds__(256) void experts_sum_kernel(const float* __restrict__ z, const int32_t* __restrict__ ids, const float* __restrict__ weights,
                                                          const void* residual, int T, int top_k, int E, int N, void* y, int ydt)
{
    const int t = blockIdx.y;
    const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= N) return;
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    const int64_t at = (int64_t)t * N + n;
    if (residual)
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = load_out(residual, ydt, at + i);
    for (int j = 0; j < top_k; j++) {
        const int64_t p = (int64_t)t * top_k + j;
        if ((unsigned)ids[p] >= (unsigned)E) continue;
        const float w = weights[p];
        const float4_t d = *reinterpret_cast<const float4_t*>(z + p * N + n);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = fmaf(w, d[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) store_out(y, ydt, at + i, v[i]);
}

template <int BITS, int XM, bool PAIR, int COLS>
void launch_few(ExpertsArgs g, int slots, hipStream_t st)
{
    constexpr int lds = few_ring<BITS, XM, COLS>() + kMaxDirect * 4;
    (void)LdsRequest<&experts_few_kernel<BITS, XM, PAIR, COLS>, lds>::registered;
    g.groups = (g.strips + 2 * COLS - 1) / (2 * COLS);
    experts_few_kernel<BITS, XM, PAIR, COLS><<<dim3(g.groups, slots), dim3(512), lds, st>>>(g);
}

template <int BITS, int OP, bool PAIR>
void launch_many(ExpertsArgs g, hipStream_t st)
{
    constexpr int lds = ManyShape<BITS, 1>::BUDGET + 1024;
    (void)LdsRequest<&experts_many_kernel<BITS, OP, PAIR>, lds>::registered;
    g.groups = (g.strips + 15) / 16;
    const int64_t items = lists_tiles_max(g.P, g.E) * g.groups;
    experts_many_kernel<BITS, OP, PAIR><<<dim3((unsigned)((items + 7) / 8 * 8)), dim3(512), lds, st>>>(g);
}

template <int BITS, int XM>
void launch_token(const TokenArgs& g, int T, hipStream_t st)
{
    constexpr int lds = RowShape<BITS, XM, false>::LDS;
    (void)LdsRequest<&experts_token_kernel<BITS, XM>, lds>::registered;
    experts_token_kernel<BITS, XM><<<dim3(g.strips, T), dim3(512), lds, st>>>(g);
}

struct Tuning {
    int cols = 0, many = 0, token = 0;
} g_tuning;

}  // namespace

void set_experts_tuning(int cols, int many, int token) { g_tuning = {cols, many, token}; }

size_t experts_lists_bytes(int64_t P, int E) { return ((size_t)(lists_order_at(P, E) + P) * 4 + 255) / 256 * 256; }

// Where the tiles of many rows beat one pass of few.  us, few / many at 16, 24, 32, 48 rows to an expert: Q4, rounded operands, up 8 of 128 of 2048 -> 2 x 768
// 64 / 65, 85 / 77, 105 / 86, 134 / 98, 2 of 8 of 4096 -> 2 x 14336 124 / 138, 143 / 146, 176 / 164, 258 / 194; exact operands 59 / 73, 76 / 88, 92 / 98, 127 / 118 and
// 116 / 150, 136 / 150, 162 / 185, 234 / 213; Q8, exact, 109 / 103, 126 / 118, 153 / 119, 196 / 132 and 204 / 227, 217 / 225, 264 / 237, 372 / 245.
bool experts_many(const WeightView& w, int E, int xdt, int64_t P, bool fast)
{
    const int thr = g_tuning.many ? g_tuning.many : w.bits == 8 ? 20 : fast ? 24 : 40;
    return xdt != kF32 && P >= thr * std::min<int64_t>(P, E);
}

// pairs of a launch (1024 at least, but for E < 17 960): a grid has fewer than 2^32 threads (at most E + P / 64 row tiles by strips / 16 workgroups of 512)
int64_t experts_pairs_max(const WeightView& w, int E) { return (((int64_t)1 << 23) / ((w.NT / E + 15) / 16) - E - 1) * kRowTile; }

size_t experts_stage_bytes(int64_t rows, int K) { return (size_t)rows * K * 2 + ((size_t)rows * 4 + 255) / 256 * 256; }

hipError_t launch_experts(const WeightView& w, int E, bool pair, const void* x, int xdt, int64_t P, int top_k, int xdiv, const int32_t* ids, void* y, int ydt,
                          int num_cus, bool fast, void* lists, void* stage, hipStream_t st)
{
    const int strips = w.NT / E, n_out = strips * 16 / (pair ? 2 : 1);
    const int64_t met = std::min<int64_t>(P, E);
    const bool many = experts_many(w, E, xdt, P, fast);
    int32_t* const L = static_cast<int32_t*>(lists);
    const bool listed = many || P > kMaxDirect;
    const int op = fast ? 2 : xdt == kF16 ? 0 : 1;
    const bool staged = many && op == 2 && xdt == kBF16;
    const int64_t rows = P / xdiv;
    uint16_t* const half = static_cast<uint16_t*>(stage);
    float* const unscale = staged ? reinterpret_cast<float*>(half + rows * w.K) : nullptr;
    if (listed) {
        int bits = 0;
        while ((1 << bits) < E) bits++;
        (void)LdsRequest<&experts_prepare_kernel, (18 * 1024 + 32) * 4>::registered;
        const int list_blocks = (int)std::min<int64_t>((P + 2047) / 2048, 32);
        experts_prepare_kernel<<<dim3((unsigned)(list_blocks + (staged ? (rows + 15) / 16 : 0))), 1024, (18 * E + 32) * 4, st>>>(
            ids, (int)P, E, bits, many_rows(w.bits, op), list_blocks, L, static_cast<const uint16_t*>(x), xdiv, w.K, half, unscale);
    }
    ExpertsArgs g = {w.base, x, ids, listed ? L : nullptr, P, xdiv, w.K, w.KT, strips, E, 0, !listed && P <= top_k, !listed && (P <= top_k || P <= E), y, ydt, n_out, nullptr};
    using std::integral_constant;
    if (many) {
        if (staged) {
            g.x = half;
            g.unscale = unscale;
        }
        auto go = [&](auto b_, auto op_) {
            if (pair) launch_many<decltype(b_)::value, decltype(op_)::value, true>(g, st);
            else launch_many<decltype(b_)::value, decltype(op_)::value, false>(g, st);
        };
        auto with_op = [&](auto b_) {
            if (op == 0) go(b_, integral_constant<int, 0>{});
            else if (op == 1) go(b_, integral_constant<int, 1>{});
            else go(b_, integral_constant<int, 2>{});
        };
        w.bits == 4 ? with_op(integral_constant<int, 4>{}) : with_op(integral_constant<int, 8>{});
        return hipGetLastError();
    }
    const int slots = g.by_pair ? (int)P : E;
    // Waves side by side, or behind each other along K where that leaves CUs without work: of strips of met experts per CU there go 16 to a
    // workgroup of eight waves side by side, 8, 4, 2.  us per call with 8 / 4 / 2 / 1 side by side, up, Q4, f16 rows: 8 of 128 experts of 2048 -> 2 x 768 at
    // 1 / 4 / 16 tokens 12.6 / 7.9 / 5.5 / 5.4, 16.2 / 13.9 / 13.9 / 15.3, 31.8 / 30.5 / 32.5 / 39.6; back, 2 of 8 of 14336 -> 4096 at 16 tokens (2048 strips) 84.5 / 48.6 /
    // 45.0 / 44.0.  Eight only on a short K (few steps to a workgroup): 8 of 256 of 1024 -> 2 x 512 at 16 tokens 15.0 / 16.4 / 19.4, Q8 20.9 / 24.0 / 29.2,
    // but Q8 6 of 64 of 2048 -> 2 x 1408 62.5 / 56.5 / 61.5.
    const int64_t work = met * strips;
    const int cols = g_tuning.cols ? g_tuning.cols : work >= (w.bits == 8 ? 12 : 32) * num_cus && w.KT <= 12 ? 8 : work > 8 * num_cus || w.KT < 4 ? 4 : work >= 4 * num_cus || w.KT < 8 ? 2 : 1;
    auto go = [&](auto b_, auto x_, auto pair_) {
        constexpr int B = decltype(b_)::value, X = decltype(x_)::value;
        constexpr bool P2 = decltype(pair_)::value;
        if (cols == 8) launch_few<B, X, P2, 8>(g, slots, st);
        else if (cols == 4) launch_few<B, X, P2, 4>(g, slots, st);
        else if (cols == 2) launch_few<B, X, P2, 2>(g, slots, st);
        else launch_few<B, X, P2, 1>(g, slots, st);
    };
    auto with_pair = [&](auto b_, auto x_) { pair ? go(b_, x_, std::true_type{}) : go(b_, x_, std::false_type{}); };
    auto with_x = [&](auto b_) {
        if (xdt == kF16) with_pair(b_, integral_constant<int, XF16>{});
        else if (xdt == kBF16) with_pair(b_, integral_constant<int, XBF16>{});
        else with_pair(b_, integral_constant<int, XF32>{});
    };
    w.bits == 4 ? with_x(integral_constant<int, 4>{}) : with_x(integral_constant<int, 8>{});
    return hipGetLastError();
}

// Token by token: no second launch and no sums in memory, but an expert's weights come once per token.  us, token by token / with sums in memory, 1, 2, 4, 8
// tokens: 8 of 128 of 768 -> 2048 6.7 / 9.3, 6.7 / 9.6, 9.4 / 11.6, 16.5 / 16.4; 8 of 256 of 512 -> 1024 5.3 / 7.9, 5.3 / 8.8, 5.5 / 9.2, 7.7 / 10.5; 2 of 8 of 14336 -> 4096
// 19.3 / 17.1, 29 / 27, 52 / 39, 97 / 43: up to 36864 tiles of weights, and no more pairs than experts.
bool experts_sum_by_token(const WeightView& w, int E, int64_t T, int top_k)
{
    if (!experts_token_serves(w)) return false;
    if (g_tuning.token) return g_tuning.token == 1;
    return T * top_k <= E && T * top_k * (w.NT / E) * w.KT <= 36864;
}

bool experts_token_serves(const WeightView& w) { return w.KT <= kTokenMaxKT; }

hipError_t launch_experts_token(const WeightView& w, int E, const void* x, int xdt, int64_t T, int top_k, const int32_t* ids, const float* weights,
                                const void* residual, void* y, int ydt, hipStream_t st)
{
    const TokenArgs g = {w.base, x, ids, weights, residual, top_k, w.K, w.KT, w.NT / E, E, (uint32_t)((((uint64_t)1 << 32) + w.KT - 1) / w.KT), y, ydt};
    auto with_x = [&](auto b_) {
        constexpr int B = decltype(b_)::value;
        if (xdt == kF16) launch_token<B, XF16>(g, (int)T, st);
        else if (xdt == kBF16) launch_token<B, XBF16>(g, (int)T, st);
        else launch_token<B, XF32>(g, (int)T, st);
    };
    w.bits == 4 ? with_x(std::integral_constant<int, 4>{}) : with_x(std::integral_constant<int, 8>{});
    return hipGetLastError();
}

hipError_t launch_experts_sum(const float* z, const int32_t* ids, const float* weights, const void* residual, int64_t T, int top_k, int E, int N, void* y,
                              int ydt, hipStream_t st)
{
    experts_sum_kernel<<<dim3((N / 4 + 255) / 256, (unsigned)T), 256, 0, st>>>(z, ids, weights, residual, (int)T, top_k, E, N, y, ydt);
    return hipGetLastError();
}

}  // namespace cybq
