// experts.hip - products of rows with the block-quantised weights of the experts they were sent to.
//
// A stack of E experts is one weight of E * n rows (n a multiple of 16: expert e is the strips [e * n / 16, (e + 1) * n / 16)).
// A pair p = t * top_k + j is token t with its j-th expert ids[p]; an id outside 0 .. E - 1 is no expert.
//
//   out[p, :] = x[p / xdiv, :] W_ids[p]^T         xdiv = top_k: the tokens' rows; 1: a row of its own for every pair
//
// Operands are exact in every kernel: the integers q (bf16 rows: the numbers 128 + u and a second product that takes the bias off), each
// group's sums times its scale in fp32.  No row statistics, no staging, and scales that leave f16's range when multiplied with q do no harm.
#include <algorithm>

#include "gemv_parts.h"

namespace cybq {

namespace {

#include "gemm_parts.h"

// ---- which rows does an expert have: the lists ------------------------------------------------------------------
//
// int32 words: [0, E]: where expert e's pairs start in the order below, [E + 1]: number of row tiles, then (4-word aligned) the tiles
// {expert, first pair, pairs, 0}, then the pairs in order of expert and, within one, of their number.
struct Lists {
    const int32_t* offsets;
    const int32_t* tile_count;
    const int4* tiles;
    const int32_t* order;
};

constexpr int kRowTile = 128;                                    // rows of a full tile
__host__ __device__ inline int64_t lists_tiles_max(int64_t P, int E) { return P / kRowTile + (P < E ? P : E); }
__host__ __device__ inline int64_t lists_tiles_at(int E) { return (E + 2 + 3) / 4 * 4; }
__host__ __device__ inline int64_t lists_order_at(int64_t P, int E) { return lists_tiles_at(E) + 4 * lists_tiles_max(P, E); }

__device__ __forceinline__ int block_exclusive_scan(int v, int* wave_sums, int* total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < waves; i++) {
        const int w = wave_sums[i];
        if (i < wave) before += w;
        all += w;
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

// One workgroup: a histogram per wave over its share of the pairs, a scan over experts and waves, then every wave places its pairs in
// order: lanes with the same expert find each other by one ballot per bit of the id, so the order does not hang on atomics.
__global__ __launch_bounds__(1024) void lists_kernel(const int32_t* __restrict__ ids, int P, int E, int bits, int32_t* __restrict__ out)
{
    extern __shared__ int hist[];                                // [16][E], then 16 wave sums
    int* const wave_sums = hist + 16 * E;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < 16 * E; i += 1024) hist[i] = 0;
    __syncthreads();
    const int share = (P + 1023) / 1024 * 64;                    // pairs per wave, whole rounds of 64
    const int lo = min(wave * share, P), hi = min(lo + share, P);
    int* const my = hist + wave * E;
    for (int p = lo + lane; p < hi; p += 64) {
        const int e = ids[p];
        if ((unsigned)e < (unsigned)E) atomicAdd(&my[e], 1);
    }
    __syncthreads();
    int count = 0;
    if (tid < E)
        for (int w = 0; w < 16; w++) {
            const int c = hist[w * E + tid];
            hist[w * E + tid] = count;
            count += c;
        }
    int total;
    const int start = block_exclusive_scan(count, wave_sums, &total);
    const int n_tiles = (count + kRowTile - 1) / kRowTile;
    int tiles_total;
    const int tile0 = block_exclusive_scan(n_tiles, wave_sums, &tiles_total);
    if (tid < E) {
        out[tid] = start;
        for (int w = 0; w < 16; w++) hist[w * E + tid] += start;
        int4* const tiles = reinterpret_cast<int4*>(out + lists_tiles_at(E));
        // an expert's rows in tiles of like size, whole blocks of 16 rows
        const int rows = n_tiles ? ((count + n_tiles - 1) / n_tiles + 15) / 16 * 16 : 0;
        for (int i = 0; i < n_tiles; i++) tiles[tile0 + i] = make_int4(tid, start + i * rows, max(0, min(rows, count - i * rows)), 0);
    }
    if (tid == 0) {
        out[E] = total;
        out[E + 1] = tiles_total;
    }
    __syncthreads();
    int32_t* const order = out + lists_order_at(P, E);
    for (int p0 = lo; p0 < hi; p0 += 64) {
        const int p = p0 + lane;
        const int e = p < hi ? ids[p] : -1;
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
        if (there) order[at] = p;
    }
}

// ---- few rows per expert ------------------------------------------------------------------------------------------
//
// Workgroup = NS strips of one expert; its waves share out K, every weight word is requested once, straight into registers, and multiplied
// by the expert's rows, 16 * RB of them at a time.  The waves' sums meet in LDS in wave order.
struct RowsArgs {
    const uint8_t* w;
    const void* x;
    const int32_t* ids;
    const int32_t* order;       // lists, or nullptr: the pairs of an expert are found among the (at most kMaxDirect) ids
    const int32_t* offsets;
    int P, xdiv, K, KT, strips, E;
    bool by_pair;               // blockIdx.y is a pair (the first of its expert does the work), else an expert
    void* y;
    int ydt, n_out;
};

constexpr int kMaxDirect = 512;

template <int XM, int RB>
struct XRegs {
    u32x4_t v[RB][XM == XF32 ? 8 : 4];
};

// eight fp32 values -> three bf16 operands that add up to them (24 significant bits: exact)
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

template <int BITS, int XM, int NS, bool PAIR, int RB, int D>
__global__ __launch_bounds__(512) void experts_rows_kernel(RowsArgs g)
{
    static_assert(NS * RB <= 4 && (!PAIR || NS % 2 == 0), "sums in LDS");
    constexpr int XS = XM == XF32 ? 4 : 2;
    __shared__ float4_t red[8][NS * RB][64];
    __shared__ int rows[kMaxDirect];
    __shared__ int n_rows, first_row;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x >> 6;
    const int slot = blockIdx.y;
    const int e = g.by_pair ? g.ids[slot] : slot;
    if ((unsigned)e >= (unsigned)g.E) return;
    const int s0 = blockIdx.x * NS;
    const int per = (g.KT + waves - 1) / waves;
    const int lo = min(wave * per, g.KT), hi = min(lo + per, g.KT);
    const WeightView wv = {g.w, 0, g.K, 0, g.KT, BITS};
    int64_t base[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) base[s] = ((int64_t)e * g.strips + min(s0 + s, g.strips - 1)) * g.KT;
    TileRegs<BITS> w[D][NS];
    auto request = [&](int d, int kt) {
#pragma unroll
        for (int s = 0; s < NS; s++) load_tile<BITS>(w[d][s], wv, base[s] + min(kt, g.KT - 1), lane);
    };
#pragma unroll
    for (int d = 0; d < D; d++) request(d, lo + d);

    // ---- the expert's rows
    const int32_t* list = rows;
    int n = 0;
    if (g.order) {
        const int a = g.offsets[e];
        n = g.offsets[e + 1] - a;
        list = g.order + a;
    } else {
        if (wave == 0) {
            int found = 0, first = g.P;
            for (int p0 = 0; p0 < g.P; p0 += 64) {
                const bool mine = p0 + lane < g.P && g.ids[p0 + lane] == e;
                const uint64_t who = __ballot(mine);
                if (mine) rows[found + __popcll(who & ((1ull << lane) - 1))] = p0 + lane;
                if (who && first == g.P) first = p0 + __builtin_ctzll(who);
                found += __popcll(who);
            }
            if (lane == 0) {
                n_rows = found;
                first_row = first;
            }
        }
        __syncthreads();
        n = n_rows;
        if (g.by_pair && first_row != slot) return;
    }
    if (n == 0) return;

    const int i16 = lane & 15, oct = lane >> 4;
    const uint32_t magic = XM == XF16 ? q4_magic_vgpr() : q4_magic_vgpr_bf16();
    const int G = g.K / kGroup;
    for (int r0 = 0; r0 < n; r0 += 16 * RB) {
        const char* row[RB];
#pragma unroll
        for (int rb = 0; rb < RB; rb++) row[rb] = static_cast<const char*>(g.x) + (int64_t)(list[min(r0 + rb * 16 + i16, n - 1)] / g.xdiv) * g.K * XS;
        float4_t acc[RB][NS];
#pragma unroll
        for (int rb = 0; rb < RB; rb++)
#pragma unroll
            for (int s = 0; s < NS; s++) acc[rb][s] = (float4_t){0.f, 0.f, 0.f, 0.f};
        if (r0)
#pragma unroll
            for (int d = 0; d < D; d++) request(d, lo + d);
        XRegs<XM, RB> x[2];
        auto request_x = [&](XRegs<XM, RB>& xr, int kt) {
#pragma unroll
            for (int rb = 0; rb < RB; rb++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    // (groups past the end of a row: its last pieces, cleared below)
                    const char* p = row[rb] + (int64_t)min(kt * kTileK + j * kGroup + oct * 8, g.K - 8) * XS;
                    if constexpr (XM == XF32) {
                        xr.v[rb][2 * j] = reinterpret_cast<const u32x4_t*>(p)[0];
                        xr.v[rb][2 * j + 1] = reinterpret_cast<const u32x4_t*>(p)[1];
                    } else {
                        xr.v[rb][j] = *reinterpret_cast<const u32x4_t*>(p);
                    }
                }
        };
        request_x(x[0], lo);
        auto step = [&](int kt, TileRegs<BITS> (&wt)[NS], const XRegs<XM, RB>& xr) {
            constexpr int PARTS = XM == XF32 ? 3 : 1;
            Frag16 b[NS][4];
#pragma unroll
            for (int s = 0; s < NS; s++) tile_operands<BITS, XM == XF16 ? XF16 : XBF16>(wt[s], magic, b[s]);
            Frag16 off;
            const uint32_t offw = BITS == 4 ? kBf16Neg136x2 : kBf16Neg128x2;
            off.u = (u32x4_t){offw, offw, offw, offw};
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    Frag16 a[3];
                    const bool past = kt * 4 + j >= G;
                    if constexpr (XM == XF32) {
                        u32x4_t p0 = xr.v[rb][2 * j], p1 = xr.v[rb][2 * j + 1];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            p0[i] = past ? 0u : p0[i];
                            p1[i] = past ? 0u : p1[i];
                        }
                        split_f32(p0, p1, a);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) a[0].u[i] = past ? 0u : xr.v[rb][j][i];
                    }
                    float4_t c = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (XM != XF16) {
#pragma unroll
                        for (int part = 0; part < PARTS; part++) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[part].b, off.b, c, 0, 0, 0);
                    }
#pragma unroll
                    for (int s = 0; s < NS; s++) {
                        float4_t d = c;
                        if constexpr (XM == XF16) {
                            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0].h, b[s][j].h, d, 0, 0, 0);
                        } else {
#pragma unroll
                            for (int part = 0; part < PARTS; part++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[part].b, b[s][j].b, d, 0, 0, 0);
                        }
                        const float sc = f16_bits_to_f32((j & 1) ? wt[s].s[j >> 1] >> 16 : wt[s].s[j >> 1] & 0xffffu);
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[rb][s][r] = fmaf(sc, d[r], acc[rb][s][r]);
                    }
                }
            }
        };
        for (int kt = lo; kt < hi; kt += D) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                if (kt + d < hi) {
                    request_x(x[(d + 1) & 1], kt + d + 1);
                    step(kt + d, w[d], x[d & 1]);
                    request(d, kt + d + D);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int rb = 0; rb < RB; rb++) red[wave][s * RB + rb][lane] = acc[rb][s];
        __syncthreads();
        constexpr int UNITS = NS * RB / (PAIR ? 2 : 1);
        for (int u = wave; u < UNITS; u += waves) {
            const int rb = u % RB, s = u / RB * (PAIR ? 2 : 1);
            float4_t v = red[0][s * RB + rb][lane], v2 = {0.f, 0.f, 0.f, 0.f};
            for (int k = 1; k < waves; k++) v += red[k][s * RB + rb][lane];
            if constexpr (PAIR) {
                v2 = red[0][(s + 1) * RB + rb][lane];
                for (int k = 1; k < waves; k++) v2 += red[k][(s + 1) * RB + rb][lane];
            }
            if (s0 + s >= g.strips) continue;
            const int col = (PAIR ? (s0 + s) / 2 : s0 + s) * 16 + i16;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = r0 + rb * 16 + oct * 4 + r;
                if (i < n) store_out(g.y, g.ydt, (int64_t)list[i] * g.n_out + col, PAIR ? silu_mul(v[r], v2[r]) : v[r]);
            }
        }
        __syncthreads();
    }
}

// ---- many rows per expert -----------------------------------------------------------------------------------------
//
// Workgroup = 8 waves side by side, a tile of up to 128 rows of one expert (16 * RB) x 16 strips; wave c has strips 2c, 2c + 1 (a gate and
// its up strip) against all rows.  Rows are gathered into LDS once per K tile, whole 128-byte lines of a row per eight lanes, pieces permuted
// so that the reads meet no bank conflicts; a wave's own weight tiles pass through LDS as well, only to be on their way without registers
// (global_load_lds).  One barrier per K tile; copies are counted by hand, they retire in order.
struct TilesArgs {
    const uint8_t* w;
    const void* x;
    const int32_t* lists;
    int64_t P;
    int xdiv, K, KT, strips, E, n_tiles;
    void* y;
    int ydt, n_out;
};

constexpr int kTilesLds = 156 * 1024;

template <int BITS, int RB>
struct TilesShape {
    static constexpr int XTILE = RB * 4096;
    static constexpr int WQ = 1024 * (BITS / 4);
    static constexpr int WTILE = 2 * WQ + 256;                   // a wave's
    static constexpr int STEP = XTILE + 8 * WTILE;
    static constexpr int FIT = kTilesLds / STEP;
    static constexpr int D = FIT > 6 ? 6 : FIT;                  // K tiles in LDS
    static constexpr int XC = (RB + 1) / 2;                      // copies per wave and K tile
    static constexpr int WC = 2 * (BITS / 4) + 1;
    static_assert(D >= 2, "LDS");
};

__device__ __forceinline__ void copy_lanes_to_lds(uint32_t lds_off, const void* base, uint32_t off, uint64_t lanes)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_mov_b64 exec, %3\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1" ::"s"(__builtin_amdgcn_readfirstlane(lds_off)), "v"(off), "s"(base), "s"(lanes));
}

template <int BITS, int XM, bool PAIR, int RB>
__device__ __forceinline__ void expert_tile(const TilesArgs& g, int e, const int32_t* list, int n, int strip0, uint8_t* smem)
{
    using S = TilesShape<BITS, RB>;
    constexpr int D = S::D;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i16 = lane & 15, oct = lane >> 4;
    const int G = g.K / kGroup;

    // X: block b = rows 16 * (b / 4) + 8 * (b / 2 % 2) .. + 8, half b % 2 of the K tile; copy c of wave w is block min(8 * c + w, ..)
    const int crow = lane >> 3, piece = (lane & 7) ^ crow;
    uint32_t xoff[S::XC];
    int xblk[S::XC];
#pragma unroll
    for (int c = 0; c < S::XC; c++) {
        xblk[c] = min(c * 8 + wave, RB * 4 - 2 + (wave & 1));
        xoff[c] = (uint32_t)(list[min((xblk[c] >> 1) * 8 + crow, n - 1)] / g.xdiv) * (uint32_t)(g.K * 2);
    }
    const int strip = min(strip0 + wave * 2, g.strips - 2 + (g.strips & 1)), second = min(strip + 1, g.strips - 1);
    const uint8_t* const wsrc = g.w + ((int64_t)e * g.strips + strip) * g.KT * kTileBytes<BITS>;
    const uint32_t wstep = (uint32_t)(second - strip) * (uint32_t)(g.KT * kTileBytes<BITS>);
    const uint32_t sc_off = (lane >= 8 ? wstep : 0u) + (uint32_t)(kTileQBytes<BITS> + (lane & 7) * 16);
    auto copy = [&](int kt_, int buf) {
        const int kt = min(kt_, g.KT - 1);
        const uint32_t at = (uint32_t)(buf * S::STEP);
#pragma unroll
        for (int c = 0; c < S::XC; c++) {
            // (groups past the end of a row: its last one; they are not multiplied)
            const int grp = min(kt * 4 + (wave & 1) * 2 + (piece >> 2), G - 1);
            copy_to_lds(at + xblk[c] * 1024, g.x, xoff[c] + (uint32_t)grp * 64u + (uint32_t)(piece & 3) * 16u);
        }
        const uint32_t src = (uint32_t)kt * (uint32_t)kTileBytes<BITS>;
        const uint32_t wat = at + S::XTILE + wave * S::WTILE;
#pragma unroll
        for (int q = 0; q < BITS / 4; q++) {
            copy_to_lds(wat + q * 1024, wsrc, src + q * 1024u + (uint32_t)lane * 16u);
            copy_to_lds(wat + S::WQ + q * 1024, wsrc, wstep + src + q * 1024u + (uint32_t)lane * 16u);
        }
        copy_lanes_to_lds(wat + 2 * S::WQ, wsrc, sc_off + src, 0xffffull);
    };
#pragma unroll
    for (int d = 0; d < D - 1; d++) copy(d, d);

    float4_t acc[RB][2];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int s = 0; s < 2; s++) acc[i][s] = (float4_t){0.f, 0.f, 0.f, 0.f};
    const uint32_t magic = XM == XF16 ? q4_magic_vgpr() : q4_magic_vgpr_bf16();
    const uint32_t raw = (uint32_t)((i16 >> 3) * 2048 + (i16 & 7) * 128 + ((oct ^ (i16 & 7)) * 16));
    Frag16 off;
    const uint32_t offw = BITS == 4 ? kBf16Neg136x2 : kBf16Neg128x2;
    off.u = (u32x4_t){offw, offw, offw, offw};

    auto multiply = [&](const uint8_t* at, int groups) {
        const uint8_t* const wp = at + S::XTILE + wave * S::WTILE;
        TileRegs<BITS> w[2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int q = 0; q < BITS / 4; q++) w[s].q[q] = *reinterpret_cast<const u32x4_t*>(wp + s * S::WQ + q * 1024 + lane * 16);
            w[s].s = *reinterpret_cast<const u32x2_t*>(wp + 2 * S::WQ + s * 128 + i16 * 8);
        }
        Frag16 b[2][4];
        tile_operands<BITS, XM>(w[0], magic, b[0]);
        tile_operands<BITS, XM>(w[1], magic, b[1]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j >= groups) break;
            float sc[2];
#pragma unroll
            for (int s = 0; s < 2; s++) sc[s] = f16_bits_to_f32((j & 1) ? w[s].s[j >> 1] >> 16 : w[s].s[j >> 1] & 0xffffu);
#pragma unroll
            for (int i = 0; i < RB; i++) {
                Frag16 a;
                a.u = *reinterpret_cast<const u32x4_t*>(at + i * 4096 + (j >> 1) * 1024 + ((j & 1) ? raw ^ 64u : raw));
                float4_t c = {0.f, 0.f, 0.f, 0.f};
                if constexpr (XM == XBF16) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, off.b, c, 0, 0, 0);
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const float4_t d = XM == XBF16 ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, b[s][j].b, c, 0, 0, 0)
                                                   : __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b[s][j].h, c, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][s][r] = fmaf(sc[s], d[r], acc[i][s][r]);
                }
            }
        }
    };
    int buf = 0;
    const int whole = G / 4;
    for (int kt = 0; kt < g.KT; kt++) {
        // this K tile's copies are there - mine, and behind the barrier everybody's - and nobody reads the last one's place any more
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((D - 2) * (S::XC + S::WC)) : "memory");
        copy(kt + D - 1, buf == 0 ? D - 1 : buf - 1);
        if (kt < whole) multiply(smem + buf * S::STEP, 4);
        else multiply(smem + buf * S::STEP, G - whole * 4);
        buf = buf + 1 == D ? 0 : buf + 1;
    }
    // (no copy may land in LDS that another workgroup has by then)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const bool there = strip0 + wave * 2 < g.strips, both = strip0 + wave * 2 + 1 < g.strips;
    if (!there) return;
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int m = i * 16 + oct * 4 + r;
            if (m >= n) continue;
            const int64_t at = (int64_t)list[m] * g.n_out;
            if constexpr (PAIR) {
                store_out(g.y, g.ydt, at + (strip0 / 2 + wave) * 16 + i16, silu_mul(acc[i][0][r], acc[i][1][r]));
            } else {
                store_out(g.y, g.ydt, at + (strip0 + wave * 2) * 16 + i16, acc[i][0][r]);
                if (both) store_out(g.y, g.ydt, at + (strip0 + wave * 2 + 1) * 16 + i16, acc[i][1][r]);
            }
        }
}

template <int BITS, int XM, bool PAIR>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void experts_tiles_kernel(TilesArgs g)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int items = g.lists[g.E + 1] * g.n_tiles;
    const int per_xcd = (items + 7) >> 3;
    const int item = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per_xcd || item >= items) return;
    const int tile_m = __builtin_amdgcn_readfirstlane(item / g.n_tiles), tile_n = item - tile_m * g.n_tiles;
    const int4 t = reinterpret_cast<const int4*>(g.lists + lists_tiles_at(g.E))[tile_m];
    const int e = __builtin_amdgcn_readfirstlane(t.x), n = __builtin_amdgcn_readfirstlane(t.z);
    const int32_t* const list = g.lists + lists_order_at(g.P, g.E) + __builtin_amdgcn_readfirstlane(t.y);
    if (n <= 0) return;
    if (n <= 16) expert_tile<BITS, XM, PAIR, 1>(g, e, list, n, tile_n * 16, smem);
    else if (n <= 32) expert_tile<BITS, XM, PAIR, 2>(g, e, list, n, tile_n * 16, smem);
    else if (n <= 64) expert_tile<BITS, XM, PAIR, 4>(g, e, list, n, tile_n * 16, smem);
    else if (n <= 96) expert_tile<BITS, XM, PAIR, 6>(g, e, list, n, tile_n * 16, smem);
    else expert_tile<BITS, XM, PAIR, 8>(g, e, list, n, tile_n * 16, smem);
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

template <int BITS, int XM, bool PAIR>
void launch_rows(const RowsArgs& g, int slots, int rows_hint, int num_cus, hipStream_t st)
{
    const int waves = std::max(1, std::min(8, g.KT));
    auto go = [&](auto kernel, int ns) { kernel<<<dim3((g.strips + ns - 1) / ns, slots), dim3(waves * 64), 0, st>>>(g); };
    if constexpr (XM == XF32) {
        go(experts_rows_kernel<BITS, XM, PAIR ? 2 : 1, PAIR, 1, 2>, PAIR ? 2 : 1);
    } else {
        if (rows_hint > 16) go(experts_rows_kernel<BITS, XM, 2, PAIR, 2, 2>, 2);
        else go(experts_rows_kernel<BITS, XM, PAIR ? 2 : 1, PAIR, 1, 4>, PAIR ? 2 : 1);
    }
}

template <int BITS, int XM, bool PAIR>
void launch_tiles(const TilesArgs& g, hipStream_t st)
{
    (void)LdsRequest<&experts_tiles_kernel<BITS, XM, PAIR>, kTilesLds>::registered;
    const int64_t items = lists_tiles_max(g.P, g.E) * g.n_tiles;
    experts_tiles_kernel<BITS, XM, PAIR><<<dim3((unsigned)((items + 7) / 8 * 8)), dim3(512), kTilesLds, st>>>(g);
}

}  // namespace

size_t experts_lists_bytes(int64_t P, int E) { return ((size_t)(lists_order_at(P, E) + P) * 4 + 255) / 256 * 256; }

hipError_t launch_experts(const WeightView& w, int E, bool pair, const void* x, int xdt, int64_t P, int xdiv, const int32_t* ids, void* y, int ydt,
                          int num_cus, void* lists, hipStream_t st)
{
    const int strips = w.NT / E, n_out = strips * 16 / (pair ? 2 : 1);
    const int64_t met = std::min<int64_t>(P, E);
    const bool many = xdt != kF32 && P >= 16 * met;
    int32_t* const L = static_cast<int32_t*>(lists);
    if (many || P > kMaxDirect) {
        int bits = 0;
        while ((1 << bits) < E) bits++;
        const int lds = (16 * E + 16) * 4;
        (void)LdsRequest<&lists_kernel, (16 * 1024 + 16) * 4>::registered;
        lists_kernel<<<1, 1024, lds, st>>>(ids, (int)P, E, bits, L);
    }
    if (many) {
        const TilesArgs g = {w.base, x, L, P, xdiv, w.K, w.KT, strips, E, (strips + 15) / 16, y, ydt, n_out};
        auto go = [&](auto bits, auto xm) {
            if (pair) launch_tiles<decltype(bits)::value, decltype(xm)::value, true>(g, st);
            else launch_tiles<decltype(bits)::value, decltype(xm)::value, false>(g, st);
        };
        using std::integral_constant;
        if (w.bits == 4) xdt == kF16 ? go(integral_constant<int, 4>{}, integral_constant<int, XF16>{}) : go(integral_constant<int, 4>{}, integral_constant<int, XBF16>{});
        else xdt == kF16 ? go(integral_constant<int, 8>{}, integral_constant<int, XF16>{}) : go(integral_constant<int, 8>{}, integral_constant<int, XBF16>{});
        return hipGetLastError();
    }
    RowsArgs g = {w.base, x, ids, nullptr, nullptr, (int)P, xdiv, w.K, w.KT, strips, E, P <= E, y, ydt, n_out};
    if (P > kMaxDirect) {
        g.offsets = L;
        g.order = L + lists_order_at(P, E);
        g.by_pair = false;
    }
    const int slots = g.by_pair ? (int)P : E, rows_hint = (int)((P + met - 1) / met);
    auto go = [&](auto bits, auto xm) {
        if (pair) launch_rows<decltype(bits)::value, decltype(xm)::value, true>(g, slots, rows_hint, num_cus, st);
        else launch_rows<decltype(bits)::value, decltype(xm)::value, false>(g, slots, rows_hint, num_cus, st);
    };
    using std::integral_constant;
    auto with = [&](auto xm) { w.bits == 4 ? go(integral_constant<int, 4>{}, xm) : go(integral_constant<int, 8>{}, xm); };
    if (xdt == kF16) with(integral_constant<int, XF16>{});
    else if (xdt == kBF16) with(integral_constant<int, XBF16>{});
    else with(integral_constant<int, XF32>{});
    return hipGetLastError();
}

hipError_t launch_experts_sum(const float* z, const int32_t* ids, const float* weights, const void* residual, int64_t T, int top_k, int E, int N, void* y,
                              int ydt, hipStream_t st)
{
    experts_sum_kernel<<<dim3((N / 4 + 255) / 256, (unsigned)T), 256, 0, st>>>(z, ids, weights, residual, (int)T, top_k, E, N, y, ydt);
    return hipGetLastError();
}

}  // namespace cybq
