// gnk_grouped.h -- MFMA products of 8-bit operands grouped by expert: rows sorted by group, group sizes known on the GPU only.
//
//   rows :  C[t, n]    = (f32(sum_k A[t, k] B[e(t), k, n]) * row_scale[t])    * col_scale[e(t), n]     (forward, gradient of the input)
//   depth:  C[e, m, n] = (f32(sum_{t in e} A[m, t] B[t, n]) * row_scale[e, m]) * col_scale[e, n]       (gradients of the weights)
//
// Group e holds rows ends[e - 1] .. ends[e] - 1 (ends[-1] = 0); rows behind the last end belong to no group and come out as zeros.
// The host knows neither the sizes nor the number of tiles: it launches the most workgroups the sizes could need (sum of ceil(T_e / BM)
// <= T / BM + E, one more for the rows behind), every workgroup scans the ends with one wave-wide prefix sum (64 groups per step) to find
// its tile, and the surplus leaves at once.  An end below an earlier one counts as that one, an end beyond T as T: the groups are disjoint and
// in order whatever `ends` holds, so that no value of it reaches outside the operands, the tile counts above or the workspaces.  A group's tile is then an ordinary tile of gnk_gemm_kernel.h / gnk_gemm_w4.h: same LDS images, fragments and epilogue.
#pragma once
#include <math.h>

#include "gnk_gemm_dispatch.h"
#include "gnk_gemm_w4.h"
#include "gnk_gemm_w4_more_asm.inc"

struct GroupedParams {
    GemmParams g;            // A, B, C, scales of the whole call; N; rows: K; depth: M
    const int *ends;
    int64_t T, E;
    int64_t b_group;         // rows: bytes from one group's B to the next
    int64_t ext_a, ext_b;    // depth: staged extents of A (>= M) and B (>= N); rows: ext_b (>= N) -- multiples of 16 for M/N-major operands
    int out_bytes, scale_bytes;
    int splits;              // depth: parts that a group's contraction is cut into (1: none); their sums go to `slab`, part by part
    void *slab;
    int64_t slab_bytes;
    int long_rows;           // depth: groups of more rows are left to a launch of their own (0: none are)
    int pieces;              // depth: this is that launch, over at most so many pieces of them; their sums go to `slab`, piece by piece
};

typedef int (*gnk_grouped_launcher)(bool depth, bool b_kmajor, const GroupedParams &p, hipStream_t st);
#define GNK_DECLARE_GROUPED(NAME) int NAME(bool depth, bool b_kmajor, const GroupedParams &p, hipStream_t st)
GNK_DECLARE_GROUPED(gnk_grouped_i8);
GNK_DECLARE_GROUPED(gnk_grouped_f8_00);
GNK_DECLARE_GROUPED(gnk_grouped_f8_01);
GNK_DECLARE_GROUPED(gnk_grouped_f8_10);
GNK_DECLARE_GROUPED(gnk_grouped_f8_11);

namespace gnk_grouped {

using namespace gnk_gemm;

// One tile: rows [lo, hi) of group e (e == E: the rows behind the last group), row tile tm of that group, column tile tn.
struct Tile {
    int e, tm, tn;
    int part;                // depth: which part of the group's rows [lo, hi) are
    int64_t lo, hi;
    bool work;               // false: a surplus workgroup
};

__device__ __forceinline__ int64_t clamp_end(int v, int64_t T) { return v < 0 ? 0 : (v < T ? v : T); }

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// inclusive prefix sum over the wave: row shifts, then the two row broadcasts (no LDS round trips)
__device__ __forceinline__ int wave_prefix(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // lane 15 of a row into the next row: rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);      // lane 31 into rows 2 and 3
    return v;
}

// inclusive running maximum over the wave, of values >= 0
__device__ __forceinline__ int wave_running_max(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
    return v;
}

// Rows [lo, hi) of group g0 + lane; group E takes the rows behind the last end, groups beyond it none.  (T < 2^31.)  ends == NULL: equal groups.
// `before`: the largest end in front of group g0, 0 for g0 = 0; this call takes it on to g0 + 64.
__device__ __forceinline__ void lane_group(const int *ends, int64_t E, int64_t T, int64_t g0, int lane, int &before, int &lo, int &hi) {
    const int64_t e = g0 + lane;
    if (!ends) {
        const int each = E > 0 ? (int)((unsigned)T / (unsigned)E) : 0;
        lo = e <= E ? (int)e * each : 0;
        hi = e < E ? lo + each : (e == E ? (int)T : lo);
        return;
    }
    lo = wave_running_max(max(before, e > 0 && e <= E ? (int)clamp_end(ends[e - 1], T) : 0));
    hi = max(lo, e < E ? (int)clamp_end(ends[e], T) : (e == E ? (int)T : 0));
    before = __builtin_amdgcn_readlane(lo, 63);
}

// Rows [lo, hi) of group e <= E alone, the same for the whole wave
__device__ __forceinline__ void one_group(const int *ends, int64_t E, int64_t T, int64_t e, int lane, int &lo, int &hi) {
    if (!ends) {
        const int each = E > 0 ? (int)((unsigned)T / (unsigned)E) : 0;
        lo = (int)e * each;
        hi = e < E ? lo + each : (int)T;
        return;
    }
    const int own = e < E ? (int)clamp_end(ends[e], T) : (int)T;
    int most = 0;
    for (int64_t i = lane; i < e; i += 64) most = max(most, (int)clamp_end(ends[i], T));
    lo = __builtin_amdgcn_readlane(wave_running_max(most), 63);
    hi = max(lo, uniform(own));
}

// Every group (and the rows behind the last one) is cut into pieces of 1 << sh rows (sh = -192: of 192 rows), numbered in group order.
constexpr int ROWS_192 = -192;
__device__ __forceinline__ int pieces_of(int rows, int sh) {
    if (sh == ROWS_192) return (int)(((unsigned)rows + 191u) / 192u);
    return (int)(((unsigned)rows + ((1u << sh) - 1)) >> sh);
}

__device__ __forceinline__ int count_pieces(const int *ends, int64_t E, int64_t T, int lane, int sh) {
    int total = 0, end = 0;
    for (int64_t g0 = 0; g0 <= E; g0 += 64) {
        int lo, hi;
        lane_group(ends, E, T, g0, lane, end, lo, hi);
        total += __builtin_amdgcn_readlane(wave_prefix(pieces_of(hi - lo, sh)), 63);
    }
    return total;
}

// Piece number `want`: its group e (E: rows of no group; -1: there are fewer pieces), its number within the group, the group's rows, and the
// number of pieces of 1 << sh2 rows in the groups in front of it.
// int8: 128 * 128 * 131071 is the largest sum of products that is sure to fit an accumulator's 32 bits.  The host knows the rows of all groups together, not of
// one: beyond LONG_ROWS of them (whole steps of every loop) a group that has more is cut into pieces of LONG_ROWS, whose sums are added in 64 bits.
constexpr int64_t INT8_TERMS = 131071;
constexpr int LONG_ROWS = 511 * 256;
static_assert(LONG_ROWS <= INT8_TERMS, "a piece's sums fit 32 bits");

struct Piece { int e, idx, lo, hi, first2; };
__device__ __forceinline__ Piece find_piece(const int *ends, int64_t E, int64_t T, int lane, int sh, int want, int sh2) {
    int before = 0, before2 = 0, end = 0;
    for (int64_t g0 = 0; g0 <= E; g0 += 64) {
        int l, h;
        lane_group(ends, E, T, g0, lane, end, l, h);
        const int n = pieces_of(h - l, sh), n2 = pieces_of(h - l, sh2);
        const int incl = wave_prefix(n) + before, incl2 = wave_prefix(n2) + before2;
        const unsigned long long hit = __ballot(incl > want);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            return {(int)g0 + src, want - __builtin_amdgcn_readlane(incl - n, src), __builtin_amdgcn_readlane(l, src), __builtin_amdgcn_readlane(h, src),
                    __builtin_amdgcn_readlane(incl2 - n2, src)};
        }
        before = __builtin_amdgcn_readlane(incl, 63);
        before2 = __builtin_amdgcn_readlane(incl2, 63);
    }
    return {-1, 0, 0, 0, 0};
}

__device__ __forceinline__ int long_pieces_of(int rows) { return rows > LONG_ROWS ? (int)(((unsigned)rows + (LONG_ROWS - 1u)) / (unsigned)LONG_ROWS) : 0; }

// Piece number `want` of the groups of more than LONG_ROWS rows, as find_piece has it (first2: the number of the group's first piece)
__device__ __forceinline__ Piece find_long_piece(const int *ends, int64_t E, int64_t T, int lane, int want) {
    int before = 0, end = 0;
    for (int64_t g0 = 0; g0 < E; g0 += 64) {
        int l, h;
        lane_group(ends, E, T, g0, lane, end, l, h);
        const int n = g0 + lane < E ? long_pieces_of(h - l) : 0, incl = wave_prefix(n) + before;
        const unsigned long long hit = __ballot(incl > want);
        if (hit) {
            const int src = __builtin_ctzll(hit), first = __builtin_amdgcn_readlane(incl - n, src);
            return {(int)g0 + src, want - first, __builtin_amdgcn_readlane(l, src), __builtin_amdgcn_readlane(h, src), first};
        }
        before = __builtin_amdgcn_readlane(incl, 63);
    }
    return {-1, 0, 0, 0, 0};
}

// rows form: tiles are counted on the device, then given to the XCDs in contiguous runs and walked in strips as tile_of_block does
template <int BM>
__device__ __forceinline__ Tile rows_tile(const GroupedParams &p, int grid_n, int lane) {
    constexpr int SH = BM == 256 ? 8 : BM == 192 ? ROWS_192 : BM == 128 ? 7 : 6;
    static_assert(BM == 256 || BM == 192 || BM == 128 || BM == 64, "row tiles");
    Tile t;
    if (p.E < 64) {                          // all groups in one wave: one load and one prefix sum give the count and the place
        int l, h, end = 0;
        lane_group(p.ends, p.E, p.T, 0, lane, end, l, h);
        const int n = pieces_of(h - l, SH), incl = wave_prefix(n), grid_m = __builtin_amdgcn_readlane(incl, 63);
        t.work = (int64_t)blockIdx.x < (int64_t)grid_m * grid_n;
        if (!t.work) return t;
        int tm;
        tile_of_block(grid_m, grid_n, tm, t.tn);
        const int src = __builtin_ctzll(__ballot(incl > tm));
        t.e = src;
        t.tm = tm - __builtin_amdgcn_readlane(incl - n, src);
        t.lo = __builtin_amdgcn_readlane(l, src);
        t.hi = __builtin_amdgcn_readlane(h, src);
        return t;
    }
    const int grid_m = count_pieces(p.ends, p.E, p.T, lane, SH);
    t.work = (int64_t)blockIdx.x < (int64_t)grid_m * grid_n;
    if (!t.work) return t;
    int tm, tn;
    tile_of_block(grid_m, grid_n, tm, tn);
    const Piece pc = find_piece(p.ends, p.E, p.T, lane, SH, tm, SH);
    t.e = pc.e; t.tm = pc.idx; t.lo = pc.lo; t.hi = pc.hi;
    t.tn = tn;
    return t;
}

// STEP: rows per step of the kernel's loop; a part is a whole number of them
template <int STEP> __device__ __forceinline__ Tile depth_tile(const GroupedParams &p, int grid_m, int grid_n, int lane) {
    Tile t;
    const int per = grid_m * grid_n * p.splits;
    int tm, tn;
    // groups in order; within one, the strips of tile_of_block without its XCD split (a group's operands fit every L2 badly anyway).  The parts (a power of
    // two of them) change fastest, so that the tiles that read the same rows run on the same XCDs.
    const int wg = (int)blockIdx.x;
    t.e = wg / per;
    int in = wg - t.e * per;
    t.part = in % p.splits;
    in /= p.splits;
    constexpr int GROUP_M = 4;
    const int width = GROUP_M * grid_n, strip = in / width, first = strip * GROUP_M, gsz = min(grid_m - first, GROUP_M), r = in - strip * width;
    tm = first + r % gsz;
    tn = r / gsz;
    t.tm = tm; t.tn = tn;
    if (p.pieces) {                          // (one part each: t.e counted the pieces)
        t.part = t.e;
        const Piece pc = find_long_piece(p.ends, p.E, p.T, lane, t.part);
        t.e = pc.e;
        t.work = pc.e >= 0;
        t.lo = pc.lo + (int64_t)pc.idx * LONG_ROWS;
        t.hi = t.lo + LONG_ROWS < pc.hi ? t.lo + LONG_ROWS : pc.hi;
        return t;
    }
    int lo, hi;
    one_group(p.ends, p.E, p.T, t.e, lane, lo, hi);
    t.lo = lo; t.hi = hi;
    if (p.splits > 1) {
        const int64_t steps = (t.hi - t.lo + STEP - 1) / STEP, each = (steps + p.splits - 1) / p.splits * STEP;
        t.lo = t.lo + t.part * each < t.hi ? t.lo + t.part * each : t.hi;
        t.hi = t.lo + each < t.hi ? t.lo + each : t.hi;
    }
    t.work = !p.long_rows || hi - lo <= p.long_rows;
    return t;
}

// The ordinary product of one tile: pointers and extents of its group.  ext_a / ext_b: staged extents (rows of A, columns of B).
template <bool DEPTH>
__device__ __forceinline__ GemmParams tile_params(const GroupedParams &p, const Tile &t, int64_t &ext_a, int64_t &ext_b) {
    GemmParams g = p.g;
    const int64_t rows = t.hi - t.lo;
    if constexpr (DEPTH) {
        g.K = rows;
        g.A += t.lo * g.lda;
        g.B += t.lo * g.ldb;
        g.C = (char *)g.C + (p.pieces ? (int64_t)t.part : (int64_t)t.part * p.E + t.e) * g.M * g.N * p.out_bytes;
        g.s0 = (const char *)g.s0 + (int64_t)t.e * g.M * p.scale_bytes;
        ext_a = p.ext_a;
    } else {
        g.M = rows;
        g.A += t.lo * g.lda;
        g.B += (int64_t)t.e * p.b_group;
        g.C = (char *)g.C + t.lo * g.N * p.out_bytes;
        g.s0 = (const char *)g.s0 + t.lo * p.scale_bytes;
        ext_a = rows;
    }
    g.s1 = (const char *)g.s1 + (g.col_scalar ? (int64_t)t.e : (int64_t)t.e * g.N) * p.scale_bytes;
    ext_b = p.ext_b;
    return g;
}

// zeros into rows [m0, min(m0 + BM, rows)) x columns [n0, min(n0 + BN, N)) of a row-major (rows, N) output
template <int BM, int BN, int NT>
__device__ __forceinline__ void zero_tile(char *C, int64_t rows, int64_t N, int64_t m0, int64_t n0, int out_bytes) {
    const int64_t m1 = m0 + BM < rows ? m0 + BM : rows, n1 = n0 + BN < N ? n0 + BN : N;
    const int64_t halves = (n1 - n0) * (out_bytes >> 1);          // outputs are 2 or 4 bytes wide
    for (int64_t m = m0; m < m1; ++m) {
        unsigned short *dst = (unsigned short *)(C + (m * N + n0) * out_bytes);
        for (int64_t i = threadIdx.x; i < halves; i += NT) dst[i] = 0;
    }
}

// ------------------------------------------------------------------------------ two-buffer kernel (any K, any group size)
// The loop of gemm_kernel (row / column epilogue) on one group's tile.  128 x 128 over four waves: 64 KiB of LDS and at most 256
// registers, two workgroups per CU.  Bound by a tile's fixed cost (~6 us: first loads, epilogue) beside 1 us per 128 k, and by whole rounds of tiles:
// 4099 rows over 16 experts, 1024 -> 4096, e4m3: 30-33 us, 3.3 TB/s of its 105 MB (21 us at a copy's rate), 1.1 PFLOP/s.
template <class Cfg, bool DEPTH>
__global__ void __launch_bounds__(Cfg::NT) __attribute__((amdgpu_waves_per_eu(Cfg::NT == 256 ? 2 : 1))) two_buffer_kernel(const GroupedParams gp) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int MT = Cfg::MT, NTL = Cfg::NTL;
    typedef typename AccT<Cfg::OP>::type acc_t;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
    const Tile tile = DEPTH ? depth_tile<GNK_BK>(gp, gp.g.grid_m, gp.g.grid_n, lane) : rows_tile<Cfg::BM>(gp, gp.g.grid_n, lane);
    if (!tile.work) return;
    const int64_t m0 = (int64_t)tile.tm * Cfg::BM, n0 = (int64_t)tile.tn * Cfg::BN;
    if (!DEPTH && tile.e == gp.E) {      // rows of no group
        zero_tile<Cfg::BM, Cfg::BN, Cfg::NT>((char *)gp.g.C + tile.lo * gp.g.N * gp.out_bytes, tile.hi - tile.lo, gp.g.N, m0, n0, gp.out_bytes);
        return;
    }
    int64_t ext_a, ext_b;
    const GemmParams p = tile_params<DEPTH>(gp, tile, ext_a, ext_b);

    char *const As0 = smem;
    char *const Bs0 = smem + 2 * Cfg::A_BYTES;
    ScalePrefetch<Cfg::BM, Cfg::BN, Cfg::NT, Cfg::EPI> spf;
    spf.issue(p, m0, n0);
    Stager<Cfg::A_KMAJOR, Cfg::BM, Cfg::NW> sa;
    Stager<Cfg::B_KMAJOR, Cfg::BN, Cfg::NW> sb;
    sa.init(p.A, p.lda, m0, ext_a, wave, lane);
    sb.init(p.B, p.ldb, n0, ext_b, wave, lane);
    acc_t acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = (acc_t){0, 0, 0, 0};

    const int nk = (int)((p.K + GNK_BK - 1) / GNK_BK), ktail = (int)(p.K % GNK_BK);
    if (nk > 0) {
        if (nk == 1 && ktail) {
            sa.issue_tail(As0, p.lda, m0, ext_a, wave, lane, ktail);
            sb.issue_tail(Bs0, p.ldb, n0, ext_b, wave, lane, ktail);
        } else {
            sa.issue(As0, wave);
            sb.issue(Bs0, wave);
        }
    }
    for (int t = 0; t < nk; ++t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const int cur = t & 1;
        if (ktail && t + 1 == nk) {
            zero_tail<Cfg::A_KMAJOR, Cfg::BM, Cfg::NT>(As0 + cur * Cfg::A_BYTES, ktail);
            zero_tail<Cfg::B_KMAJOR, Cfg::BN, Cfg::NT>(Bs0 + cur * Cfg::B_BYTES, ktail);
            __syncthreads();
        }
        if (t + 1 < nk) {
            if (ktail && t + 2 == nk) {
                sa.issue_tail(As0 + (cur ^ 1) * Cfg::A_BYTES, p.lda, m0, ext_a, wave, lane, ktail);
                sb.issue_tail(Bs0 + (cur ^ 1) * Cfg::B_BYTES, p.ldb, n0, ext_b, wave, lane, ktail);
            } else {
                sa.issue(As0 + (cur ^ 1) * Cfg::A_BYTES, wave);
                sb.issue(Bs0 + (cur ^ 1) * Cfg::B_BYTES, wave);
            }
        }
        compute_step<Cfg, false>(As0 + cur * Cfg::A_BYTES, Bs0 + cur * Cfg::B_BYTES, acc, wm, wn, lane);
    }
    spf.park(p, smem + Cfg::LDS_BYTES);
    __syncthreads();
    run_epilogue<Cfg>(p, acc, nullptr, smem, wave, lane, m0 + wm * Cfg::WTM, n0 + wn * Cfg::WTN, (const float *)(smem + Cfg::LDS_BYTES),
                      wm * Cfg::WTM, wn * Cfg::WTN);
}

// ------------------------------------------------------------------------------ 64 x 64, ring of four stages (few rows: latency and the weights' bytes)
// Few tiles leave one or two workgroups on a CU, and a group of a few rows is bound by the bytes of its weights: what counts is how much is in
// flight.  Three 128-k stages of 16 KiB are, behind the one being read (2 workgroups per CU: ~50 KiB of weights in flight per CU), one barrier per
// stage.  Stage t lands before the barrier of step t (vmcnt leaves the pieces of t + 1 and t + 2 in flight); the buffer of stage t - 1, which every
// wave has read by then, takes stage t + 3 behind it.  Towards the end nothing is left to issue and the wait is for everything.
// 16 rows over 8 experts, 1024 -> 4096, int8: 7.9-8.4 us a call for 30 MB of weights, 3.5 TB/s (5.9 us at a copy's rate; the rest is the launch and the
// first loads); depth form, 1021 rows over 8 experts to 512 x 256: 5 us.
// KG = 2 (at most one workgroup per CU): a second set of four waves with a ring of its own takes every other step; the two halves are added in LDS.
// 16 rows over 4 experts, 4096 -> 1024: 17.7 -> 11.6 us with B K-major, 23.2 -> 18.2 N-major (rows of 64 bytes are half lines); 5632 -> 2048, one row: 18.2 -> 15.0.
template <class Cfg, bool DEPTH, int KG>
__global__ void __launch_bounds__(Cfg::NT * KG) __attribute__((amdgpu_waves_per_eu(2))) ring_kernel(const GroupedParams gp) {
    extern __shared__ __attribute__((aligned(16))) char smem_all[];
    constexpr int MT = Cfg::MT, NTL = Cfg::NTL, NST = 4, STAGE = Cfg::A_BYTES + Cfg::B_BYTES, RING = NST * STAGE, NT = Cfg::NT * KG;
    constexpr int PIECES = (Cfg::BM + Cfg::BN) / 8 / Cfg::NW;      // LDS-DMA instructions per wave and stage
    static_assert(KG == 1 || KG == 2, "one or two sets of waves");
    typedef typename AccT<Cfg::OP>::type acc_t;
    const int lane = threadIdx.x & 63;
    const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave_all / Cfg::NW, wave = wave_all % Cfg::NW;
    const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
    char *const smem = smem_all + kg * RING;
    const Tile tile = DEPTH ? depth_tile<GNK_BK>(gp, gp.g.grid_m, gp.g.grid_n, lane) : rows_tile<Cfg::BM>(gp, gp.g.grid_n, lane);
    if (!tile.work) return;
    const int64_t m0 = (int64_t)tile.tm * Cfg::BM, n0 = (int64_t)tile.tn * Cfg::BN;
    if (!DEPTH && tile.e == gp.E) {
        zero_tile<Cfg::BM, Cfg::BN, NT>((char *)gp.g.C + tile.lo * gp.g.N * gp.out_bytes, tile.hi - tile.lo, gp.g.N, m0, n0, gp.out_bytes);
        return;
    }
    int64_t ext_a, ext_b;
    const GemmParams p = tile_params<DEPTH>(gp, tile, ext_a, ext_b);
    ScalePrefetch<Cfg::BM, Cfg::BN, Cfg::NT, EPI_ROWCOL> spf;
    spf.issue(p, m0, n0);
    Stager<Cfg::A_KMAJOR, Cfg::BM, Cfg::NW> sa;
    Stager<Cfg::B_KMAJOR, Cfg::BN, Cfg::NW> sb;
    sa.init(p.A, p.lda, m0, ext_a, wave, lane);
    sb.init(p.B, p.ldb, n0, ext_b, wave, lane);
    if constexpr (KG > 1) {
        sa.base += kg * sa.step;
        sb.base += kg * sb.step;
        sa.step *= KG;
        sb.step *= KG;
    }
    acc_t acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = (acc_t){0, 0, 0, 0};
    const int nk_all = (int)((p.K + GNK_BK - 1) / GNK_BK), ktail = (int)(p.K % GNK_BK), last = nk_all - 1;
    const int nk = (nk_all + KG - 1 - kg) / KG, nk_most = (nk_all + KG - 1) / KG;      // this set's steps kg, kg + KG, ...
    auto fetch = [&](int t) {
        char *const As = smem + (t % NST) * STAGE, *const Bs = As + Cfg::A_BYTES;
        if (ktail && t * KG + kg == last) {
            sa.issue_tail(As, p.lda, m0, ext_a, wave, lane, ktail);
            sb.issue_tail(Bs, p.ldb, n0, ext_b, wave, lane, ktail);
        } else {
            sa.issue(As, wave);
            sb.issue(Bs, wave);
        }
    };
    for (int t = 0; t < NST - 1 && t < nk; ++t) fetch(t);
    for (int t = 0; t < nk_most; ++t) {
        static_assert(2 * PIECES <= 63, "vmcnt holds 6 bits");
        if (t + NST - 2 < nk) asm volatile("s_waitcnt vmcnt(%0)" : : "i"((NST - 2) * PIECES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (ktail && t == last / KG) {                                // every thread clears its share of the tail, whichever set owns it
            char *const Az = smem_all + (last % KG) * RING + (t % NST) * STAGE, *const Bz = Az + Cfg::A_BYTES;
            zero_tail<Cfg::A_KMAJOR, Cfg::BM, NT>(Az, ktail);
            zero_tail<Cfg::B_KMAJOR, Cfg::BN, NT>(Bz, ktail);
            __syncthreads();
        }
        if (t + NST - 1 < nk) fetch(t + NST - 1);
        char *const As = smem + (t % NST) * STAGE, *const Bs = As + Cfg::A_BYTES;
        if (t < nk) compute_step<Cfg, false>(As, Bs, acc, wm, wn, lane);
    }
    float *const lsc = (float *)(smem_all + KG * RING);
    spf.park(p, (char *)lsc);
    __syncthreads();
    if constexpr (KG > 1) {
        // the second set's sums through its own ring, free now
        char *const sums = smem_all + RING;
        if (kg == 1)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NTL; ++j) *(GNK_LDS acc_t *)(GNK_LDS char *)(sums + 16 * (((wave * MT + i) * NTL + j) * 64 + lane)) = acc[i][j];
        __syncthreads();
        if (kg == 1) return;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] += *(const GNK_LDS acc_t *)(const GNK_LDS char *)(sums + 16 * (((wave * MT + i) * NTL + j) * 64 + lane));
    }
    run_epilogue<Cfg>(p, acc, nullptr, smem, wave, lane, m0 + wm * Cfg::WTM, n0 + wn * Cfg::WTN, lsc, wm * Cfg::WTM, wn * Cfg::WTN);
}

// columns 64 H .. 64 H + 63 of a wave's 96 x 128 results (int8): six accumulator rows of 16, the epilogue of a 192 x 256 tile
template <class Cfg, int H, int I> __device__ __forceinline__ void fetch_row_192(v4i (&acc)[6][4]) {
    int r[16];
    w4_read16<8 * H + I>(r);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[I][j] = (v4i){r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]};
}
template <class Cfg, int H>
__device__ __forceinline__ void finish_half_192(const GemmParams &p, char *smem, int wave, int lane, int64_t mwave, int64_t nwave, const float *lsc, int mlw, int nlw) {
    typedef GemmCfg<192, 256, 2, 4, Cfg::A_KMAJOR, Cfg::B_KMAJOR, OP_I8, 0, 0, EPI_ROWCOL> ECfg;
    v4i acc[6][4];
    fetch_row_192<Cfg, H, 0>(acc); fetch_row_192<Cfg, H, 1>(acc); fetch_row_192<Cfg, H, 2>(acc);
    fetch_row_192<Cfg, H, 3>(acc); fetch_row_192<Cfg, H, 4>(acc); fetch_row_192<Cfg, H, 5>(acc);
    run_epilogue<ECfg>(p, acc, nullptr, smem, wave * 2 + H, lane, mwave, nwave + 64 * H, lsc, mlw, nlw + 64 * H);
}

// ------------------------------------------------------------------------------ 256 x 256, one wave per SIMD (gnk_gemm_w4.h)
// rows: K % 256 == 0, the dense loop on the group's tile.  depth: the contraction ends where the group does, so the loop reads through buffer
// descriptors that end there too: k-rows past the end are out of range and arrive in LDS as zeros, which add nothing in int8 and fp8; the loop
// runs over ceil(T_e / 256) * 256 of them (a group without rows: once over zeros).  Host-checked: T * pitch < 2^32 (the descriptors' sizes).
// BM = 192 (rows, int8): the same loop with three quarters of the rows, for tile counts that leave the last round of 256-row tiles nearly empty.
// Bound by the matrix cores and ~12 us per tile in which they stand still (first loads, epilogue; one workgroup per CU leaves nothing to run meanwhile):
// int8 over 8 experts, rows form 32768 x 2048 -> 5632 (twelve rounds of 16 steps): 350-370 us, 2.1 POP/s, matrix pipes 57 % busy; depth form 5632 x 2048
// over the same rows (three rounds of 32 steps): 301-328 us, 2.4 POP/s, 69 %; e4m3 298-313.  192: 16384 x 4096 -> 1024 over 32 experts in two rounds: 86-88 us, 1.6 POP/s.
template <class Cfg, bool DEPTH, int BM = 256>
__global__ void __launch_bounds__(256) w4_kernel(const GroupedParams gp) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef typename W4Select<Cfg, Cfg::OP>::type K;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const Tile tile = DEPTH ? depth_tile<256>(gp, gp.g.grid_m, gp.g.grid_n, lane) : rows_tile<BM>(gp, gp.g.grid_n, lane);
    if (!tile.work) return;
    constexpr int WTM = BM / 2;
    const int64_t m0 = (int64_t)tile.tm * BM, n0 = (int64_t)tile.tn * 256;
    if (!DEPTH && tile.e == gp.E) {
        zero_tile<BM, 256, 256>((char *)gp.g.C + tile.lo * gp.g.N * gp.out_bytes, tile.hi - tile.lo, gp.g.N, m0, n0, gp.out_bytes);
        return;
    }
    int64_t ext_a, ext_b;
    const GemmParams p = tile_params<DEPTH>(gp, tile, ext_a, ext_b);

    const int t = threadIdx.x;
    const int64_t mi = m0 + t < p.M - 1 ? m0 + t : p.M - 1;
    const int64_t ni = p.col_scalar ? 0 : (n0 + t < p.N - 1 ? n0 + t : p.N - 1);
    unsigned raw_r = 0, raw_c = 0;
    if constexpr (Cfg::EPI == EPI_ROWCOL) {
        raw_r = gnk_load_raw_rt(p.s0, p.scale_dtype, mi);
        raw_c = gnk_load_raw_rt(p.s1, p.scale_dtype, ni);
    }

    StagerW4<Cfg::A_KMAJOR> sa;
    StagerW4<Cfg::B_KMAJOR> sb;
    sa.init(p.A, p.lda, m0, ext_a, wave, lane);
    sb.init(p.B, p.ldb, n0, ext_b, wave, lane);

    const unsigned lds0 = (unsigned)(uintptr_t)(GNK_LDS char *)smem;
    const unsigned va = lds0 + K::frag0(Cfg::A_KMAJOR, wm * WTM, lane);
    const unsigned vb = lds0 + 4 * Cfg::OPER_BYTES + K::frag0(Cfg::B_KMAJOR, wn * 128, lane);
    const unsigned alo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)sa.base), ahi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)sa.base >> 32));
    const unsigned blo = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)sb.base), bhi = __builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)sb.base >> 32));
    const unsigned stepa = __builtin_amdgcn_readfirstlane((unsigned)sa.step), stepb = __builtin_amdgcn_readfirstlane((unsigned)sb.step);
    const unsigned ldsw = __builtin_amdgcn_readfirstlane(lds0 + wave * 1024);
#define GNK_GROUPED_W4_IN                                                                                                             \
                 [alo] "s"(alo), [ahi] "s"(ahi), [blo] "s"(blo), [bhi] "s"(bhi), [stepa] "s"(stepa), [stepb] "s"(stepb),              \
                 [lds] "s"(ldsw), [nit] "s"(nit), [va] "v"(va), [vb] "v"(vb),                                                         \
                 [oa0] "v"(sa.off[0]), [oa1] "v"(sa.off[1]), [oa2] "v"(sa.off[2]), [oa3] "v"(sa.off[3]),                              \
                 [ob0] "v"(sb.off[0]), [ob1] "v"(sb.off[1]), [ob2] "v"(sb.off[2]), [ob3] "v"(sb.off[3]),                              \
                 [fa] "i"(Cfg::FA), [fb] "i"(Cfg::FB)
    if constexpr (DEPTH) {
        const int nit = uniform(p.K > 0 ? (int)((p.K + 255) >> 8) : 1);
        // the bytes from the tile's first column in its first row to the end of the group's last row
        const unsigned abytes = __builtin_amdgcn_readfirstlane(p.K > 0 ? (unsigned)(p.K * p.lda - m0) : 0u);
        const unsigned bbytes = __builtin_amdgcn_readfirstlane(p.K > 0 ? (unsigned)(p.K * p.ldb - n0) : 0u);
        if constexpr (Cfg::OP == OP_I8)
            asm volatile(GNK_W4_ASM_I8_MM_RAGGED : : GNK_GROUPED_W4_IN, [abytes] "s"(abytes), [bbytes] "s"(bbytes) : GNK_W4_CLOBBERS_RAGGED);
        else
            asm volatile(GNK_W4_ASM_F8_MM_RAGGED : : GNK_GROUPED_W4_IN, [abytes] "s"(abytes), [bbytes] "s"(bbytes) : GNK_W4_CLOBBERS_RAGGED);
    } else {
        const int ns = (int)(p.K / Cfg::SK);   // a multiple of 4, >= 4 (host-checked)
        const int nit = __builtin_amdgcn_readfirstlane(ns >> 2), rem = __builtin_amdgcn_readfirstlane(ns - 1);
#define GNK_GROUPED_W4_RUN(TEXT)                                                                                                      \
        asm volatile(TEXT : : GNK_GROUPED_W4_IN, [rem] "s"(rem), [oa4] "v"(sa.off[4]), [oa5] "v"(sa.off[5]), [oa6] "v"(sa.off[6]),    \
                     [oa7] "v"(sa.off[7]), [ob4] "v"(sb.off[4]), [ob5] "v"(sb.off[5]), [ob6] "v"(sb.off[6]), [ob7] "v"(sb.off[7])     \
                     : GNK_W4_CLOBBERS)
        if constexpr (Cfg::OP == OP_I8) {
            if constexpr (BM == 192 && Cfg::B_KMAJOR) GNK_GROUPED_W4_RUN(GNK_W4_ASM_I8_KK_192);
            else if constexpr (BM == 192) GNK_GROUPED_W4_RUN(GNK_W4_ASM_I8_KM_192);
            else if constexpr (Cfg::B_KMAJOR) GNK_GROUPED_W4_RUN(GNK_W4_ASM_I8_KK);
            else GNK_GROUPED_W4_RUN(GNK_W4_ASM_I8_KM);
        } else {
            if constexpr (Cfg::B_KMAJOR) GNK_GROUPED_W4_RUN(GNK_W4_ASM_F8_KK);
            else GNK_GROUPED_W4_RUN(GNK_W4_ASM_F8_KM);
        }
#undef GNK_GROUPED_W4_RUN
    }
#undef GNK_GROUPED_W4_IN
    // the asm ends behind vmcnt(0) + a barrier: LDS is free for the epilogue
    float *const lsc = (float *)(smem + Cfg::LDS_BYTES);
    if (BM == 256 || (int)threadIdx.x < BM) *(GNK_LDS float *)(GNK_LDS char *)((char *)lsc + 4 * threadIdx.x) = gnk_raw_to_f32_rt(raw_r, p.scale_dtype);
    *(GNK_LDS float *)(GNK_LDS char *)((char *)lsc + 4 * (BM + threadIdx.x)) = gnk_raw_to_f32_rt(raw_c, p.scale_dtype);      // behind the rows' (EpiScales)
    __syncthreads();
    if constexpr (BM == 192) {
        finish_half_192<Cfg, 0>(p, smem, wave, lane, m0 + wm * WTM, n0 + wn * 128, lsc, wm * WTM, wn * 128);
        finish_half_192<Cfg, 1>(p, smem, wave, lane, m0 + wm * WTM, n0 + wn * 128, lsc, wm * WTM, wn * 128);
    } else {
        K::template finish_half<0>(p, smem, wave, lane, m0 + wm * 128, n0 + wn * 128, lsc, wm * 128, wn * 128);
        K::template finish_half<1>(p, smem, wave, lane, m0 + wm * 128, n0 + wn * 128, lsc, wm * 128, wn * 128);
    }
}

// most row tiles the groups can need: every group wastes less than one tile, and the rows behind the last group are one group more
static inline int64_t max_row_tiles(int64_t T, int64_t E, int64_t bm) {
    const int64_t by_rows = T / bm + E + 1;
    return by_rows < T ? by_rows : T;       // no tile is empty
}

template <class Kernel> static int reserve_lds(Kernel k, int bytes, std::atomic<bool> (&done)[64]) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return gnk_fail(GNK_ERR_LAUNCH, "grouped mm: no current HIP device");
    if (!done[dev].load(std::memory_order_acquire)) {      // opt in to > 64 KiB of dynamic LDS once per device and kernel
        if (hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
            return gnk_fail(GNK_ERR_LAUNCH, "grouped mm: cannot reserve %d bytes of LDS", bytes);
        done[dev].store(true, std::memory_order_release);
    }
    return GNK_OK;
}

// A group's contraction in parts (few tiles, many rows: 1024 x 1024 over 32768 rows are 64 tiles of 256 steps, two thirds of the chip idle): every part's sum
// lands in a slab of its own and this kernel adds them in order (so that equal calls give equal bits), scales and rounds once.  HBM-bound; V = 4 adjacent
// columns per thread where N allows.  Whole calls, one part -> the parts chosen, int8: 1024 x 1024 over 32768 rows 182 -> 49 us (16 parts, 1.4 POP/s; the slabs,
// 67 MB written and read, are half of it), 4096 x 1024 252 -> 115 (4), 64 x 64 127 -> 16 (32), four groups of 512 x 512 51 -> 28 (8).
// The parts of an int8 sum fit 32 bits; the sum of all of them does for up to INT8_TERMS rows, WIDE otherwise (64 bits: 1024 x 1024 in 16 parts 51 -> 52 us).
template <int OP, bool WIDE> struct JoinT { typedef float type; };
template <> struct JoinT<OP_I8, false> { typedef int type; };
template <> struct JoinT<OP_I8, true> { typedef long long type; };

// `count` sums `stride` bytes apart, V adjacent columns each, added in order, scaled, rounded and stored at element `out_at` of C
template <int OP, int V, bool WIDE>
__device__ __forceinline__ void join_columns(const char *src, int64_t stride, int count, float rs, const float (&cs)[V], char *__restrict__ C, int64_t out_at, int out_dtype) {
    typedef typename AccT<OP>::type acc_t;                   // v4i or v4f
    typename JoinT<OP, WIDE>::type acc[V];
#pragma unroll
    for (int r = 0; r < V; ++r) acc[r] = 0;
    constexpr int FLIGHT = 8;                                // loads in flight (four: 20 instead of 16 us for 64 x 64 in 32 parts)
    for (int k0 = 0; k0 < count; k0 += FLIGHT) {
        acc_t part[FLIGHT];
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k) {                   // past the end the last one again, for nothing
            const char *at = src + (k0 + k < count ? k0 + k : count - 1) * stride;
            if constexpr (V == 4) part[k] = *(const acc_t *)at;
            else __builtin_memcpy(&part[k], at, 4);
        }
#pragma unroll
        for (int k = 0; k < FLIGHT; ++k)
            if (k0 + k < count)
#pragma unroll
                for (int r = 0; r < V; ++r) acc[r] += part[k][r];
    }
    float v[V];
#pragma unroll
    for (int r = 0; r < V; ++r) v[r] = __fmul_rn(__fmul_rn((float)acc[r], rs), cs[r]);
    if constexpr (V == 4) {
        if (out_dtype == GNK_F32) *(v4f *)(C + 4 * out_at) = (v4f){v[0], v[1], v[2], v[3]};
        else if (out_dtype == GNK_BF16) *(v2i *)(C + 2 * out_at) = (v2i){(int)gnk_pack2_bf16(v[0], v[1]), (int)gnk_pack2_bf16(v[2], v[3])};
        else *(v2i *)(C + 2 * out_at) = (v2i){(int)gnk_pack2_f16(v[0], v[1]), (int)gnk_pack2_f16(v[2], v[3])};
    } else {
        gnk_store_scalar_rt(C, out_dtype, out_at, v[0]);
    }
}

template <int OP, int V, bool WIDE>
__global__ void __launch_bounds__(256) join_kernel(const void *__restrict__ slab, char *__restrict__ C, const char *__restrict__ s0, const char *__restrict__ s1, int64_t E,
                                                   int64_t M, int64_t N, int splits, int scale_dtype, int col_scalar, int out_dtype) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, total = E * M * N;
    if (i >= total) return;
    const int64_t row = i / N, n = i - row * N, e = row / M;
    float cs[V];
#pragma unroll
    for (int r = 0; r < V; ++r) cs[r] = gnk_load_scalar_rt(s1, scale_dtype, col_scalar ? e : e * N + n + r);
    join_columns<OP, V, WIDE>((const char *)slab + 4 * i, total * 4, splits, gnk_load_scalar_rt(s0, scale_dtype, row), cs, C, i, out_dtype);
}

// The pieces of the groups of more than LONG_ROWS rows: the workgroups of a group's first piece (blockIdx.y) add them all.  5632 x 2048, groups of 139000 and 1000
// rows: 14 us of 1410.
template <int V>
__global__ void __launch_bounds__(256) join_long_kernel(const GroupedParams p) {
    const Piece pc = find_long_piece(p.ends, p.E, p.T, threadIdx.x & 63, (int)blockIdx.y);
    if (pc.e < 0 || pc.idx != 0) return;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, each = p.g.M * p.g.N;
    if (i >= each) return;
    const int64_t m = i / p.g.N, n = i - m * p.g.N, e = pc.e;
    float cs[V];
#pragma unroll
    for (int r = 0; r < V; ++r) cs[r] = gnk_load_scalar_rt(p.g.s1, p.g.scale_dtype, p.g.col_scalar ? e : e * p.g.N + n + r);
    join_columns<OP_I8, V, true>((const char *)p.slab + ((int64_t)blockIdx.y * each + i) * 4, each * 4, long_pieces_of(pc.hi - pc.lo),
                        gnk_load_scalar_rt(p.g.s0, p.g.scale_dtype, e * p.g.M + m), cs, (char *)p.g.C, e * each + i, p.g.out_dtype);
}

static inline bool join_quads(const GroupedParams &p) { return p.g.N % 4 == 0 && ((uintptr_t)p.g.C & 15) == 0; }

template <int OP> int join_parts(const GroupedParams &p, hipStream_t st) {
    const int64_t total = p.E * p.g.M * p.g.N;
    const bool quads = join_quads(p);
    const int64_t blocks = (total / (quads ? 4 : 1) + 255) / 256;
    const auto args = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, p.slab, (char *)p.g.C, (const char *)p.g.s0, (const char *)p.g.s1, p.E, p.g.M, p.g.N, p.splits,
                           p.g.scale_dtype, p.g.col_scalar, p.g.out_dtype);
    };
    if (OP == OP_I8 && p.T > INT8_TERMS) quads ? args(join_kernel<OP, 4, true>) : args(join_kernel<OP, 1, true>);
    else quads ? args(join_kernel<OP, 4, false>) : args(join_kernel<OP, 1, false>);
    return gnk_check_launch("grouped mm: joining the parts");
}

static inline int join_long(const GroupedParams &p, hipStream_t st) {
    const bool quads = join_quads(p);
    const int64_t blocks = (p.g.M * p.g.N / (quads ? 4 : 1) + 255) / 256;
    if (blocks >= (1LL << 31)) return gnk_fail(GNK_ERR_UNSUPPORTED, "grouped mm: too many outputs");
    const dim3 grid((unsigned)blocks, (unsigned)p.pieces);
    if (quads) hipLaunchKernelGGL((join_long_kernel<4>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((join_long_kernel<1>), grid, dim3(256), 0, st, p);
    return gnk_check_launch("grouped mm: joining the pieces of long groups");
}

// Tile sizes of a launch over the whole grid; KERNEL with its LDS.
template <class Kernel> int launch_tiles(Kernel kernel, std::atomic<bool> (&done)[64], int lds, int threads, bool depth, int bm, int bn, const GroupedParams &p0, hipStream_t st) {
    GroupedParams p = p0;
    p.g.grid_n = (int)((p.g.N + bn - 1) / bn);
    p.g.grid_m = depth ? (int)((p.g.M + bm - 1) / bm) : 0;
    const int64_t blocks = (depth ? (p.pieces ? p.pieces : p.E) * p.g.grid_m * p.splits : max_row_tiles(p.T, p.E, bm)) * p.g.grid_n;
    if (blocks >= (1LL << 31)) return gnk_fail(GNK_ERR_UNSUPPORTED, "grouped mm: too many tiles");
    const int rc = reserve_lds(kernel, lds, done);
    if (rc) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, st, p);
    return gnk_check_launch("grouped mm");
}

template <class Cfg, bool DEPTH> int launch_two_buffer(const GroupedParams &p, hipStream_t st) {
    static std::atomic<bool> done[64];
    return launch_tiles(two_buffer_kernel<Cfg, DEPTH>, done, Cfg::LDS_BYTES + ScalePrefetch<Cfg::BM, Cfg::BN, Cfg::NT, Cfg::EPI>::BYTES, Cfg::NT, DEPTH, Cfg::BM,
                        Cfg::BN, p, st);
}

template <class Cfg, bool DEPTH, int KG> int launch_ring_of(const GroupedParams &p, hipStream_t st) {
    static std::atomic<bool> done[64];
    return launch_tiles(ring_kernel<Cfg, DEPTH, KG>, done, KG * 4 * (Cfg::A_BYTES + Cfg::B_BYTES) + (Cfg::BM + Cfg::BN) * 4, KG * Cfg::NT, DEPTH, Cfg::BM, Cfg::BN, p, st);
}
template <class Cfg, bool DEPTH> int launch_ring(const GroupedParams &p, int kg, hipStream_t st) {
    return kg == 2 ? launch_ring_of<Cfg, DEPTH, 2>(p, st) : launch_ring_of<Cfg, DEPTH, 1>(p, st);
}

template <class Cfg, bool DEPTH, int BM = 256> int launch_w4(const GroupedParams &p, hipStream_t st) {
    static std::atomic<bool> done[64];
    return launch_tiles(w4_kernel<Cfg, DEPTH, BM>, done, Cfg::LDS_BYTES + 2048, 256, DEPTH, BM, 256, p, st);
}

// Tile choice by a cost model in us on the sizes that the host knows: groups of T / E rows, half a tile of edge each.  Constants fitted to forced runs of every
// variant over 16 .. 32768 rows, 1 .. 64 groups, K, N = 512 .. 5632: a 256 x 256 or 192 x 256 workgroup (one per CU) costs 11-12 + 1.08 / 0.86 per 128 k, a
// 128 x 128 one (two per CU) 6 + 1.0 with both operands K-major, 1.5 with B N-major, 1.3 in the depth form, a 64 x 64 one 5 + 0.55, or 0.33 with
// two sets of waves, one per CU.
// Parts of a contraction (depth, 128 and 256 tiles): a second launch and the slabs, written and read at about 4 TB/s.
constexpr int VARIANT_192 = 100;             // beside gnk_set_gemm_variant's numbers: 192 x 256 (int8, rows form)
constexpr int MAX_SPLITS = 32;
struct Plan { int variant, splits, kg; };      // kg: sets of waves of the 64 x 64 kernel

static inline Plan choose_variant(int64_t T, int64_t groups_n, int64_t M, int64_t N, int64_t K, bool depth, bool b_kmajor, bool can_w4, bool can_192, int forced) {
    const double cus = (double)gnk_num_cus(), rows = (double)T, E = (double)(groups_n > 0 ? groups_n : 1);
    const double groups = E * (1.0 - pow(1.0 - 1.0 / E, rows));      // groups that a uniform router leaves with a row
    auto tiles = [&](double bm, double bn) {
        const double gn = ceil((double)N / bn);
        if (depth) return E * ceil((double)M / bm) * gn;
        // sizes spread: where a group has half a tile or more on average, some have more than one
        const double m = rows / bm + 0.5 * groups, fill = groups > 0 ? rows / groups / bm : 0.0, least = groups * (1.0 + 0.3 * (fill < 0.5 ? fill : 0.5));
        return (m > least ? m : least) * gn;
    };
    // whole rounds, but the number of row tiles is an estimate: the mean over 5 % less, 5 % and 15 % more of them (depth: it is known)
    auto rounds = [&](double n, double slots) {
        return depth ? ceil(n / slots) : (ceil(0.95 * n / slots) + ceil(1.05 * n / slots) + ceil(1.15 * n / slots)) / 3.0;
    };
    // two workgroups per CU run at different times: the rounds of the 128 x 128 kernel smear
    auto smeared = [&](double n, double slots) { return n <= slots ? 1.0 : n / slots + 0.25; };
    const double ks = depth ? rows / E / 128.0 : (double)K / 128.0;
    const double edge = depth ? 1.0 : 0.0;       // a 256-k step of the ragged loop is half empty on average
    Plan best = {GNK_VARIANT_128, 1, 1};
    double t_best = 1e30;
    auto offer = [&](int variant, int splits, double t, int kg = 1) {
        if (t < t_best && (forced < 0 || forced == variant)) { t_best = t; best = {variant, splits, kg}; }
    };
    offer(GNK_VARIANT_64X128, 1, rounds(tiles(64, 64), 2.0 * cus) * (5.0 + 0.55 * ks));
    if (ks >= 4.0) offer(GNK_VARIANT_64X128, 1, rounds(tiles(64, 64), cus) * (5.0 + 0.33 * ks), 2);
    if (can_w4) offer(GNK_VARIANT_256_W4, 1, rounds(tiles(256, 256), cus) * (12.0 + 1.08 * (ks + edge)));
    if (can_192) offer(VARIANT_192, 1, rounds(tiles(192, 256), cus) * (11.0 + 0.86 * ks) / 0.98);
    offer(GNK_VARIANT_128, 1, smeared(tiles(128, 128), 2.0 * cus) * (6.0 + (depth ? 1.3 : b_kmajor ? 1.0 : 1.5) * ks));
    if (depth)
        for (int s = 2; s <= MAX_SPLITS && ks / s >= 4.0; s *= 2) {
            const double join = 4.0 + 8.0 * s * E * (double)M * (double)N / 4.0e6;
            offer(GNK_VARIANT_128, s, smeared(tiles(128, 128) * s, 2.0 * cus) * (6.0 + 1.3 * ks / s) + join);
            if (can_w4) offer(GNK_VARIANT_256_W4, s, rounds(tiles(256, 256) * s, cus) * (12.0 + 1.08 * (ks / s + edge)) + join);
        }
    return best;
}

static inline int64_t split_bytes(int splits, int64_t E, int64_t M, int64_t N) { return splits > 1 ? splits * E * M * N * 4 : 0; }

// pieces that groups of more than LONG_ROWS rows can come to, T rows in all: the sum of ceil(rows / LONG_ROWS) over at most T / (LONG_ROWS + 1) groups
static inline int64_t most_long_pieces(int64_t T) { return T / LONG_ROWS + T / (LONG_ROWS + 1); }

template <int OP, int FA, int FB> int launch(bool depth, bool b_kmajor, const GroupedParams &p0, hipStream_t st) {
    const bool can_w4 = depth ? p0.T * (p0.g.lda > p0.g.ldb ? p0.g.lda : p0.g.ldb) < (1LL << 32) : p0.g.K >= 256 && p0.g.K % 256 == 0;
    const bool can_192 = OP == OP_I8 && !depth && can_w4;
    // gnk_set_gemm_variant: 1, 5 and 6 force the 128 x 128, the 256 x 256 (where it can run) and the 64 x 64 kernel, 0 the 192 x 256 one
    int forced = gnk_forced_variant_get();
    if (forced == GNK_VARIANT_256 && can_192) forced = VARIANT_192;
    else if ((forced != GNK_VARIANT_128 && forced != GNK_VARIANT_64X128 && forced != GNK_VARIANT_256_W4) || (forced == GNK_VARIANT_256_W4 && !can_w4)) forced = -1;
    const Plan plan = choose_variant(p0.T, p0.E, p0.g.M, p0.g.N, p0.g.K, depth, b_kmajor, can_w4, can_192, forced);
    const int variant = plan.variant;
    GroupedParams p = p0;
    p.splits = plan.splits;
    while (p.splits > 1 && split_bytes(p.splits, p.E, p.g.M, p.g.N) > p.slab_bytes) p.splits /= 2;       // no room for the parts: fewer of them
    const auto plain_sums = [&](GroupedParams q) {
        q.g.C = q.slab;
        q.g.out_dtype = OP == OP_I8 ? GNK_I32 : GNK_F32;
        q.out_bytes = 4;
        return variant == GNK_VARIANT_256_W4 ? launch_w4<PP2Cfg<false, false, OP, FA, FB, EPI_PLAIN>, true>(q, st)
                                             : launch_two_buffer<GemmCfg<128, 128, 2, 2, false, false, OP, FA, FB, EPI_PLAIN>, true>(q, st);
    };
    if constexpr (OP == OP_I8) {
        // parts of at most LONG_ROWS rows, whoever has them, or groups of more in pieces
        if (depth && p.T > LONG_ROWS && p.splits * (int64_t)LONG_ROWS < p.T) {
            p.splits = 1;
            p.long_rows = LONG_ROWS;
            GroupedParams q = p;
            q.pieces = (int)most_long_pieces(p.T);
            if (p.slab_bytes < q.pieces * p.g.M * p.g.N * 4)
                return gnk_fail(GNK_ERR_WORKSPACE, "grouped_scaled_mm: int8 sums over %lld rows need the workspace of gnk_grouped_scaled_mm_depth_split_bytes", (long long)p.T);
            int rc = plain_sums(q);
            if (!rc) rc = join_long(q, st);
            if (rc) return rc;
        }
    }
    if (p.splits > 1) {
        const int rc = plain_sums(p);
        return rc ? rc : join_parts<OP>(p, st);
    }
    if constexpr (OP == OP_I8) {
        if (variant == VARIANT_192)
            return b_kmajor ? launch_w4<PP2Cfg<true, true, OP, FA, FB, EPI_ROWCOL>, false, 192>(p, st)
                            : launch_w4<PP2Cfg<true, false, OP, FA, FB, EPI_ROWCOL>, false, 192>(p, st);
    }
    if (variant == GNK_VARIANT_256_W4) {
        if (depth) return launch_w4<PP2Cfg<false, false, OP, FA, FB, EPI_ROWCOL>, true>(p, st);
        if (b_kmajor) return launch_w4<PP2Cfg<true, true, OP, FA, FB, EPI_ROWCOL>, false>(p, st);
        return launch_w4<PP2Cfg<true, false, OP, FA, FB, EPI_ROWCOL>, false>(p, st);
    }
    if (variant == GNK_VARIANT_64X128) {
        if (depth) return launch_ring<GemmCfg<64, 64, 4, 1, false, false, OP, FA, FB, EPI_ROWCOL>, true>(p, plan.kg, st);
        if (b_kmajor) return launch_ring<GemmCfg<64, 64, 4, 1, true, true, OP, FA, FB, EPI_ROWCOL>, false>(p, plan.kg, st);
        return launch_ring<GemmCfg<64, 64, 4, 1, true, false, OP, FA, FB, EPI_ROWCOL>, false>(p, plan.kg, st);
    }
    if (depth) return launch_two_buffer<GemmCfg<128, 128, 2, 2, false, false, OP, FA, FB, EPI_ROWCOL>, true>(p, st);
    if (b_kmajor) return launch_two_buffer<GemmCfg<128, 128, 2, 2, true, true, OP, FA, FB, EPI_ROWCOL>, false>(p, st);
    return launch_two_buffer<GemmCfg<128, 128, 2, 2, true, false, OP, FA, FB, EPI_ROWCOL>, false>(p, st);
}

}  // namespace gnk_grouped

#define GNK_DEFINE_GROUPED(NAME, OP, FA, FB) \
    int NAME(bool depth, bool b_kmajor, const GroupedParams &p, hipStream_t st) { return gnk_grouped::launch<OP, FA, FB>(depth, b_kmajor, p, st); }
