// gnk_ortho.hip -- orthogonalisation of matrices by Newton-Schulz products on the 16-bit matrix cores (gfx950).
//
//   X_0 = G / max(|G|_F, eps);   S = X X^T (wide) or X^T X (tall),  Q = a I + b S + c S^2,  X <- Q X (wide) or X Q (tall),   `steps` times
//
// Three products per step.  Everything between them is kept in fp16 with power-of-two scales and accumulated in fp32: the polynomial amplifies what
// is small (by a per step where S is near 0), and with it the rounding of the intermediate matrices; bf16's 8 bits leave 1-5 % in the result, fp16's
// 11 bits an eighth of that at the same matrix rate.  Ranges: |X| <= 1 element by element while its singular values stay around 1, so
//   X_0 as G 2^p with |G|_F 2^p in [2^14, 2^15): no rounding at all for bf16 and fp16 inputs (1 / |G|_F goes into the products' factors);
//   later X as X 2^10, S as S 2^10, Q - mu I as (Q - mu I) 2^s with |a| + 2 |b| + 4 |c| < 2^(14 - s): nothing overflows, and what underflows is
//   below 2^-24.  mu = p(mean of S's diagonal), p(s) = a + b s + c s^2, is about the mean of Q's diagonal, which otherwise carries most of Q's rounding error:
//   three quarters of the whole result's for flat matrices (36 x 2230: 2.6e-3 -> 2.0e-3 of the result's norm, 1.7e-3 of which is the output's bf16).  mu X is added in fp32 where Q X is stored.  From 512 rows on the
//   rounding of X is most of the error (512 x 512: 1.4e-3 of 1.6e-3) and the second read of X costs 15 % of that product: mu = 0 there.
// That is an eighth of what a bf16 result is rounded by and five times a fp16 result's rounding, so results of 11 and 24 bits (fp16, fp32) are computed with every
// matrix in two fp16 parts, hi + lo (PAIRS; 22 bits, no mu): a product is hi hi + lo hi + hi lo, one loop over three times the contraction.  Off by 2.1e-4 of the
// norm for fp16, its rounding, and 1-3e-6 for fp32, where one part each gave 1.1e-3; 999 x 333 207 us instead of 120, 8 x 2048 x 5632 8.8 ms instead of 2.9.
// Shapes are padded with zeros to multiples of 128 in the workspace: zero rows and columns stay zero through every product.
//
// The products: `wide` S = X X^T reads both operands along K, Q X reads X as it lies (N-contiguous, transposed on the way out of LDS); `tall` S = X^T X
// reads X as it lies on both sides, X Q reads along K (Q is symmetric); S^2 = S S^T.  So nothing is ever transposed in memory.
// Bound: the matrix cores, m^2 n + m^3 + 2 m^2 n operations per step (m <= n; S and S^2 are symmetric).
// Measured, bf16, five steps: 8 x 2048 x 5632 2.88 ms, 1.1 PFLOP/s (a large fp16 product reaches 1.42); 2048 x 5632 650 us; 2048 x 2048 428 us; 999 x 333 120 us,
// 64 x 64 67 us: 17 dependent launches of 3-10 us, 0.8 us apart.  (Requesting the epilogue's reads and the diagonal ahead of the loop changed nothing there.)
#include <math.h>
#include <string.h>

#include "gnk_gemm_w4.h"
#include "gnk_gemm_w4_more_asm.inc"

namespace {

using namespace gnk_gemm;

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr int64_t MU_ROWS = 512;             // smaller sides below this: Q without its mean diagonal
constexpr int PAD = 128;                     // rows and columns of every intermediate are padded to this
constexpr float SX = 1024.0f, SS = 1024.0f;  // scales of X (after step 0) and S
constexpr int MAX_PARTS = 256;               // partial sums of squares per matrix

// Epilogues: GRAM acc * f;  POLY acc * f + D * g + (on the diagonal) (h - mu) k, D = S;  UPDATE (acc + D * k mu) * f, D = X
enum { GRAM = 0, POLY = 1, UPDATE = 2 };

struct Product {
    const char *A, *B;
    void *C;
    const char *D;                           // POLY: the matrix S; UPDATE: X
    int64_t ba, bb, bc, bd;                  // bytes from one matrix of the stack to the next
    int64_t a_lo, b_lo, c_lo, d_lo;          // PAIRS: bytes from the hi part to the lo part (c_lo = 0: the result has none)
    int64_t M, N, K;                         // output extents that are stored; K a multiple of 128
    int64_t lda, ldb, ldd;                   // bytes
    int64_t ext_a, ext_b;                    // staged extents (elements, >= M / N, multiples of 128)
    float f, g, h, k;
    float c0, c1, c2;                        // POLY: mu = c0 + c1 s + c2 s^2, s = diag_scale * (sum of D's diagonal)
    float diag_scale;
    float *mu;                               // per matrix: written by POLY's first tile, read by UPDATE; NULL: mu = 0
    const float *fdev;                       // GRAM, UPDATE: a further factor per matrix (step 0), or NULL
    int fstride;
    int out_dtype;
    int batch, grid_m, grid_n;
    int parts;                               // PAIRS, 128 and 64 tiles: 3, or 1 where neither factor has a lo part
};

// Tile of a workgroup: the XCDs take contiguous runs of tiles (matrices one after the other), each walked in strips of four tile rows.
// SYM: only the tiles on and above the diagonal, row by row; the others are their mirror images (store_mirror).
template <bool SYM> __host__ __device__ __forceinline__ int tiles_of(const Product &p) { return SYM ? p.grid_m * (p.grid_m + 1) / 2 : p.grid_m * p.grid_n; }

template <bool SYM> __device__ __forceinline__ void batch_tile(const Product &p, int &b, int &tm, int &tn) {
    const int per = tiles_of<SYM>(p), nwg = per * p.batch;
    const int xcd = (int)blockIdx.x & 7, idx = (int)blockIdx.x >> 3, q = nwg >> 3, r = nwg & 7;
    const int wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
    b = wg / per;
    int in = wg - b * per;
    if constexpr (SYM) {
        tm = 0;
        while (in >= p.grid_m - tm) in -= p.grid_m - tm++;
        tn = tm + in;
    } else {
        const int width = 4 * p.grid_n, strip = in / width, first = strip * 4, gsz = min(p.grid_m - first, 4), rest = in - strip * width;
        tm = first + rest % gsz;
        tn = rest / gsz;
    }
}

// What an epilogue needs beside the accumulators
struct Finish {
    const char *D;
    float f, d, diag;                        // value = acc * f + D * d (+ diag on the diagonal)
};

// acc (lane: row m, columns n .. n + 3) -> the stored value
template <int EPI, bool PAIRS = false>
__device__ __forceinline__ void finish_value(const Product &p, const Finish &fin, v4f &acc, int64_t m, int64_t n) {
    if constexpr (EPI == GRAM) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] *= fin.f;
    } else {
        const int64_t mm = m < p.ext_a ? m : p.ext_a - 1, nn = n < p.ext_b ? n : p.ext_b - 4;
        const char *at = fin.D + mm * p.ldd + 2 * nn;
        const v4h d = *(const v4h *)at;
        v4h lo = {0, 0, 0, 0};
        if constexpr (PAIRS) lo = *(const v4h *)(at + p.d_lo);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            acc[r] = __builtin_fmaf(acc[r], fin.f, (PAIRS ? (float)d[r] + (float)lo[r] : (float)d[r]) * fin.d);
            if (EPI == POLY && m == n + r) acc[r] += fin.diag;
        }
    }
}

// POLY: this thread's part of the sum of S's diagonal (issued ahead of the products), and the workgroup's sum of them: every workgroup of a matrix adds the
// same numbers in the same order
template <int NT> __device__ __forceinline__ float diagonal_part(const Product &p, int b) {
    const char *D = p.D + b * p.bd;
    float s = 0.0f;
    if (!p.mu) return s;
    for (int64_t i = threadIdx.x; i < p.ext_a; i += NT) s += (float)*(const _Float16 *)(D + i * (p.ldd + 2));
    return s;
}
template <int NT> __device__ __forceinline__ float workgroup_sum(float s, char *lds) {
#pragma unroll
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d, 64);
    if ((threadIdx.x & 63) == 0) *(GNK_LDS float *)(GNK_LDS char *)(lds + 4 * (threadIdx.x >> 6)) = s;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) t += *(const GNK_LDS float *)(const GNK_LDS char *)(lds + 4 * w);
    __syncthreads();                         // the caller goes on using this LDS
    return t;
}

template <int EPI> __device__ __forceinline__ Finish make_finish(const Product &p, int b, bool first_tile, float diagonal_sum) {
    Finish fin = {nullptr, p.f, 0.0f, 0.0f};
    if constexpr (EPI != POLY) fin.f = p.fdev ? p.f * p.fdev[(int64_t)b * p.fstride] : p.f;
    if constexpr (EPI != GRAM) fin.D = p.D + b * p.bd;
    if constexpr (EPI == UPDATE) fin.d = p.mu[b] * p.k * fin.f;
    if constexpr (EPI == POLY) {
        const float s = diagonal_sum * p.diag_scale, mu = p.mu ? __builtin_fmaf(s, __builtin_fmaf(s, p.c2, p.c1), p.c0) : 0.0f;
        fin.d = p.g;
        fin.diag = (p.h - mu) * p.k;
        if (p.mu && first_tile && threadIdx.x == 0) p.mu[b] = mu;
    }
    return fin;
}

__device__ __forceinline__ GemmParams store_params(const Product &p, int b) {
    GemmParams g;
    __builtin_memset(&g, 0, sizeof(g));
    g.C = (char *)p.C + b * p.bc;
    g.M = p.M; g.N = p.N; g.K = p.K;
    g.out_dtype = p.out_dtype;
    return g;
}

// The transpose of a wave's 16 MT x 64 results (fp16 output, rows m0 .., columns n0 ..; both inside the padded matrix), through its slice of LDS:
// image [64 n][16 MT m], 16-byte chunk c of row n at c ^ 2 ((n >> 2) & 3), so that the four lane groups of a write land in different banks; rows of
// 32 MT bytes go out whole.
template <int MT> __device__ __forceinline__ void store_mirror(const Product &p, char *C, const v4f (&acc)[MT][4], char *region, int lane, int64_t m0, int64_t n0) {
    constexpr int PITCH = 32 * MT, CHUNKS = 2 * MT;
    static_assert(MT >= 4, "the swizzle needs eight chunks per row");
    if (m0 + 16 * MT > p.ext_a || n0 + 64 > p.ext_b) return;                  // padding tiles beyond the matrix (extents are multiples of 128)
    const int g = lane >> 4, ml = lane & 15;
    asm volatile("" ::: "memory");           // behind the wave's earlier reads of the slice
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = 16 * j + 4 * g + r, c = (2 * i + (ml >> 3)) ^ (2 * g);
                *(GNK_LDS _Float16 *)(GNK_LDS char *)(region + n * PITCH + 16 * c + 2 * (ml & 7)) = (_Float16)acc[i][j][r];
            }
#pragma unroll
    for (int u = 0; u < CHUNKS; ++u) {                                         // 64 rows x CHUNKS chunks over 64 lanes
        const int e = u * 64 + lane, n = e / CHUNKS, c = e % CHUNKS;
        const v4i v = *(const GNK_LDS v4i *)(const GNK_LDS char *)(region + n * PITCH + 16 * (c ^ (2 * ((n >> 2) & 3))));
        gnk_store16_out(C + 2 * ((n0 + n) * p.N + m0) + 16 * c, v);
    }
}

// ------------------------------------------------------------------------------ tiles of 128 or 64 with a ring of LDS stages
// This wave's pieces of one operand's 64-k step (BM rows x 128 bytes, or 64 k-rows x 2 BM bytes)
template <bool KMAJOR, int BM> struct Stager16 {
    static constexpr int NP = BM / 32;
    const char *base;
    unsigned off[NP];
    int64_t step;
    __device__ __forceinline__ void init(const char *ptr, int64_t ld, int64_t r0, int wave, int lane) {
        base = KMAJOR ? ptr + r0 * ld : ptr + 2 * r0;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int p = (i * 4 + wave) * 64 + lane;
            int r, c;
            if constexpr (KMAJOR) gnk_kmaj_stage_src(p, r, c);
            else gnk_mn16_stage_src<2 * BM>(p, r, c);
            off[i] = (unsigned)(r * ld + 16 * c);
        }
        step = KMAJOR ? 128 : 64 * ld;
    }
    __device__ __forceinline__ void issue(char *tile, int wave) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
            __builtin_amdgcn_global_load_lds((const GNK_GLOBAL void *)(base + off[i]), (GNK_LDS void *)(tile + (i * 4 + wave) * 1024), 16, 0, 0);
        base += step;
    }
};

template <bool KMAJOR, int BM> __device__ __forceinline__ v8h frag16(const char *tile, int rb, int ks, int lane) {
    v4i v;
    if constexpr (KMAJOR) {
        v = *(const GNK_LDS v4i *)(const GNK_LDS char *)(tile + gnk_kmaj_frag_offset(rb, ks, lane));
    } else {
        const int o = gnk_mn16_frag_offset<2 * BM>(rb, ks, lane);
        const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((GNK_LDS v4s *)(tile + o)));
        const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((GNK_LDS v4s *)(tile + o + 8 * BM)));
        v = (v4i){lo[0], lo[1], hi[0], hi[1]};
    }
    return __builtin_bit_cast(v8h, v);
}

// BM = 128: 2 x 2 waves of 64 x 64, two stages (64 KiB: two workgroups per CU).  BM = 64: 2 x 2 waves of 32 x 32 would halve the fragment reads, but the
// stores want 64 columns per wave: 4 x 1 waves of 16 x 64; four stages (64 KiB) because few tiles are bound by the latency of a step, not by its work.
// KG = 2 (at most one workgroup per CU): a second set of four waves with a ring of its own takes every other step of the contraction; the two
// halves meet in LDS, in the same order on both sides, and then one set stores the tile and the other its mirror image.  KG = 4 (64 tiles, from 24 steps on):
// four sets with two stages each.  100 x 4096 153 -> 137 us, 3000 x 400 206 -> 184, 1024 x 1024 fp16 360 -> 322; with 16 steps 121 -> 118 for one part, but
// 207 -> 216 us for pairs' 18 (999 x 333), with 8 slower everywhere.
// Bound by latency: a launch with one step takes 3 us, each further 64-k step of a set 0.7 (fragment reads, barrier), so 333 x 333 over K = 1024 takes 8.2 us.
// Two sets instead of one, tiles of 128: 2048 x 2048 530 -> 428 us, 2048 x 5632 749 -> 652 us (whole calls).
template <int BM, int KG> struct RingShape {
    static constexpr int WM = BM == 128 ? 2 : 4, WN = BM == 128 ? 2 : 1, MT = BM / WM / 16, NST = BM == 128 || KG == 4 ? 2 : 4, OPER = BM * 128, STAGE = 2 * OPER;
    static constexpr int LDS = NST * STAGE;
};

// PAIRS: the steps of hi hi, then lo hi, then hi lo; the result is stored as hi = fp16(v) and lo = fp16(v - hi), the last one in its own type.
template <int BM, int KG, bool AK, bool BK, int EPI, bool SYM, bool PAIRS>
__global__ void __launch_bounds__(256 * KG) __attribute__((amdgpu_waves_per_eu(KG == 4 ? 4 : 2))) product_ring_kernel(const Product p) {
    extern __shared__ __attribute__((aligned(16))) char smem_all[];
    typedef RingShape<BM, KG> R;
    static_assert(KG == 1 || KG == 2 || (KG == 4 && BM == 64), "sets of waves");
    typedef GemmCfg<BM, BM, R::WM, R::WN, AK, BK, OP_F8, 0, 0, EPI_PLAIN> Cfg;     // fp32 accumulators and the epilogue's maps
    constexpr int MT = R::MT, NST = R::NST, PIECES = 2 * BM / 32;
    const int lane = threadIdx.x & 63;
    const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = KG == 1 ? 0 : wave_all >> 2, wave = wave_all & 3;
    char *const smem = smem_all + kg * R::LDS;
    const int wm = wave / R::WN, wn = wave % R::WN;
    int b, tm, tn;
    batch_tile<SYM>(p, b, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BM;
    Stager16<AK, BM> sa;
    Stager16<BK, BM> sb;
    sa.init(p.A + b * p.ba, p.lda, m0, wave, lane);
    sb.init(p.B + b * p.bb, p.ldb, n0, wave, lane);
    const float diag = EPI == POLY ? diagonal_part<256 * KG>(p, b) : 0.0f;
    v4f acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (v4f){0.f, 0.f, 0.f, 0.f};
    const int nk_one = (int)(p.K / 64), nk_all = PAIRS ? p.parts * nk_one : nk_one;
    const int nk = (nk_all + KG - 1 - kg) / KG, nk_most = KG == 1 ? nk : (nk_all + KG - 1) / KG;      // steps kg, kg + KG, ...
    const char *const a0 = sa.base, *const b0 = sb.base;
    if constexpr (KG > 1 && !PAIRS) {
        sa.base += kg * sa.step;
        sb.base += kg * sb.step;
        sa.step *= KG;
        sb.step *= KG;
    }
    auto fetch = [&](int t) {
        if constexpr (PAIRS) {
            const int step = t * KG + kg, part = step >= 2 * nk_one ? 2 : (step >= nk_one ? 1 : 0), k = step - part * nk_one;
            sa.base = a0 + (part == 1 ? p.a_lo : 0) + k * sa.step;
            sb.base = b0 + (part == 2 ? p.b_lo : 0) + k * sb.step;
        }
        char *const into = smem + (t % NST) * R::STAGE;
        sa.issue(into, wave);
        sb.issue(into + R::OPER, wave);
    };
    for (int t = 0; t < NST - 1 && t < nk; ++t) fetch(t);
    for (int t = 0; t < nk_most; ++t) {
        // stage t has landed; t + 1 .. t + NST - 2 may stay in flight
        if (t + NST - 2 < nk) asm volatile("s_waitcnt vmcnt(%0)" : : "i"((NST - 2) * PIECES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        char *const As = smem + (t % NST) * R::STAGE, *const Bs = As + R::OPER;
        if (t + NST - 1 < nk) fetch(t + NST - 1);                      // into the buffer of stage t - 1, which every wave has read
        if (KG > 1 && t >= nk) break;                                  // the other set has one step more
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            v8h fa[MT], fb[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) fb[j] = frag16<BK, BM>(Bs, wn * 64 + 16 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[i] = frag16<AK, BM>(As, wm * 16 * MT + 16 * i, ks, lane);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[j], fa[i], acc[i][j], 0, 0, 0);
        }
    }
    if constexpr (KG > 1) {
        __syncthreads();                                               // both rings are free
        // every set's sums (at most all rings together), added in the order of the sets wherever they are wanted
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) *(GNK_LDS v4f *)(GNK_LDS char *)(smem_all + kg * BM * BM * 4 + 16 * (((wave * MT + i) * 4 + j) * 64 + lane)) = acc[i][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v4f sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KG; ++k) sum += *(const GNK_LDS v4f *)(const GNK_LDS char *)(smem_all + k * BM * BM * 4 + 16 * (((wave * MT + i) * 4 + j) * 64 + lane));
                acc[i][j] = sum;
            }
    }
    float diag_sum = 0.0f;
    if constexpr (EPI == POLY) {
        __syncthreads();
        diag_sum = workgroup_sum<256 * KG>(diag, smem_all);
    }
    const Finish fin = make_finish<EPI>(p, b, tm == 0 && tn == 0, diag_sum);
    const int64_t mw = m0 + wm * 16 * MT, nw = n0 + wn * 64;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) finish_value<EPI, PAIRS>(p, fin, acc[i][j], mw + 16 * i + (lane & 15), nw + 16 * j + 4 * (lane >> 4));
    GemmParams g = store_params(p, b);
#pragma unroll
    for (int part = 0; part < (PAIRS ? 2 : 1); ++part) {
        if constexpr (PAIRS) {
            if (part == 1) {
                if (!p.c_lo) break;
                g.C = (char *)g.C + p.c_lo;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] -= (float)(_Float16)acc[i][j][r];
            }
        }
        __syncthreads();                                               // the staging below overwrites the rings, or the hi part's staging
        if (kg == 0) run_epilogue<Cfg>(g, acc, nullptr, smem, wave, lane, mw, nw);
        if constexpr (SYM) {
            if (tm != tn) {
                if constexpr (MT >= 4) {
                    if (kg == KG - 1) store_mirror<MT>(p, (char *)g.C, acc, smem + R::LDS / 2 + wave * (64 * 32 * MT), lane, mw, nw);
                } else {
                    // 16 rows per wave: transposed rows of 32 bytes would waste the stores; the four waves put theirs side by side first
                    // (KG = 2: the second set does, in its own ring's LDS; both pass the barrier)
                    char *const T = smem + R::LDS / 2;                 // [64 n][64 m] fp16, rows of 128 bytes, 16-byte chunk c at c ^ (n & 7)
                    const int gq = lane >> 4, ml = lane & 15;
                    if (kg == KG - 1)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int n = 16 * j + 4 * gq + r, c = (2 * wave + (ml >> 3)) ^ (n & 7);
                            *(GNK_LDS _Float16 *)(GNK_LDS char *)(T + n * 128 + 16 * c + 2 * (ml & 7)) = (_Float16)acc[0][j][r];
                        }
                    __syncthreads();
                    if (kg == KG - 1)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int e = u * 256 + ((int)threadIdx.x & 255), n = e >> 3, c = e & 7;
                        const v4i v = *(const GNK_LDS v4i *)(const GNK_LDS char *)(T + n * 128 + 16 * (c ^ (n & 7)));
                        gnk_store16_out((char *)g.C + 2 * ((n0 + n) * p.N + m0) + 16 * c, v);
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------ 256 x 256 tiles, one wave per SIMD (gnk_gemm_w4.h)
// The 8-bit loop with 16-bit fragments: a 64-byte stage holds 32 k, so K must be a multiple of 128 (four stages per iteration).
// 8 x 2048 x 5632: the matrix pipes are busy 65 % (S), 50 % (Q, the shortest contraction) and 71 % (X) of the time.
template <bool KMAJOR> struct StagerW4H {
    const char *base;
    unsigned off[8];
    int64_t step;
    __device__ __forceinline__ void init(const char *ptr, int64_t ld, int64_t r0, int64_t extent, int wave, int lane) {
        base = KMAJOR ? ptr + r0 * ld : ptr + 2 * r0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int p = (i * 4 + wave) * 64 + lane;
            if constexpr (KMAJOR) {
                int r, c;
                gnk_kmaj_stage_src(p, r, c);
                const int64_t rmax = extent - 1 - r0, row = r < rmax ? r : rmax;
                off[i] = (unsigned)(row * ld + 16 * c);
            } else {
                int k, c;
                gnk_mn16_stage_src<512>(p & 1023, k, c);
                const int64_t cmax = 2 * (extent - r0) - 16, col = 16 * c < cmax ? 16 * c : cmax;
                off[i] = (unsigned)(k * ld + col);        // pieces 4-7 repeat 0-3 (unused)
            }
        }
        step = KMAJOR ? 128 : 32 * ld;
    }
};

template <int H, int I> __device__ __forceinline__ void fetch_row(v4f (&acc)[8][4]) {
    int r[16];
    w4_read16<8 * H + I>(r);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        acc[I][j] = (v4f){__int_as_float(r[4 * j]), __int_as_float(r[4 * j + 1]), __int_as_float(r[4 * j + 2]), __int_as_float(r[4 * j + 3])};
}

// columns 64 H .. 64 H + 63 of the wave tile: accumulators -> values -> memory
template <class Cfg, int EPI, int H, bool PAIRS>
__device__ __forceinline__ void finish_half(const Product &p, GemmParams g, int b, bool mirror, const Finish &fin, char *smem, int wave, int lane, int64_t mw, int64_t nw) {
    v4f acc[8][4];
    fetch_row<H, 0>(acc); fetch_row<H, 1>(acc); fetch_row<H, 2>(acc); fetch_row<H, 3>(acc);
    fetch_row<H, 4>(acc); fetch_row<H, 5>(acc); fetch_row<H, 6>(acc); fetch_row<H, 7>(acc);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) finish_value<EPI, PAIRS>(p, fin, acc[i][j], mw + 16 * i + (lane & 15), nw + 64 * H + 16 * j + 4 * (lane >> 4));
    // all through the same slice of LDS: a wave's accesses stay in order
    if constexpr (!PAIRS) {
        run_epilogue<Cfg>(g, acc, nullptr, smem, wave * 2 + H, lane, mw, nw + 64 * H);
        if (mirror) store_mirror<8>(p, (char *)g.C, acc, smem + (wave * 2 + H) * 16384, lane, mw, nw + 64 * H);
    } else {                                                                  // no mirror images here (choose_tile)
#pragma nounroll
        for (int part = 0; part < (p.c_lo ? 2 : 1); ++part) {                 // hi, then what it leaves; not unrolled: registers
            run_epilogue<Cfg>(g, acc, nullptr, smem, wave * 2 + H, lane, mw, nw + 64 * H);
            g.C = (char *)g.C + p.c_lo;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] -= (float)(_Float16)acc[i][j][r];
        }
    }
}

// PAIRS: the loop three times, the second and third on top of the first one's sums (lo hi, hi lo).
template <bool AK, bool BK, int EPI, bool SYM, bool PAIRS>
__global__ void __launch_bounds__(256) product256_kernel(const Product p) {
    static_assert(!PAIRS || (AK && !SYM), "with mirror images: too many registers");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef GemmCfg<256, 256, 2, 4, AK, BK, OP_F8, 0, 0, EPI_PLAIN> Cfg;      // the epilogue's maps: 128 x 64 halves of a wave's 128 x 128
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    int b, tm, tn;
    batch_tile<SYM>(p, b, tm, tn);
    const int64_t m0 = (int64_t)tm * 256, n0 = (int64_t)tn * 256;
    StagerW4H<AK> sa;
    StagerW4H<BK> sb;
    sa.init(p.A + b * p.ba, p.lda, m0, p.ext_a, wave, lane);
    sb.init(p.B + b * p.bb, p.ldb, n0, p.ext_b, wave, lane);
    const float diag = EPI == POLY ? diagonal_part<256>(p, b) : 0.0f;
    const unsigned lds0 = (unsigned)(uintptr_t)(GNK_LDS char *)smem;
    const unsigned va = lds0 + (AK ? gnk_kmaj_frag_offset(wm * 128, 0, lane) : gnk_mn16_frag_offset<512>(wm * 128, 0, lane));
    const unsigned vb = lds0 + 65536 + (BK ? gnk_kmaj_frag_offset(wn * 128, 0, lane) : gnk_mn16_frag_offset<512>(wn * 128, 0, lane));
    const auto low = [](const char *at) { return (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)at); };
    const auto high = [](const char *at) { return (unsigned)__builtin_amdgcn_readfirstlane((unsigned)((uintptr_t)at >> 32)); };
    const unsigned stepa = __builtin_amdgcn_readfirstlane((unsigned)sa.step), stepb = __builtin_amdgcn_readfirstlane((unsigned)sb.step);
    const unsigned ldsw = __builtin_amdgcn_readfirstlane(lds0 + wave * 1024);
    const int ns = (int)(p.K / 32);
    const int nit = __builtin_amdgcn_readfirstlane(ns >> 2), rem = __builtin_amdgcn_readfirstlane(ns - 1);
#define GNK_ORTHO_RUN(TEXT, A, B)                                                                                                     \
    asm volatile(TEXT : : [alo] "s"(low(A)), [ahi] "s"(high(A)), [blo] "s"(low(B)), [bhi] "s"(high(B)), [stepa] "s"(stepa), [stepb] "s"(stepb),      \
                 [lds] "s"(ldsw), [nit] "s"(nit), [rem] "s"(rem), [va] "v"(va), [vb] "v"(vb),                                         \
                 [oa0] "v"(sa.off[0]), [oa1] "v"(sa.off[1]), [oa2] "v"(sa.off[2]), [oa3] "v"(sa.off[3]),                              \
                 [oa4] "v"(sa.off[4]), [oa5] "v"(sa.off[5]), [oa6] "v"(sa.off[6]), [oa7] "v"(sa.off[7]),                              \
                 [ob0] "v"(sb.off[0]), [ob1] "v"(sb.off[1]), [ob2] "v"(sb.off[2]), [ob3] "v"(sb.off[3]),                              \
                 [ob4] "v"(sb.off[4]), [ob5] "v"(sb.off[5]), [ob6] "v"(sb.off[6]), [ob7] "v"(sb.off[7]) : GNK_W4_CLOBBERS)
    const char *const A = sa.base, *const B = sb.base;
    if constexpr (AK && BK) GNK_ORTHO_RUN(GNK_W4_ASM_F16_KK, A, B);
    else if constexpr (AK) GNK_ORTHO_RUN(GNK_W4_ASM_F16_KM, A, B);
    else GNK_ORTHO_RUN(GNK_W4_ASM_F16_MM, A, B);
    if constexpr (PAIRS) {
        const char *const Al = A + p.a_lo, *const Bl = B + p.b_lo;
        if constexpr (AK && BK) { GNK_ORTHO_RUN(GNK_W4_ASM_F16_KK_ADD, Al, B); GNK_ORTHO_RUN(GNK_W4_ASM_F16_KK_ADD, A, Bl); }
        else { GNK_ORTHO_RUN(GNK_W4_ASM_F16_KM_ADD, Al, B); GNK_ORTHO_RUN(GNK_W4_ASM_F16_KM_ADD, A, Bl); }
    }
#undef GNK_ORTHO_RUN
    // the asm ends behind vmcnt(0) + a barrier: LDS is free for the epilogue
    float diag_sum = 0.0f;
    if constexpr (EPI == POLY) diag_sum = workgroup_sum<256>(diag, smem);
    const Finish fin = make_finish<EPI>(p, b, tm == 0 && tn == 0, diag_sum);
    const GemmParams g = store_params(p, b);
    const int64_t mw = m0 + wm * 128, nw = n0 + wn * 128;
    const bool mirror = SYM && tm != tn;
    finish_half<Cfg, EPI, 0, PAIRS>(p, g, b, mirror, fin, smem, wave, lane, mw, nw);
    finish_half<Cfg, EPI, 1, PAIRS>(p, g, b, mirror, fin, smem, wave, lane, mw, nw);
}

// ------------------------------------------------------------------------------ sums of squares, conversion
// V consecutive elements as floats: one 16-byte load, or a single element
template <int DT, int V> __device__ __forceinline__ void load_floats(const void *p, int64_t i, float (&f)[V]) {
    if constexpr (V == 1) {
        f[0] = gnk_load_scalar<DT>(p, i);
    } else if constexpr (DT == GNK_F32) {
        const v4f v = *(const v4f *)((const float *)p + i);
        f[0] = v[0]; f[1] = v[1]; f[2] = v[2]; f[3] = v[3];
    } else {
        const v4i v = *(const v4i *)((const unsigned short *)p + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned w = (unsigned)v[k];
            f[2 * k] = gnk_raw_to_f32<DT>(w & 0xffffu);
            f[2 * k + 1] = gnk_raw_to_f32<DT>(w >> 16);
        }
    }
}
template <int DT> constexpr int VEC = DT == GNK_F32 ? 4 : 8;

// Partial sums of squares: HBM-bound (8 x 2048 x 5632 bf16: 38 us, 4.8 TB/s).  fp64: the squares of any fp32 fit, and nothing is lost on the way.
template <int DT, int V>
__global__ void __launch_bounds__(256) square_sum_kernel(const void *__restrict__ G, double *__restrict__ parts, int64_t numel, int nparts) {
    const int64_t b = blockIdx.y, words = numel / V, per = (words + nparts - 1) / nparts, i0 = (int64_t)blockIdx.x * per, i1 = i0 + per < words ? i0 + per : words;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t i = i0 + threadIdx.x; i < i1; i += 256 * 4) {
        float f[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) {                                 // four loads in flight; past the end zeros
#pragma unroll
            for (int k = 0; k < V; ++k) f[u][k] = 0.0f;
            if (i + 256 * u < i1) load_floats<DT, V>(G, b * numel + (i + 256 * u) * V, f[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int k = 0; k < V; ++k) s[u] = fma((double)f[u][k], (double)f[u][k], s[u]);
    }
    double t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d, 64);
    __shared__ double red[4];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
    __syncthreads();
    if (threadIdx.x == 0) parts[b * nparts + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// G 2^p as fp16 (PAIRS: and what that leaves, x_lo bytes behind), padded; fac[b] = {factor of step 0's S, factor of step 0's update}: what takes G 2^p back to X_0.  HBM-bound (8 x 2048 x 5632
// bf16: 59 us, 6.3 TB/s; most of G is still in the last-level cache).
template <int DT, int V>
__global__ void __launch_bounds__(256) convert_kernel(const void *__restrict__ G, unsigned short *__restrict__ X, int64_t x_lo, const double *__restrict__ parts, float *__restrict__ fac,
                                                      int64_t rows, int64_t cols, int64_t rows_p, int64_t cols_p, int nparts, float eps) {
    const int64_t b = blockIdx.y;
    __shared__ double total;
    if (threadIdx.x < 64) {                                           // every block adds in the same order
        double t = 0.0;
        for (int k = threadIdx.x; k < nparts; k += 64) t += parts[b * nparts + k];
#pragma unroll
        for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d, 64);
        if (threadIdx.x == 0) total = t;
    }
    __syncthreads();
    const double norm = sqrt(total);
    int p = 0;
    double inv = 1.0 / (norm > (double)eps ? norm : (double)eps);
    const bool finite = norm < 1.0e300;                                // false for NaN and Inf: every output becomes NaN through the factors
    if (finite && norm > 0.0) p = 14 - ilogb(norm);
    if (!finite) inv = __builtin_nan("");
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const double x0 = ldexp(inv, -p);
        fac[2 * b] = (float)(x0 * x0);
        fac[2 * b + 1] = (float)x0;
    }
    const int64_t per_row = cols_p / 8, octets = rows_p * per_row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < octets; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per_row, c = (i - r * per_row) * 8;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.0f;
        if (finite && r < rows && c < cols) {
            const int64_t at = (b * rows + r) * cols + c;
            if constexpr (V > 1) {                                     // cols is a multiple of V
#pragma unroll
                for (int h = 0; h < 8 / V; ++h) {
                    if (c + h * V < cols) {
                        float w[V];
                        load_floats<DT, V>(G, at + h * V, w);
#pragma unroll
                        for (int k = 0; k < V; ++k) v[h * V + k] = w[k];
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (c + k < cols) v[k] = gnk_load_scalar<DT>(G, at + k);
            }
        }
        v4i o;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], p);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = (int)gnk_pack2_f16(v[2 * k], v[2 * k + 1]);
        char *const dst = (char *)(X + (b * rows_p + r) * cols_p + c);
        *(v4i *)dst = o;
        if (x_lo) {                                                    // PAIRS
#pragma unroll
            for (int k = 0; k < 4; ++k)
                o[k] = (int)gnk_pack2_f16(v[2 * k] - (float)(_Float16)v[2 * k], v[2 * k + 1] - (float)(_Float16)v[2 * k + 1]);
            *(v4i *)(dst + x_lo) = o;
        }
    }
}

template <int BM, int KG, bool AK, bool BK, int EPI, bool SYM, bool PAIRS = false> int launch(const Product &p0, hipStream_t st) {
    constexpr int LDS_TOTAL = BM == 256 ? 131072 : KG * RingShape<BM == 256 ? 128 : BM, KG>::LDS;
    void (*kernel)(const Product);
    if constexpr (BM == 256) kernel = product256_kernel<AK, BK, EPI, SYM, PAIRS>;
    else kernel = product_ring_kernel<BM, KG, AK, BK, EPI, SYM, PAIRS>;
    Product p = p0;
    p.grid_m = (int)((p.ext_a + BM - 1) / BM);
    p.grid_n = (int)((p.ext_b + BM - 1) / BM);
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return gnk_fail(GNK_ERR_LAUNCH, "orthogonalize: no current HIP device");
    if (!attr_set[dev].load(std::memory_order_acquire)) {
        if (hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_TOTAL) != hipSuccess)
            return gnk_fail(GNK_ERR_LAUNCH, "orthogonalize: cannot reserve LDS");
        attr_set[dev].store(true, std::memory_order_release);
    }
    const int64_t blocks = (int64_t)tiles_of<SYM>(p) * p.batch;
    if (blocks >= (1LL << 31)) return gnk_fail(GNK_ERR_UNSUPPORTED, "orthogonalize: too many tiles");
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256 * KG), LDS_TOTAL, st, p);
    return gnk_check_launch("orthogonalize");
}

int64_t up(int64_t v) { return (v + PAD - 1) / PAD * PAD; }

struct Plan {
    int64_t rp, cp, lo;                      // padded rows, columns, and the smaller of them
    int64_t x_bytes, s_bytes;                // one matrix
    int nparts;
    int64_t off_x0, off_x1, off_s, off_q, off_parts, off_fac, off_mu, total;
    int64_t lo_part;                         // pairs: bytes from a matrix's hi part to its lo part, 0 without
};

// Results of more than bf16's 8 bits: matrices in two parts
bool wants_pairs(int out_dtype) { return out_dtype != GNK_BF16; }

Plan make_plan(int64_t batch, int64_t rows, int64_t cols, bool pairs) {
    Plan p;
    p.rp = up(rows); p.cp = up(cols);
    p.lo = rows <= cols ? p.rp : p.cp;
    p.x_bytes = 2 * p.rp * p.cp;
    p.s_bytes = 2 * p.lo * p.lo;
    const int64_t want = (rows * cols + 4095) / 4096;
    p.nparts = (int)(want < MAX_PARTS ? (want > 0 ? want : 1) : MAX_PARTS);
    p.off_x0 = 0;
    p.off_x1 = p.off_x0 + batch * p.x_bytes;
    p.off_s = p.off_x1 + batch * p.x_bytes;
    p.off_q = p.off_s + batch * p.s_bytes;
    p.lo_part = pairs ? p.off_q + batch * p.s_bytes : 0;
    p.off_parts = p.off_q + batch * p.s_bytes + p.lo_part;
    p.off_fac = p.off_parts + (batch * p.nparts * 8 + 15) / 16 * 16;
    p.off_mu = p.off_fac + (batch * 8 + 15) / 16 * 16;
    p.total = p.off_mu + (batch * 4 + 15) / 16 * 16;
    return p;
}

// Tile size of a product over `batch` matrices, and its time by the cost model of the dense products (gnk_api.hip: us per round of workgroups, one
// 256 x 256 or two smaller ones per CU; a step is 64 k) with whole rounds and without (what is left where another launch fills the last one).
struct Choice { int bm, kg; double rounds_us, work_us; };
Choice choose_tile(int64_t ext_a, int64_t ext_b, int64_t K, bool sym, int64_t batch, bool pairs) {
    const double cus = (double)gnk_num_cus(), ks = (double)K / 64.0 * (pairs ? 3.0 : 1.0);
    auto tiles = [&](int64_t bm) {
        const double gm = (double)((ext_a + bm - 1) / bm), gn = (double)((ext_b + bm - 1) / bm);
        return (sym ? gm * (gm + 1) / 2 : gm * gn) * (double)batch;
    };
    auto priced = [&](int bm, int kg, double slots, double per) { return Choice{bm, kg, ceil(tiles(bm) / slots) * per, tiles(bm) / slots * per}; };
    Choice c256 = priced(256, 1, cus, (pairs ? 20.0 : 12.0) + 1.3 * ks);      // pairs: three loops' first loads, two stores
    // hi, lo and both mirror images together take more registers than the accumulators leave: the compiler would put values into those that are not read yet
    const bool can256 = !(pairs && sym);
    if (!can256) c256.rounds_us = 1e30;
    const Choice c128 = tiles(128) <= cus && ks >= 4.0 ? priced(128, 2, cus, 7.0 + 0.55 * ks) : priced(128, 1, 2.0 * cus, 6.0 + 1.0 * ks);
    const int kg = tiles(64) <= cus ? (ks >= 24.0 ? 4 : ks >= 4.0 ? 2 : 1) : 1;
    const Choice c64 = priced(64, kg, 2.0 * cus, 4.0 + (kg == 4 ? 0.2 : kg == 2 ? 0.3 : 0.5) * ks);
    const int forced = gnk_forced_variant_get();      // gnk_set_gemm_variant: 1, 5 and 6 force the 128, 256 and 64 tiles here as well
    if (forced == 6 || (forced != 1 && forced != 5 && c64.rounds_us <= c128.rounds_us && c64.rounds_us <= c256.rounds_us)) return c64;
    if (can256 && (forced == 5 || (forced != 1 && c256.rounds_us <= c128.rounds_us))) return c256;
    return c128;
}

// The tiles of a step's three products, chosen for the whole stack however it is split: the results do not depend on the split.  `two`: as two chains of half
// the stack each, where that is worth the second stream: large products (below B m^2 n = 1e11 two short chains get in each other's way: 8 x 1024 x 4096 734 us
// alone, 966 us as two) whose last rounds are partly empty.  8 x 2048 x 5632: 3.35 -> 2.89 ms, 2 x 4096 x 4096: 2.84 -> 2.36.
struct Schedule { Choice gram, poly, next; bool two; };
Schedule make_schedule(const Plan &pl, int64_t batch, int64_t rows, int64_t cols, bool pairs) {
    Schedule s;
    s.gram = choose_tile(pl.lo, pl.lo, rows <= cols ? pl.cp : pl.rp, true, batch, pairs);
    s.poly = choose_tile(pl.lo, pl.lo, pl.lo, true, batch, pairs);
    s.next = choose_tile(pl.rp, pl.cp, pl.lo, false, batch, pairs);
    const double rounds = s.gram.rounds_us + s.poly.rounds_us + s.next.rounds_us, work = s.gram.work_us + s.poly.work_us + s.next.work_us;
    s.two = batch > 1 && (double)batch * (double)pl.lo * (double)pl.rp * (double)pl.cp >= 1.0e11 && work <= 0.9 * rounds;
    return s;
}

template <bool AK, bool BK, int EPI, bool SYM> int run_product(const Product &p, const Choice &c, hipStream_t st) {
    if (c.bm == 256) return launch<256, 1, AK, BK, EPI, SYM>(p, st);
    if (c.bm == 128) return c.kg == 2 ? launch<128, 2, AK, BK, EPI, SYM>(p, st) : launch<128, 1, AK, BK, EPI, SYM>(p, st);
    if (c.kg == 4) return launch<64, 4, AK, BK, EPI, SYM>(p, st);
    if (c.kg == 2) return launch<64, 2, AK, BK, EPI, SYM>(p, st);
    return launch<64, 1, AK, BK, EPI, SYM>(p, st);
}

template <bool AK, bool BK, int EPI, bool SYM> int run_pairs(const Product &p, const Choice &c, hipStream_t st) {
    if constexpr (!SYM)
        if (c.bm == 256) return launch<256, 1, AK, BK, EPI, SYM, true>(p, st);
    if (c.bm == 128) return c.kg == 2 ? launch<128, 2, AK, BK, EPI, SYM, true>(p, st) : launch<128, 1, AK, BK, EPI, SYM, true>(p, st);
    if (c.kg == 4) return launch<64, 4, AK, BK, EPI, SYM, true>(p, st);
    return c.kg == 2 ? launch<64, 2, AK, BK, EPI, SYM, true>(p, st) : launch<64, 1, AK, BK, EPI, SYM, true>(p, st);
}

template <int DT> int read_input(const void *G, char *X, double *parts, float *fac, int64_t batch, int64_t rows, int64_t cols, const Plan &pl, float eps, hipStream_t st) {
    const dim3 g1((unsigned)pl.nparts, (unsigned)batch);
    const int64_t octets = pl.rp * pl.cp / 8, want = (octets + 255) / 256;
    const dim3 g2((unsigned)(want < 1024 ? want : 1024), (unsigned)batch);
    if (cols % VEC<DT> == 0 && ((uintptr_t)G & 15) == 0) {
        hipLaunchKernelGGL((square_sum_kernel<DT, VEC<DT>>), g1, dim3(256), 0, st, G, parts, rows * cols, pl.nparts);
        hipLaunchKernelGGL((convert_kernel<DT, VEC<DT>>), g2, dim3(256), 0, st, G, (unsigned short *)X, pl.lo_part, parts, fac, rows, cols, pl.rp, pl.cp, pl.nparts, eps);
    } else {
        hipLaunchKernelGGL((square_sum_kernel<DT, 1>), g1, dim3(256), 0, st, G, parts, rows * cols, pl.nparts);
        hipLaunchKernelGGL((convert_kernel<DT, 1>), g2, dim3(256), 0, st, G, (unsigned short *)X, pl.lo_part, parts, fac, rows, cols, pl.rp, pl.cp, pl.nparts, eps);
    }
    return gnk_check_launch("orthogonalize");
}

// A second stream for half of a stack.  Its products depend on nothing of the other half, so the two chains fill each other's last, partly empty rounds of
// workgroups.  One stream per device, made on first use and kept; calls that overlap only queue behind each other on it.  Not used while the caller's
// stream is being captured (fork() then says no): a captured stream must not be shared.
struct SideStream {
    hipStream_t stream = nullptr;
    hipEvent_t ev = nullptr;
    bool fork(hipStream_t st) {
        hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(st, &cs) != hipSuccess || cs != hipStreamCaptureStatusNone) {
            (void)hipGetLastError();
            return false;
        }
        static std::atomic<hipStream_t> made[64];
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return false;
        stream = made[dev].load(std::memory_order_acquire);
        if (!stream) {
            hipStream_t fresh = nullptr, none = nullptr;
            if (hipStreamCreateWithFlags(&fresh, hipStreamNonBlocking) != hipSuccess) return false;
            if (made[dev].compare_exchange_strong(none, fresh)) stream = fresh;
            else {
                (void)hipStreamDestroy(fresh);
                stream = none;
            }
        }
        if (hipEventCreateWithFlags(&ev, hipEventDisableTiming) != hipSuccess) return false;
        if (hipEventRecord(ev, st) == hipSuccess && hipStreamWaitEvent(stream, ev, 0) == hipSuccess) return true;
        (void)hipEventDestroy(ev);
        return false;
    }
    int join(hipStream_t st) {
        const bool ok = hipEventRecord(ev, stream) == hipSuccess && hipStreamWaitEvent(st, ev, 0) == hipSuccess;
        (void)hipEventDestroy(ev);               // released by the runtime once it has completed
        if (ok) return GNK_OK;
        (void)hipStreamSynchronize(stream);      // never hand the workspace back with work in flight on it
        return gnk_fail(GNK_ERR_LAUNCH, "orthogonalize: cannot join the second stream");
    }
};

}  // namespace

extern "C" int64_t gnk_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    return make_plan(batch, rows, cols, true).total;
}

extern "C" int64_t gnk_orthogonalize_workspace_bytes_of(int out_dtype, int64_t batch, int64_t rows, int64_t cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    return make_plan(batch, rows, cols, wants_pairs(out_dtype)).total;
}

extern "C" int gnk_orthogonalize_chains(int out_dtype, int64_t batch, int64_t rows, int64_t cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    const bool pairs = wants_pairs(out_dtype);
    return make_schedule(make_plan(batch, rows, cols, pairs), batch, rows, cols, pairs).two ? 2 : 1;
}

extern "C" int gnk_orthogonalize(const void *G, int g_dtype, void *out, int out_dtype, int64_t batch, int64_t rows, int64_t cols, int steps, float a, float b, float c,
                                 float eps, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *name = "orthogonalize";
    if (batch < 0 || rows < 0 || cols < 0) return gnk_fail(GNK_ERR_BAD_ARG, "%s: negative dimension", name);
    if (!gnk_is_float_dtype(g_dtype) || !gnk_is_float_dtype(out_dtype)) return gnk_fail(GNK_ERR_BAD_ARG, "%s: dtype codes %d, %d are not bf16/f16/f32", name, g_dtype, out_dtype);
    if (steps < 1 || steps > 100) return gnk_fail(GNK_ERR_BAD_ARG, "%s: %d steps", name, steps);
    const float cmax = fabsf(a) + 2.0f * fabsf(b) + 4.0f * fabsf(c);
    if (!(cmax < 1.0e4f) || !(eps >= 0.0f)) return gnk_fail(GNK_ERR_BAD_ARG, "%s: coefficients (%g, %g, %g), eps %g", name, a, b, c, eps);
    if (batch > 65535 || rows > (1 << 20) || cols > (1 << 20)) return gnk_fail(GNK_ERR_UNSUPPORTED, "%s: %lld matrices of %lld x %lld", name, (long long)batch, (long long)rows, (long long)cols);
    if (batch == 0 || rows == 0 || cols == 0) return GNK_OK;
    if (!G || !out) return gnk_fail(GNK_ERR_BAD_ARG, "%s: null pointer", name);
    const bool pairs = wants_pairs(out_dtype);
    const Plan pl = make_plan(batch, rows, cols, pairs);
    if (!workspace || workspace_bytes < pl.total || ((uintptr_t)workspace & 15) != 0)
        return gnk_fail(GNK_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %lld bytes", name, (long long)pl.total);
    int rc = gnk_init();
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    char *const ws = (char *)workspace;
    double *const parts = (double *)(ws + pl.off_parts);
    float *const fac = (float *)(ws + pl.off_fac);
    char *const X0 = ws + pl.off_x0, *const X1 = ws + pl.off_x1;
    char *const S_all = ws + pl.off_s, *const Q_all = ws + pl.off_q;
    rc = g_dtype == GNK_BF16 ? read_input<GNK_BF16>(G, X0, parts, fac, batch, rows, cols, pl, eps, st)
         : g_dtype == GNK_F16 ? read_input<GNK_F16>(G, X0, parts, fac, batch, rows, cols, pl, eps, st)
                              : read_input<GNK_F32>(G, X0, parts, fac, batch, rows, cols, pl, eps, st);
    if (rc) return rc;

    const bool wide = rows <= cols;
    float sq = 32768.0f;                     // scale of Q - mu I: |Q|, |mu| <= |a| + 2 |b| + 4 |c| while the singular values stay below sqrt 2
    while (sq * cmax >= 16384.0f) sq *= 0.5f;
    const bool with_mu = !pairs && (wide ? rows : cols) < MU_ROWS;
    const int64_t lo = pl.lo, ldx = 2 * pl.cp, lds = 2 * lo;
    const Schedule plan = make_schedule(pl, batch, rows, cols, pairs);
    const Choice c_gram = plan.gram, c_poly = plan.poly, c_next = plan.next;
    // one step of matrices b0 .. b0 + n - 1 on stream s
    auto one_step = [&](int it, int64_t b0, int64_t n, hipStream_t s) -> int {
        const bool last = it + 1 == steps;
        char *const X = (it & 1 ? X1 : X0) + b0 * pl.x_bytes, *const Xn = (it & 1 ? X0 : X1) + b0 * pl.x_bytes;
        char *const S = S_all + b0 * pl.s_bytes, *const Q = Q_all + b0 * pl.s_bytes;
        Product p;
        memset(&p, 0, sizeof(p));
        p.batch = (int)n;
        p.fstride = 2;
        p.a_lo = p.b_lo = p.c_lo = p.d_lo = pl.lo_part;
        p.mu = with_mu ? (float *)(ws + pl.off_mu) + b0 : nullptr;
        // S
        p.A = p.B = X; p.ba = p.bb = pl.x_bytes; p.lda = p.ldb = ldx;
        p.C = S; p.bc = pl.s_bytes;
        p.M = p.N = p.ext_a = p.ext_b = lo;
        p.K = wide ? pl.cp : pl.rp;
        p.f = it == 0 ? SS : SS / (SX * SX);
        p.fdev = it == 0 ? fac + 2 * b0 : nullptr;
        p.out_dtype = GNK_F16;
        p.parts = it == 0 && g_dtype != GNK_F32 ? 1 : 3;                       // X_0 of 16-bit inputs is exact
        int rc = pairs  ? (wide ? run_pairs<true, true, GRAM, true>(p, c_gram, s) : run_pairs<false, false, GRAM, true>(p, c_gram, s))
                 : wide ? run_product<true, true, GRAM, true>(p, c_gram, s)
                        : run_product<false, false, GRAM, true>(p, c_gram, s);
        if (rc) return rc;
        p.parts = 3;
        // Q - mu I = (a - mu) I + b S + c S^2
        p.A = p.B = S; p.ba = p.bb = pl.s_bytes; p.lda = p.ldb = lds;
        p.C = Q; p.bc = pl.s_bytes;
        p.D = S; p.bd = pl.s_bytes; p.ldd = lds;
        p.K = lo;
        p.f = c * sq / (SS * SS); p.g = b * sq / SS; p.h = a; p.k = sq;
        p.c0 = a; p.c1 = b; p.c2 = c; p.diag_scale = 1.0f / (SS * (float)(wide ? rows : cols));
        p.fdev = nullptr;
        rc = pairs ? run_pairs<true, true, POLY, true>(p, c_poly, s) : run_product<true, true, POLY, true>(p, c_poly, s);
        if (rc) return rc;
        // X <- Q X or X Q: the product with Q - mu I, and mu X
        p.A = wide ? Q : X; p.ba = wide ? pl.s_bytes : pl.x_bytes; p.lda = wide ? lds : ldx;
        p.B = wide ? X : Q; p.bb = wide ? pl.x_bytes : pl.s_bytes; p.ldb = wide ? ldx : lds;
        p.bc = last ? rows * cols * gnk_dtype_size(out_dtype) : pl.x_bytes;
        p.C = last ? (char *)out + b0 * p.bc : Xn;
        p.ext_a = pl.rp; p.ext_b = pl.cp;
        p.M = last ? rows : pl.rp; p.N = last ? cols : pl.cp;
        p.D = X; p.bd = pl.x_bytes; p.ldd = ldx; p.k = sq;
        p.K = lo;
        p.out_dtype = last ? out_dtype : GNK_F16;
        p.f = (last ? 1.0f : SX) / (it == 0 ? sq : sq * SX);
        p.fdev = it == 0 ? fac + 2 * b0 + 1 : nullptr;
        if (last) p.c_lo = 0;
        if (pairs) return wide ? run_pairs<true, false, GRAM, false>(p, c_next, s) : run_pairs<true, true, GRAM, false>(p, c_next, s);
        if (with_mu) return wide ? run_product<true, false, UPDATE, false>(p, c_next, s) : run_product<true, true, UPDATE, false>(p, c_next, s);
        return wide ? run_product<true, false, GRAM, false>(p, c_next, s) : run_product<true, true, GRAM, false>(p, c_next, s);
    };
    SideStream side;
    const bool two = plan.two && side.fork(st);
    const int64_t half = two ? batch / 2 : batch;
    for (int it = 0; it < steps && !rc; ++it) {
        rc = one_step(it, 0, half, st);
        if (two && !rc) rc = one_step(it, half, batch - half, side.stream);
    }
    if (two) {
        const int joined = side.join(st);
        if (!rc) rc = joined;
    }
    return rc;
}
