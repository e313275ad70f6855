// gnk_grouped.hip -- entry points of the products grouped by expert (gnk_grouped.h) and the quantizer in front of their weight gradients.
#include "gnk_grouped.h"

#include <string.h>

namespace {

using namespace gnk_grouped;

// ------------------------------------------------------------------------------ operands the LDS-DMA cannot take
// The kernels read 16-byte chunks: rows form wants A K-contiguous and B K- or N-contiguous, depth form both row (t) by row, always with
// 16-byte aligned pitches and a contiguous extent that is a multiple of 16.  Anything else is copied once into the caller's workspace:
// dst[g][r][c] = src[g sg + r sr + c sc], c padded with zeros up to `cp`.  HBM-bound; 16 bytes per thread:
// 16384 x 2048 bytes from an odd pitch 12 us, 5.4 TB/s; transposed 19 us, 3.5 TB/s.
__global__ void __launch_bounds__(256)
repack_kernel(const char *__restrict__ src, char *__restrict__ dst, int64_t R, int64_t C, int64_t cp, int64_t sg, int64_t sr, int64_t sc, int64_t chunks) {
    const int64_t per_row = cp / 16;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        // neighbouring threads take neighbouring bytes of the source where it is contiguous
        const int64_t grp = i / (R * per_row), in = i - grp * (R * per_row);
        const int64_t r = sc == 1 ? in / per_row : in % R, ch = sc == 1 ? in - r * per_row : in / R;
        const char *s = src + grp * sg + r * sr + 16 * ch * sc;
        const int64_t left = C - 16 * ch;
        v4i v = {0, 0, 0, 0};
        if (sc == 1 && left >= 16) {
            __builtin_memcpy(&v, s, 16);
        } else {
            unsigned char b[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) b[k] = k < left ? (unsigned char)s[k * sc] : 0;
            __builtin_memcpy(&v, b, 16);
        }
        *(v4i *)(dst + (grp * R + r) * cp + 16 * ch) = v;
    }
}

int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }

// One operand as the kernels want it: G groups of R rows of C contiguous bytes at `pitch`.
struct Staged {
    bool copy;
    int64_t G, R, C, sg, sr, sc;      // the source
    int64_t bytes() const { return copy ? G * R * up16(C) : 0; }
    int64_t pitch() const { return copy || R == 1 ? up16(C) : sr; }
    int64_t group() const { return copy ? R * up16(C) : (G == 1 ? 0 : sg); }
};

constexpr int64_t MAX_PITCH = 1LL << 22;      // 256 rows of a tile stay within 32-bit offsets

Staged stage(const void *ptr, int64_t G, int64_t R, int64_t C, int64_t sg, int64_t sr, int64_t sc) {
    Staged s = {true, G, R, C, sg, sr, sc};
    if (C == 1) s.sc = sc = 1;
    s.copy = !(((uintptr_t)ptr & 15) == 0 && sc == 1 && C % 16 == 0 && (R == 1 || (sr >= C && sr % 16 == 0 && sr <= MAX_PITCH)) &&
               (G == 1 || sg % 16 == 0));
    return s;
}

const char *repack(const Staged &s, const void *src, char *&ws, hipStream_t st, int &rc) {
    if (!s.copy) return (const char *)src;
    char *dst = ws;
    ws += s.bytes();
    const int64_t chunks = s.G * s.R * (up16(s.C) / 16);
    if (chunks > 0) {
        const int64_t want = (chunks + 255) / 256, cap = (int64_t)gnk_num_cus() * 32;
        hipLaunchKernelGGL(repack_kernel, dim3((unsigned)(want < cap ? want : cap)), dim3(256), 0, st, (const char *)src, dst, s.R, s.C, up16(s.C),
                           s.sg, s.sr, s.sc, chunks);
        rc = gnk_check_launch("grouped mm: operand copy");
    }
    return dst;
}

struct RowsPlan { Staged a, b; bool b_kmajor; };
struct DepthPlan { Staged a, b; };

RowsPlan plan_rows(const void *A, const void *B, int64_t T, int64_t E, int64_t N, int64_t K, int64_t sat, int64_t sak, int64_t sbe, int64_t sbk, int64_t sbn) {
    RowsPlan p;
    p.a = stage(A, 1, T, K, 0, sat, sak);
    // B as it lies, K- or N-contiguous; K-contiguous where it is neither (or both: a single column or row)
    const Staged bk = stage(B, E, N, K, sbe, sbn, sbk), bn = stage(B, E, K, N, sbe, sbk, sbn);
    p.b_kmajor = !bk.copy || (bn.copy && !(sbn == 1 && sbk != 1));
    p.b = p.b_kmajor ? bk : bn;
    return p;
}

DepthPlan plan_depth(const void *A, const void *B, int64_t T, int64_t M, int64_t N, int64_t sam, int64_t sat, int64_t sbt, int64_t sbn) {
    return {stage(A, 1, T, M, 0, sat, sam), stage(B, 1, T, N, 0, sbt, sbn)};
}

int check_call(const char *name, int a_dtype, int b_dtype, int out_dtype, int scale_dtype, int64_t T, int64_t E, int64_t d0, int64_t d1) {
    if (T < 0 || E < 0 || d0 < 0 || d1 < 0) return gnk_fail(GNK_ERR_BAD_ARG, "%s: negative dimension", name);
    if (T >= (1LL << 31)) return gnk_fail(GNK_ERR_UNSUPPORTED, "%s: group ends are 32-bit, %lld rows are too many", name, (long long)T);
    if (E >= (1LL << 20)) return gnk_fail(GNK_ERR_UNSUPPORTED, "%s: %lld groups are too many", name, (long long)E);
    if (d0 > MAX_PITCH || d1 > MAX_PITCH) return gnk_fail(GNK_ERR_UNSUPPORTED, "%s: feature sizes beyond %lld are not supported", name, (long long)MAX_PITCH);
    if ((double)(E > 0 ? E : 1) * (double)up16(d0) * (double)up16(d1) > 4.0e18)      // what a copy of the operands would take, in 64 bits
        return gnk_fail(GNK_ERR_UNSUPPORTED, "%s: %lld groups of %lld x %lld are too many", name, (long long)E, (long long)d0, (long long)d1);
    const bool i8 = a_dtype == GNK_I8 && b_dtype == GNK_I8, f8 = gnk_is_f8(a_dtype) && gnk_is_f8(b_dtype);
    if (!i8 && !f8) return gnk_fail(GNK_ERR_BAD_ARG, "%s: operands must be both int8 or both fp8 (got dtype codes %d, %d)", name, a_dtype, b_dtype);
    if (!gnk_is_float_dtype(scale_dtype)) return gnk_fail(GNK_ERR_BAD_ARG, "%s: scale dtype code %d is not bf16/f16/f32", name, scale_dtype);
    if (!gnk_is_float_dtype(out_dtype)) return gnk_fail(GNK_ERR_BAD_ARG, "%s: output dtype code %d is not bf16/f16/f32", name, out_dtype);
    return GNK_OK;
}

gnk_grouped_launcher pick(int a_dtype, int b_dtype) {
    if (a_dtype == GNK_I8) return gnk_grouped_i8;
    static const gnk_grouped_launcher f8[2][2] = {{gnk_grouped_f8_00, gnk_grouped_f8_01}, {gnk_grouped_f8_10, gnk_grouped_f8_11}};
    return f8[a_dtype == GNK_E5M2][b_dtype == GNK_E5M2];
}

int take_workspace(const char *name, const Staged &a, const Staged &b, void *ws, int64_t ws_bytes) {
    const int64_t need = a.bytes() + b.bytes();
    if (need == 0) return GNK_OK;
    if (!ws || ws_bytes < need || ((uintptr_t)ws & 15) != 0)
        return gnk_fail(GNK_ERR_WORKSPACE, "%s: these strides need a 16-byte aligned workspace of %lld bytes", name, (long long)need);
    return GNK_OK;
}

}  // namespace

extern "C" int64_t gnk_grouped_scaled_mm_rows_workspace_bytes(const void *A, const void *B, int64_t T, int64_t E, int64_t N, int64_t K, int64_t sat,
                                                              int64_t sak, int64_t sbe, int64_t sbk, int64_t sbn) {
    if (T <= 0 || E <= 0 || N <= 0 || K <= 0) return 0;
    const RowsPlan p = plan_rows(A, B, T, E, N, K, sat, sak, sbe, sbk, sbn);
    return p.a.bytes() + p.b.bytes();
}

extern "C" int gnk_grouped_scaled_mm_rows(const void *A, int a_dtype, const void *B, int b_dtype, void *C, int out_dtype, const void *row_scale,
                                          const void *col_scale, int scale_dtype, int col_scale_is_scalar, const int32_t *ends, int64_t T, int64_t E,
                                          int64_t N, int64_t K, int64_t sat, int64_t sak, int64_t sbe, int64_t sbk, int64_t sbn, void *workspace,
                                          int64_t workspace_bytes, void *stream) {
    const char *name = "grouped_scaled_mm";
    int rc = check_call(name, a_dtype, b_dtype, out_dtype, scale_dtype, T, E, N, K);
    if (rc) return rc;
    if (a_dtype == GNK_I8 && K > INT8_TERMS)
        return gnk_fail(GNK_ERR_UNSUPPORTED, "%s: int8 sums over %lld products may not fit 32 bits (at most %lld)", name, (long long)K, (long long)INT8_TERMS);
    if (T == 0 || N == 0) return GNK_OK;
    if (!C || !row_scale || (E > 0 && (!ends || !col_scale || (K > 0 && (!A || !B))))) return gnk_fail(GNK_ERR_BAD_ARG, "%s: null pointer", name);
    rc = gnk_init();
    if (rc) return rc;
    if (E == 0) K = 0;                       // no group: zeros, nothing is read
    const RowsPlan plan = plan_rows(A, B, T, E, N, K, sat, sak, sbe, sbk, sbn);
    rc = take_workspace(name, plan.a, plan.b, workspace, workspace_bytes);
    if (rc) return rc;
    char *ws = (char *)workspace;
    hipStream_t st = (hipStream_t)stream;
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.g.A = repack(plan.a, A, ws, st, rc);
    if (rc) return rc;
    p.g.B = repack(plan.b, B, ws, st, rc);
    if (rc) return rc;
    p.g.C = C; p.g.s0 = row_scale; p.g.s1 = col_scale; p.g.N = N; p.g.K = K;
    p.g.lda = plan.a.pitch(); p.g.ldb = plan.b.pitch();
    p.g.out_dtype = out_dtype; p.g.scale_dtype = scale_dtype; p.g.col_scalar = col_scale_is_scalar != 0;
    p.ends = ends; p.T = T; p.E = E; p.b_group = plan.b.group();
    p.ext_b = plan.b_kmajor ? N : up16(N);
    p.out_bytes = gnk_dtype_size(out_dtype); p.scale_bytes = gnk_dtype_size(scale_dtype);
    return pick(a_dtype, b_dtype)(false, plan.b_kmajor, p, st);
}

extern "C" int64_t gnk_grouped_scaled_mm_depth_workspace_bytes(const void *A, const void *B, int64_t T, int64_t M, int64_t N, int64_t sam, int64_t sat,
                                                               int64_t sbt, int64_t sbn) {
    if (T <= 0 || M <= 0 || N <= 0) return 0;
    const DepthPlan p = plan_depth(A, B, T, M, N, sam, sat, sbt, sbn);
    return p.a.bytes() + p.b.bytes();
}

extern "C" int64_t gnk_grouped_scaled_mm_depth_split_bytes(int64_t T, int64_t E, int64_t M, int64_t N) {
    if (T <= 0 || E <= 0 || M <= 0 || N <= 0 || E >= (1LL << 20) || M > MAX_PITCH || N > MAX_PITCH) return 0;
    const int64_t pitch = up16(M > N ? M : N);
    const int f = gnk_forced_variant_get(), forced = f == GNK_VARIANT_128 || f == GNK_VARIANT_64X128 || (f == GNK_VARIANT_256_W4 && T * pitch < (1LL << 32)) ? f : -1;
    const int64_t parts = split_bytes(choose_variant(T, E, M, N, 0, true, false, T * pitch < (1LL << 32), false, forced).splits, E, M, N);
    const int64_t long_groups = T > LONG_ROWS ? most_long_pieces(T) * M * N * 4 : 0;
    return parts > long_groups ? parts : long_groups;
}

extern "C" int gnk_grouped_scaled_mm_depth(const void *A, int a_dtype, const void *B, int b_dtype, void *C, int out_dtype, const void *row_scale,
                                           const void *col_scale, int scale_dtype, int col_scale_is_scalar, const int32_t *ends, int64_t T, int64_t E,
                                           int64_t M, int64_t N, int64_t sam, int64_t sat, int64_t sbt, int64_t sbn, void *workspace,
                                           int64_t workspace_bytes, void *stream) {
    const char *name = "grouped_scaled_mm";
    int rc = check_call(name, a_dtype, b_dtype, out_dtype, scale_dtype, T, E, M, N);
    if (rc) return rc;
    if (E == 0 || M == 0 || N == 0) return GNK_OK;
    if (!C || !row_scale || !col_scale || !ends || (T > 0 && (!A || !B))) return gnk_fail(GNK_ERR_BAD_ARG, "%s: null pointer", name);
    rc = gnk_init();
    if (rc) return rc;
    const DepthPlan plan = plan_depth(A, B, T, M, N, sam, sat, sbt, sbn);
    rc = take_workspace(name, plan.a, plan.b, workspace, workspace_bytes);
    if (rc) return rc;
    char *ws = (char *)workspace;
    hipStream_t st = (hipStream_t)stream;
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.g.A = repack(plan.a, A, ws, st, rc);
    if (rc) return rc;
    p.g.B = repack(plan.b, B, ws, st, rc);
    if (rc) return rc;
    p.g.C = C; p.g.s0 = row_scale; p.g.s1 = col_scale; p.g.M = M; p.g.N = N;
    p.g.lda = plan.a.pitch(); p.g.ldb = plan.b.pitch();
    p.g.out_dtype = out_dtype; p.g.scale_dtype = scale_dtype; p.g.col_scalar = col_scale_is_scalar != 0;
    p.ends = ends; p.T = T; p.E = E;
    p.ext_a = up16(M); p.ext_b = up16(N);
    // what the caller gave beyond the copies may hold the sums of a split contraction
    const int64_t copies = (plan.a.bytes() + plan.b.bytes() + 15) / 16 * 16;
    if (workspace && workspace_bytes > copies && ((uintptr_t)workspace & 15) == 0) {
        p.slab = (char *)workspace + copies;
        p.slab_bytes = workspace_bytes - copies;
    }
    p.out_bytes = gnk_dtype_size(out_dtype); p.scale_bytes = gnk_dtype_size(scale_dtype);
    return pick(a_dtype, b_dtype)(true, false, p, st);
}

// ------------------------------------------------------------------------------ quantizer (HBM-bound)
// scale[e, c] = max_{t in e} |x[t, c]| * fl(1 / 127);  q[t, c] = clip(rne(x[t, c] / max(scale[e(t), c], eps)), -128, 127)
//
// The maximum runs along the strided dimension of each group, so the pass splits as the dense column-wise quantizer does: kernel 1 writes
// one row of partial maxima (fp32 bit patterns: integer order, NaN above Inf) per piece of 1 << sh rows of a group -- no atomics, nothing
// to clear -- and kernel 2 takes 128-row pieces, reduces the (at most 33) partial rows of its group and quantizes.  A thread owns VEC
// adjacent columns (16 bytes; one column for pitches or widths that are no multiple of 16 bytes).
// 32768 x 5632 bf16 in 8 groups: 65-69 us for the maxima (5.5 TB/s) and 113-121 for the second read and the int8 (4.8 TB/s), 180 us together; a single read
// would take 110, but 369 MB do not stay in the 256 MB of last-level cache, and going through it in column chunks that do was slower at every chunk
// size (193-628 us: short rows, more launches).
namespace {

constexpr int GQ_ROWS_SH = 7;                  // rows of a kernel-2 piece
constexpr int GQ_PARTS = 32;                   // kernel 1: at most this many whole pieces over all groups

// The scale is amax * fl(1 / 127), as eager torch computes `amax / 127` on a device (a division by a host scalar becomes a product with its
// reciprocal): at most 1.5 fp32 steps from the quotient, where gnk_quantize_int8 has the correctly rounded one.  Values next to a tie can
// round the other way than there; nothing else differs.
constexpr float GQ_INV127 = 1.0f / 127.0f;

int partial_shift(int64_t T) {
    int sh = GQ_ROWS_SH;
    while ((T >> sh) > GQ_PARTS) ++sh;
    return sh;
}

// VEC adjacent elements as loaded (one 16-byte word, or the bits of a single element) and as floats
template <int DT, int VEC> __device__ __forceinline__ v4i load_vec(const char *p) {
    if constexpr (VEC == 1) return (v4i){(int)gnk_load_raw<DT>(p, 0), 0, 0, 0};
    else return *(const v4i *)p;
}
template <int DT, int VEC> __device__ __forceinline__ void floats_of(const v4i &raw, float (&f)[VEC]) {
    if constexpr (VEC == 1) {
        f[0] = gnk_raw_to_f32<DT>((unsigned)raw[0]);
    } else if constexpr (DT == GNK_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __int_as_float(raw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned w = (unsigned)raw[i];
            f[2 * i] = gnk_raw_to_f32<DT>(w & 0xffffu);
            f[2 * i + 1] = gnk_raw_to_f32<DT>(w >> 16);
        }
    }
}

// divisors of VEC columns from their maxima (fp32 bit patterns), and the scales
template <int DT, int VEC>
__device__ __forceinline__ bool divisors(const unsigned *amax, float eps, GnkDivisor (&dv)[VEC], void *scale, int64_t at, bool write) {
    bool fast = true;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float s = __fmul_rn(__uint_as_float(amax[j]), GQ_INV127);
        dv[j].set(gnk_clamp_min_nan(s, eps));
        fast = fast && dv[j].ok();
        if (write) gnk_store_scalar_rt(scale, DT, at + j, s);
    }
    return fast;
}

// VEC elements of row r from column col0 on: quantized and stored
template <int DT, int VEC, bool SR>
__device__ __forceinline__ void quant_store(const v4i &word, int64_t r, int64_t col0, int64_t C, const GnkDivisor (&dv)[VEC], bool fast, int8_t *__restrict__ q,
                                            unsigned long long seed, unsigned long long offset) {
    float f[VEC];
    floats_of<DT, VEC>(word, f);
    int qi[VEC];
    float u[VEC];
    if constexpr (SR) {
        const unsigned long long idx0 = (unsigned long long)(r * C + col0);
        if (VEC > 1 && ((idx0 + offset) & 3ull) == 0) {      // one Philox block per four elements
#pragma unroll
            for (int h = 0; h < VEC / 4; ++h) {
                float w[4];
                gnk_sr_uniform4(seed, offset, idx0 + 4 * h, w);
#pragma unroll
                for (int k = 0; k < 4; ++k) u[4 * h + k] = w[k];
            }
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) u[j] = gnk_sr_uniform(seed, offset, idx0 + j);
        }
    }
    if (fast) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) qi[j] = SR ? gnk_sr_clip_i8(dv[j].quot(f[j]), u[j]) : gnk_rne_clip_i8(dv[j].quot(f[j]));
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) qi[j] = SR ? gnk_sr_clip_i8(f[j] / dv[j].d, u[j]) : gnk_rne_clip_i8_any(f[j] / dv[j].d);
    }
    int8_t *dst = q + r * C + col0;
    if constexpr (VEC == 8) {
        v2i o;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            o[h] = (qi[4 * h] & 0xff) | ((qi[4 * h + 1] & 0xff) << 8) | ((qi[4 * h + 2] & 0xff) << 16) | (int)((unsigned)(qi[4 * h + 3] & 0xff) << 24);
        __builtin_nontemporal_store(o, (v2i *)dst);
    } else if constexpr (VEC == 4) {
        *(int *)dst = (qi[0] & 0xff) | ((qi[1] & 0xff) << 8) | ((qi[2] & 0xff) << 16) | (int)((unsigned)(qi[3] & 0xff) << 24);
    } else {
        dst[0] = (int8_t)qi[0];
    }
}

// Small calls (T <= GQ_ONCE_ROWS): one workgroup takes a group's CL * VEC columns from the maximum to the last store -- one launch, no partial maxima, no
// search for its rows.  A thread keeps its first eight rows in registers; a group with more is read again from L2.  Bound by its two barriers and the
// launch: 1021 x 512 bf16 in 8 groups 5 us (7.8 us a call, the host's side).
constexpr int64_t GQ_ONCE_ROWS = 2048;

template <int DT, int VEC, int CL, bool SR>
__global__ void __launch_bounds__(256)
group_quant_once_kernel(const char *__restrict__ x, int8_t *__restrict__ q, void *__restrict__ scale, const int *__restrict__ ends, int64_t T, int64_t E, int64_t C,
                        int64_t row_bytes, int64_t col_bytes, float eps, unsigned long long seed, unsigned long long offset) {
    constexpr int RL = 256 / CL, KEEP = 8;
    const int cl = threadIdx.x % CL, rl = threadIdx.x / CL;
    const int64_t col0 = ((int64_t)blockIdx.x * CL + cl) * VEC, e = blockIdx.y;
    int lo, hi;
    one_group(ends, E, T, e, threadIdx.x & 63, lo, hi);
    if (e == E) {                                // rows of no group
        if (col0 < C)
            for (int64_t r = lo + rl; r < hi; r += RL)
#pragma unroll
                for (int j = 0; j < VEC; ++j) q[r * C + col0 + j] = 0;
        return;
    }
    const char *src = x + (col0 < C ? col0 : 0) * col_bytes;
    unsigned mw[4] = {0u, 0u, 0u, 0u};
    v4i keep[KEEP];
    for (int64_t r0 = lo + rl; r0 < hi; r0 += RL * KEEP) {
        v4i raw[KEEP];
#pragma unroll
        for (int u = 0; u < KEEP; ++u) {
            raw[u] = (v4i){0, 0, 0, 0};
            if (r0 + RL * u < hi) raw[u] = load_vec<DT, VEC>(src + (r0 + RL * u) * row_bytes);
        }
#pragma unroll
        for (int u = 0; u < KEEP; ++u) {
#pragma unroll
            for (int j = 0; j < (VEC == 1 ? 1 : 4); ++j) {
                if constexpr (DT == GNK_F32) { const unsigned a = (unsigned)raw[u][j] & 0x7fffffffu; mw[j] = a > mw[j] ? a : mw[j]; }
                else mw[j] = gnk_pk_max_u16(mw[j], (unsigned)raw[u][j] & 0x7fff7fffu);
            }
            if (r0 == lo + rl) keep[u] = raw[u];
        }
    }
    const v4i most = {(int)mw[0], (int)mw[1], (int)mw[2], (int)mw[3]};
    float m[VEC];
    floats_of<DT, VEC>(most, m);
    __shared__ unsigned red[RL][CL * VEC + 1];
    __shared__ unsigned cm[CL * VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) red[rl][cl * VEC + j] = __float_as_uint(m[j]);
    __syncthreads();
    for (int c = threadIdx.x; c < CL * VEC; c += 256) {
        unsigned v = red[0][c];
#pragma unroll
        for (int i = 1; i < RL; ++i) v = red[i][c] > v ? red[i][c] : v;
        cm[c] = v;
    }
    __syncthreads();
    if (col0 >= C) return;
    GnkDivisor dv[VEC];
    const bool fast = divisors<DT, VEC>(cm + cl * VEC, eps, dv, scale, e * C + col0, rl == 0);
#pragma unroll
    for (int u = 0; u < KEEP; ++u) {
        const int64_t r = lo + rl + RL * u;
        if (r < hi) quant_store<DT, VEC, SR>(keep[u], r, col0, C, dv, fast, q, seed, offset);
    }
    for (int64_t r = lo + rl + RL * KEEP; r < hi; r += RL) quant_store<DT, VEC, SR>(load_vec<DT, VEC>(src + r * row_bytes), r, col0, C, dv, fast, q, seed, offset);
}

template <int DT, int VEC, int CL>
__global__ void __launch_bounds__(256)
group_absmax_kernel(const char *__restrict__ x, unsigned *__restrict__ partial, const int *__restrict__ ends, int64_t T, int64_t E, int64_t C, int64_t row_bytes,
                    int64_t col_bytes, int sh) {
    constexpr int RL = 256 / CL, U = 16;
    const int lane = threadIdx.x & 63;
    const Piece pc = find_piece(ends, E, T, lane, sh, (int)blockIdx.y, sh);
    if (pc.e < 0 || pc.e == E) return;
    const int64_t r0 = pc.lo + ((int64_t)pc.idx << sh), r1 = r0 + (1LL << sh) < pc.hi ? r0 + (1LL << sh) : pc.hi;
    const int cl = threadIdx.x % CL, rl = threadIdx.x / CL;
    const int64_t col0 = ((int64_t)blockIdx.x * CL + cl) * VEC;
    unsigned mw[4] = {0u, 0u, 0u, 0u};                    // per loaded word: two packed 16-bit patterns, or one fp32 pattern
    if (col0 < C) {
        const char *src = x + col0 * col_bytes;
        for (int64_t r = r0 + rl; r < r1; r += RL * U) {
            v4i raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {                  // 16 loads in flight; a row past the piece counts for nothing
                raw[u] = (v4i){0, 0, 0, 0};
                if (r + RL * u < r1) raw[u] = load_vec<DT, VEC>(src + (r + RL * u) * row_bytes);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < (VEC == 1 ? 1 : 4); ++j) {
                    if constexpr (DT == GNK_F32) { const unsigned a = (unsigned)raw[u][j] & 0x7fffffffu; mw[j] = a > mw[j] ? a : mw[j]; }
                    else mw[j] = gnk_pk_max_u16(mw[j], (unsigned)raw[u][j] & 0x7fff7fffu);
                }
        }
    }
    const v4i most = {(int)mw[0], (int)mw[1], (int)mw[2], (int)mw[3]};
    float m[VEC];
    floats_of<DT, VEC>(most, m);
    __shared__ unsigned red[RL][CL * VEC + 1];
#pragma unroll
    for (int j = 0; j < VEC; ++j) red[rl][cl * VEC + j] = __float_as_uint(m[j]);
    __syncthreads();
    for (int c = threadIdx.x; c < CL * VEC; c += 256) {
        unsigned v = red[0][c];
#pragma unroll
        for (int i = 1; i < RL; ++i) v = red[i][c] > v ? red[i][c] : v;
        const int64_t col = (int64_t)blockIdx.x * CL * VEC + c;
        if (col < C) partial[(int64_t)blockIdx.y * C + col] = v;
    }
}

template <int DT, int VEC, int CL, bool SR, int ROWS_SH>
__global__ void __launch_bounds__(256)
group_quant_kernel(const char *__restrict__ x, int8_t *__restrict__ q, void *__restrict__ scale, const unsigned *__restrict__ partial,
                   const int *__restrict__ ends, int64_t T, int64_t E, int64_t C, int64_t row_bytes, int64_t col_bytes, int sh, float eps,
                   unsigned long long seed, unsigned long long offset) {
    constexpr int RL = 256 / CL, NIT = (1 << ROWS_SH) / RL, U = NIT < 16 ? NIT : 16;
    const int lane = threadIdx.x & 63;
    const int cl = threadIdx.x % CL, rl = threadIdx.x / CL;
    const int64_t col0 = ((int64_t)blockIdx.x * CL + cl) * VEC;
    if (blockIdx.y == 0) {                       // groups without rows have no piece: their scale (0) is written here
        int end = 0;
        for (int64_t g0 = 0; g0 < E; g0 += 64) {
            int l, h;
            lane_group(ends, E, T, g0, lane, end, l, h);
            unsigned long long none = __ballot(g0 + lane < E && h == l);
            while (none) {
                const int64_t g = g0 + __builtin_ctzll(none);
                none &= none - 1;
                if (rl == 0 && col0 < C)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) gnk_store_scalar_rt(scale, DT, g * C + col0 + j, 0.0f);
            }
        }
    }
    const Piece pc = find_piece(ends, E, T, lane, ROWS_SH, (int)blockIdx.y, sh);
    if (pc.e < 0) return;
    const int64_t r0 = pc.lo + ((int64_t)pc.idx << ROWS_SH), r1 = r0 + (1LL << ROWS_SH) < pc.hi ? r0 + (1LL << ROWS_SH) : pc.hi;
    if (pc.e == E) {                             // rows of no group
        if (col0 < C)
            for (int64_t r = r0 + rl; r < r1; r += RL)
#pragma unroll
                for (int j = 0; j < VEC; ++j) q[r * C + col0 + j] = 0;
        return;
    }
    // The first 16 rows of this thread are loaded before the partial maxima are waited for.
    const char *src = x + (col0 < C ? col0 : 0) * col_bytes;
    v4i raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t r = r0 + rl + RL * u;
        raw[u] = (v4i){0, 0, 0, 0};
        if (r < r1) raw[u] = load_vec<DT, VEC>(src + r * row_bytes);
    }
    const int nparts = pieces_of(pc.hi - pc.lo, sh);
    __shared__ unsigned cm[CL * VEC];
    for (int c = threadIdx.x; c < CL * VEC; c += 256) {
        const int64_t col = (int64_t)blockIdx.x * CL * VEC + c;
        unsigned v = 0u;
        if (col < C)
            for (int k0 = 0; k0 < nparts; k0 += 8) {
                unsigned w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = k0 + k < nparts ? partial[(int64_t)(pc.first2 + k0 + k) * C + col] : 0u;
#pragma unroll
                for (int k = 0; k < 8; ++k) v = w[k] > v ? w[k] : v;
            }
        cm[c] = v;
    }
    __syncthreads();
    if (col0 >= C) return;
    GnkDivisor dv[VEC];
    const bool fast = divisors<DT, VEC>(cm + cl * VEC, eps, dv, scale, (int64_t)pc.e * C + col0, pc.idx == 0 && rl == 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t r = r0 + rl + RL * u;
        if (r < r1) quant_store<DT, VEC, SR>(raw[u], r, col0, C, dv, fast, q, seed, offset);
    }
    for (int64_t r = r0 + rl + RL * U; r < r1; r += RL) quant_store<DT, VEC, SR>(load_vec<DT, VEC>(src + r * row_bytes), r, col0, C, dv, fast, q, seed, offset);
}

template <int DT, bool VECTOR>
int launch_group_quant(const void *x, int8_t *q, void *scale, const int *ends, int64_t T, int64_t E, int64_t C, int64_t sxt, int64_t sxc, float eps, int sr,
                       uint64_t seed, uint64_t offset, unsigned *partial, hipStream_t st) {
    constexpr int ES = DT == GNK_F32 ? 4 : 2, VEC = VECTOR ? 16 / ES : 1, CL = VECTOR ? 32 : 64;
    if (T <= GQ_ONCE_ROWS && E < 65535) {
        constexpr int CLO = VECTOR ? 8 : 32;
        const dim3 g((unsigned)((C + CLO * VEC - 1) / (CLO * VEC)), (unsigned)(E + 1));
        if (sr)
            hipLaunchKernelGGL((group_quant_once_kernel<DT, VEC, CLO, true>), g, dim3(256), 0, st, (const char *)x, q, scale, ends, T, E, C, sxt * ES, sxc * ES, eps, seed, offset);
        else
            hipLaunchKernelGGL((group_quant_once_kernel<DT, VEC, CLO, false>), g, dim3(256), 0, st, (const char *)x, q, scale, ends, T, E, C, sxt * ES, sxc * ES, eps, seed, offset);
        return gnk_check_launch("quantize_int8_grouped");
    }
    const int sh = partial_shift(T);
    const unsigned gx = (unsigned)((C + CL * VEC - 1) / (CL * VEC));
    // 128-row pieces once they fill the chip; below that a thread's 16 rows of arithmetic (~5 us) are the kernel's length, and 32-row ones quarter it
    const int rows_sh = max_row_tiles(T, E, 128) * (int64_t)gx * 2 >= 3 * (int64_t)gnk_num_cus() || max_row_tiles(T, E, 32) > 65535 ? GQ_ROWS_SH : 5;
    const int64_t p1 = max_row_tiles(T, E, 1LL << sh), p2 = max_row_tiles(T, E, 1LL << rows_sh);
    // gridDim.y carries the pieces
    const dim3 g1(gx, (unsigned)(p1 > 0 ? p1 : 1)), g2(gx, (unsigned)(p2 > 0 ? p2 : 1));
    hipLaunchKernelGGL((group_absmax_kernel<DT, VEC, CL>), g1, dim3(256), 0, st, (const char *)x, partial, ends, T, E, C, sxt * ES, sxc * ES, sh);
#define GNK_GQ_RUN(SR, SH)                                                                                                                             \
    hipLaunchKernelGGL((group_quant_kernel<DT, VEC, CL, SR, SH>), g2, dim3(256), 0, st, (const char *)x, q, scale, partial, ends, T, E, C, sxt * ES,      \
                       sxc * ES, sh, eps, seed, offset)
    if (sr) {
        if (rows_sh == 5) GNK_GQ_RUN(true, 5);
        else GNK_GQ_RUN(true, GQ_ROWS_SH);
    } else {
        if (rows_sh == 5) GNK_GQ_RUN(false, 5);
        else GNK_GQ_RUN(false, GQ_ROWS_SH);
    }
#undef GNK_GQ_RUN
    return gnk_check_launch("quantize_int8_grouped");
}

}  // namespace

extern "C" int64_t gnk_quantize_int8_grouped_workspace_bytes(int64_t T, int64_t E, int64_t C) {
    if (T <= 0 || E <= 0 || C <= 0 || (T <= GQ_ONCE_ROWS && E < 65535)) return 0;
    return max_row_tiles(T, E, 1LL << partial_shift(T)) * C * 4;
}

extern "C" int gnk_quantize_int8_grouped(const void *x, int x_dtype, const int32_t *ends, int64_t T, int64_t E, int64_t C, int64_t sxt, int64_t sxc, int8_t *q,
                                         void *scale, float eps, int sr, uint64_t seed, uint64_t offset, void *workspace, int64_t workspace_bytes,
                                         void *stream) {
    const char *name = "quantize_int8_grouped";
    if (T < 0 || E < 0 || C < 0) return gnk_fail(GNK_ERR_BAD_ARG, "%s: negative dimension", name);
    if (!gnk_is_float_dtype(x_dtype)) return gnk_fail(GNK_ERR_BAD_ARG, "%s: input dtype code %d is not bf16/f16/f32", name, x_dtype);
    if (T >= (1LL << 31) || E >= (1LL << 20) || C > MAX_PITCH) return gnk_fail(GNK_ERR_UNSUPPORTED, "%s: %lld rows, %lld groups, %lld columns are too many", name, (long long)T, (long long)E, (long long)C);
    const int64_t pieces = max_row_tiles(T, E, 1LL << GQ_ROWS_SH);
    if (pieces > 65535) return gnk_fail(GNK_ERR_UNSUPPORTED, "%s: %lld rows in %lld groups are too many", name, (long long)T, (long long)E);
    if (C == 0 || (T == 0 && E == 0)) return GNK_OK;
    if ((T > 0 && (!x || !q)) || (E > 0 && !scale)) return gnk_fail(GNK_ERR_BAD_ARG, "%s: null pointer", name);
    const int64_t need = gnk_quantize_int8_grouped_workspace_bytes(T, E, C);
    if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 3) != 0))
        return gnk_fail(GNK_ERR_WORKSPACE, "%s: needs a workspace of %lld bytes", name, (long long)need);
    int rc = gnk_init();
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    const int es = gnk_dtype_size(x_dtype), vec = 16 / es;
    const bool vector = sxc == 1 && C % vec == 0 && ((uintptr_t)x & 15) == 0 && (sxt * es) % 16 == 0 && ((uintptr_t)q & (vec - 1)) == 0;
#define GNK_GQ(DT)                                                                                                                                    \
    (vector ? launch_group_quant<DT, true>(x, q, scale, ends, T, E, C, sxt, sxc, eps, sr, seed, offset, (unsigned *)workspace, st)                    \
            : launch_group_quant<DT, false>(x, q, scale, ends, T, E, C, sxt, sxc, eps, sr, seed, offset, (unsigned *)workspace, st))
    if (x_dtype == GNK_BF16) return GNK_GQ(GNK_BF16);
    if (x_dtype == GNK_F16) return GNK_GQ(GNK_F16);
    return GNK_GQ(GNK_F32);
#undef GNK_GQ
}
