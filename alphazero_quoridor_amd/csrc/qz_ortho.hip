// qz_ortho.hip -- orthogonalising updates by Newton-Schulz products, and the optimiser step around it.
//
//   X_0 = U / max(|U|_F, 1e-7);  X <- a X + (b A + c A A) X with A = X X^T, `steps` times, on the shorter side (a tall matrix is
//   worked on as its transpose), a, b, c = 3.4445, -4.7750, 2.0315: every singular value moves towards 1.
//   The optimiser step: M <- mu M + (1 - mu) G;  U = G + mu (M - G) (Nesterov) or M;  W <- W (1 - lr decay) - lr scale X.
//
// Three products per step, all of the form C = P Q^T with both operands stored along the summed axis:
//   A = X X^T (symmetric: the lower tiles, mirrored);  B = b A + c A A (A is symmetric, so A A = A A^T; symmetric again);
//   X'^T = a X^T + X^T B (B symmetric): rows of X^T against rows of B.  So X is kept in both orientations.
// float32 accuracy on the fp16 matrix pipe: every value is hi + lo, two fp16 numbers of the value times 4096 (a 22-bit
// significand; all entries are below 4 in magnitude, so 4096 keeps hi in range and lo out of the subnormals down to 2^-15; an entry below
// that is kept to 2^-36 absolute, so a row far smaller than the rest keeps fewer digits than float32 would give it), and a
// product is hi hi + hi lo + lo hi with float32 accumulation, whatever the result's type: hi hi alone leaves a bfloat16 result up to
// 2.9e-3 off float64 (updates of flat or sparse spectra, 1,024 x 4,096) where its own rounding is 1.66e-3.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qz_ortho.h"

#pragma clang fp contract(fast)

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr double NS_A_64 = 3.4445, NS_B_64 = -4.7750, NS_C_64 = 2.0315;
constexpr float NS_A = (float)NS_A_64, NS_B = (float)NS_B_64, NS_C = (float)NS_C_64, NORM_FLOOR = 1e-7f;
constexpr float SCALE = 4096.f, INV_SCALE = 1.f / 4096.f, INV_SCALE2 = 1.f / (4096.f * 4096.f);
constexpr int MAX_MATS = 20;      // matrices per launch: their descriptors travel as kernel arguments (captured graphs keep them)
constexpr int MAX_PARTS = 1024;    // partial sums of |U|^2 per matrix

// one matrix, s = shorter side, l = longer; sp, lp = padded to the tile.  The planes are fp16, hi first, then lo.
struct Mat {
    const void* update;
    void* out;
    float* momentum;
    float* param;
    _Float16 *x, *xt0, *xt1, *a, *b;  // [2][sp][lp], [2][lp][sp], [2][lp][sp], [2][sp][sp], [2][sp][sp]
    double* parts;
    int64_t ld, out_ld;
    float scale;
    int32_t rows, cols, sp, lp, nparts;
    int32_t pbase;  // first of its partial products in this launch (products split along K)
};
struct Mats {
    Mat m[MAX_MATS];
    int32_t start[MAX_MATS + 1];  // first workgroup of each matrix in this launch
    int32_t count;
    OrthoStep o;
};
// What one launch of the product kernel covers: tiles base .. of its list, whole (quarters = 0) or as four tiles of half the side.
// kc > 0: every tile's sum is split into pieces of about kc stages, whose partial sums go to `partial`, one tile's worth per workgroup.
struct Part {
    int32_t base, quarters, odd, last, kc;
    float* partial;
};
__host__ __device__ constexpr int pieces_of(int stages, int kc) { return stages < kc ? 1 : (stages + kc / 2) / kc; }
static_assert(sizeof(Mats) + 64 <= 4096, "kernel arguments");

__device__ __forceinline__ int find_mat(const Mats& M, int wg) {
    int i = 0;  // (a fixed number of comparisons: the starts arrive in two scalar loads instead of one after the other)
#pragma unroll
    for (int k = 1; k < MAX_MATS; k++) i += k < M.count && wg >= M.start[k];
    return i;
}
__device__ __forceinline__ float load_elem(const void* p, int64_t i, int dtype) {
    if (dtype == 0) return static_cast<const float*>(p)[i];
    if (dtype == 1) return __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
    return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store_elem(void* p, int64_t i, int dtype, float v) {
    if (dtype == 0) static_cast<float*>(p)[i] = v;
    else if (dtype == 1) static_cast<__bf16*>(p)[i] = (__bf16)v;
    else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// ---- momentum, and the partial sums of |U|^2 (float64: the squares of float32 gradients may leave float32's range).
// U itself goes to the place of xt1, which the first step writes only after the split has read it.
__global__ __launch_bounds__(256) void k_ns_prepare(Mats M) {
    __shared__ double sh[256];
    const int i = find_mat(M, blockIdx.x);
    const Mat& m = M.m[i];
    const int wg = blockIdx.x - M.start[i];
    float* u = reinterpret_cast<float*>(m.xt1);
    double s = 0.0;
    auto one = [&](float v, int64_t e) {  // element e of the matrix, row by row
        if (M.o.muon) {
            const float old = m.momentum[e], mom = old + (v - old) * (1.f - M.o.momentum);
            m.momentum[e] = mom;
            v = M.o.nesterov ? v + (mom - v) * M.o.momentum : mom;
            u[e] = v;
        }
        s += (double)v * (double)v;
    };
    if (m.ld == m.cols || m.rows == 1) {  // one run of memory: four elements at a time where its start allows it
        const int64_t size = (int64_t)m.rows * m.cols;
        const bool wide = M.o.dtype == 0 && ((uintptr_t)m.update & 15) == 0 && (!M.o.muon || ((uintptr_t)m.momentum & 15) == 0);
        const int64_t quads = wide ? size >> 2 : 0;
        for (int64_t q = (int64_t)wg * 256 + threadIdx.x; q < quads; q += (int64_t)m.nparts * 256) {
            float4 g = static_cast<const float4*>(m.update)[q];
            if (M.o.muon) {
                float4 k = reinterpret_cast<const float4*>(m.momentum)[q];
                float* gv = &g.x;
                float* kv = &k.x;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    kv[e] = kv[e] + (gv[e] - kv[e]) * (1.f - M.o.momentum);
                    gv[e] = M.o.nesterov ? gv[e] + (kv[e] - gv[e]) * M.o.momentum : kv[e];
                }
                reinterpret_cast<float4*>(m.momentum)[q] = k;
                reinterpret_cast<float4*>(u)[q] = g;
            }
            s += (double)g.x * (double)g.x + (double)g.y * (double)g.y + ((double)g.z * (double)g.z + (double)g.w * (double)g.w);
        }
        for (int64_t e = (quads << 2) + (int64_t)wg * 256 + threadIdx.x; e < size; e += (int64_t)m.nparts * 256) one(load_elem(m.update, e, M.o.dtype), e);
    } else {  // rows apart: a workgroup takes rows, or pieces of 4,096 columns of them where there are few rows
        const int pieces = (m.cols + 4095) >> 12;
        for (int64_t p = wg; p < (int64_t)m.rows * pieces; p += m.nparts) {
            const int64_t r = p / pieces;
            const int c0 = (int)(p - r * pieces) << 12, c1 = c0 + 4096 < m.cols ? c0 + 4096 : m.cols;
            for (int c = c0 + threadIdx.x; c < c1; c += 256) one(load_elem(m.update, r * m.ld + c, M.o.dtype), r * m.cols + c);
        }
    }
    sh[threadIdx.x] = s;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) m.parts[wg] = sh[0];
}

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    const float t = v * SCALE;
    hi = (_Float16)t;
    lo = (_Float16)(t - (float)hi);
}

// ---- X_0 = U / |U| as hi / lo planes in both orientations, zero in the padding.  One workgroup = a 64 x 64 tile.
__global__ __launch_bounds__(256) void k_ns_split(Mats M) {
    __shared__ double sh[256];
    __shared__ float tile[64][65];
    const int i = find_mat(M, blockIdx.x);
    const Mat& m = M.m[i];
    const int wg = blockIdx.x - M.start[i], tiles_l = m.lp >> 6;
    const int s0 = (wg / tiles_l) << 6, l0 = (wg % tiles_l) << 6;
    double s = 0.0;
    for (int k = threadIdx.x; k < m.nparts; k += 256) s += m.parts[k];
    sh[threadIdx.x] = s;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    const double norm = sqrt(sh[0]);
    const double inv = 1.0 / (norm < (double)NORM_FLOOR ? (double)NORM_FLOOR : norm);  // (as a float32 it loses its digits from a norm of 2^126 on)
    const bool tall = m.rows > m.cols;
    const void* src = M.o.muon ? (const void*)m.xt1 : m.update;
    const int64_t ld = M.o.muon ? m.cols : m.ld;
    const int dtype = M.o.muon ? 0 : M.o.dtype;
    const int rr0 = tall ? l0 : s0, cc0 = tall ? s0 : l0;
    const int c = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < 64; r += 4) {
        float v = 0.f;
        if (rr0 + r < m.rows && cc0 + c < m.cols) v = (float)((double)load_elem(src, (int64_t)(rr0 + r) * ld + cc0 + c, dtype) * inv);
        if (tall) tile[c][r] = v;  // tile[s][l]
        else tile[r][c] = v;
    }
    __syncthreads();
    const int64_t plane = (int64_t)m.sp * m.lp;
    for (int r = threadIdx.x >> 6; r < 64; r += 4) {
        _Float16 hi, lo;
        split(tile[r][c], hi, lo);
        const int64_t e = (int64_t)(s0 + r) * m.lp + l0 + c;
        m.x[e] = hi;
        m.x[plane + e] = lo;
        split(tile[c][r], hi, lo);
        const int64_t t = (int64_t)(l0 + r) * m.sp + s0 + c;
        m.xt0[t] = hi;
        m.xt0[plane + t] = lo;
    }
}

// ---- C = P Q^T, one TxT tile per workgroup of four waves (2 x 2), K in steps of 32 through LDS.
// Measured at 4096^3: the product with X 478 us (862 TFLOP/s of fp16 products; this card's library product reaches 1,163), the matrix
// pipe busy for half of the cycles at 1.9 GHz, LDS reads and writes about as long; no bank conflicts; L2 hits 88 %.
// LDS rows are 64 bytes = four 16-byte chunks; chunk q of row r sits at q ^ ((r >> 2) & 3), so that the sixteen lanes that one
// pass of a 16-byte read serves fall on sixteen different bank groups.
enum { KIND_GRAM = 0, KIND_POLY = 1, KIND_APPLY = 2 };
constexpr int BK = 32;

template <int T>
struct GemmShared {
    half8 p[2][2][T * 4];  // [stage][hi | lo][row, chunk]
    half8 q[2][2][T * 4];
};

// Workgroup b runs on XCD b mod 8, each with an L2 of its own: consecutive tiles go to the same XCD.
__device__ __forceinline__ int xcd_order(int b, int n) {
    const int x = b & 7, per = n >> 3, rem = n & 7;
    return x * per + (x < rem ? x : rem) + (b >> 3);
}
// Tiles in bands of eight rows, column by column inside a band: 64 consecutive ones share 8 + 8 panels.
__device__ __forceinline__ void tile_full(int w, int tm, int tn, int& ti, int& tj) {
    const int band = w / (8 * tn), r = w - band * 8 * tn, left = tm - 8 * band, h = left < 8 ? left : 8;
    ti = 8 * band + r % h;
    tj = r / h;
}
__device__ __forceinline__ void tile_lower(int w, int t, int& ti, int& tj) {  // 32 I^2 + 4 I tiles lie before band I
    int I = (int)sqrtf((float)w * (1.f / 32.f));
    while (32 * (I + 1) * (I + 1) + 4 * (I + 1) <= w) I++;
    while (I > 0 && 32 * I * I + 4 * I > w) I--;
    int r = w - (32 * I * I + 4 * I);
    const int left = t - 8 * I, h = left < 8 ? left : 8;
    if (r < 8 * I * h) {
        ti = 8 * I + r % h;
        tj = r / h;
        return;
    }
    r -= 8 * I * h;
    int i = 0;
    while (r > i) r -= ++i;
    ti = 8 * I + i;
    tj = 8 * I + r;
}

// Four rows of one column of a symmetric product: A = P P^T as it is, or b A + c A A (A[row][col] = A[col][row]), as planes, and the
// mirrored tile (a tile on the diagonal computes both halves; they may differ in the last bit, lo hi and hi lo being added the other way
// round there).
template <int KIND>
__device__ __forceinline__ void store_symmetric(const Mat& m, bool mirror, int row, int col, float (&v)[4]) {
    const int64_t plane = (int64_t)m.sp * m.sp;
    _Float16* dst = KIND == KIND_GRAM ? m.a : m.b;
    half4 hi, lo;
    if (KIND == KIND_POLY) {
        const half4 ah = *reinterpret_cast<const half4*>(m.a + (int64_t)col * m.sp + row);
        const half4 al = *reinterpret_cast<const half4*>(m.a + plane + (int64_t)col * m.sp + row);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = NS_B * (((float)ah[e] + (float)al[e]) * INV_SCALE) + NS_C * v[e];
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        _Float16 a, b;
        split(v[e], a, b);
        hi[e] = a;
        lo[e] = b;
    }
    *reinterpret_cast<half4*>(dst + (int64_t)col * m.sp + row) = hi;
    *reinterpret_cast<half4*>(dst + plane + (int64_t)col * m.sp + row) = lo;
    if (mirror) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            dst[(int64_t)(row + e) * m.sp + col] = hi[e];
            dst[plane + (int64_t)(row + e) * m.sp + col] = lo[e];
        }
    }
}

// A wave's 32 x 64 part of C (rows rb .., columns cb ..; two accumulators side by side) as planes of c_new C + c_old old: to
// across[column][row], and to along[row][column] too unless the tile lies on the diagonal of a symmetric product.  Through 8 KB of LDS
// that the stages have left: float32 sums in, rows out (the old values, laid out like `along`, in on the way), then the halves in once
// more and columns out.  Every access to memory is 16 bytes a lane and 64 bytes or more a row; straight from the accumulators it is 2
// bytes a lane for rows and 8 bytes a column (X' of 1024 x 4096 and its transpose: 92 us, 79 us so; of four 1024 x 1024 with them: 149 and
// 120 us).
template <bool OLD>
__device__ __forceinline__ void store_both(const floatx16 (&acc)[2], char* mine, int rb, int cb, const _Float16* old, _Float16* along, _Float16* across,
                                           int64_t plane, int64_t ld_along, int64_t ld_across, float c_old, float c_new, bool both) {
    auto order = [] {  // a wave's LDS accesses keep their order; the compiler is kept to it
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    };
    const int lane = threadIdx.x & 63, r32 = lane & 31, h = lane >> 5;
    float* const f = reinterpret_cast<float*>(mine);         // [32 rows][64 columns]
    _Float16* const hh = reinterpret_cast<_Float16*>(mine);  // [hi | lo][32][64], chunk q of row r at q ^ 2 (r >> 3)
    half8 hi[4], lo[4];
    if (OLD) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int id = lane + 64 * i;
            const int64_t t = (int64_t)(rb + (id >> 3)) * ld_along + cb + 8 * (id & 7);
            hi[i] = *reinterpret_cast<const half8*>(old + t);
            lo[i] = *reinterpret_cast<const half8*>(old + plane + t);
        }
    }
#pragma unroll
    for (int y = 0; y < 2; y++)
#pragma unroll
        for (int e = 0; e < 16; e++) f[(8 * (e >> 2) + 4 * h + (e & 3)) * 64 + 32 * y + r32] = acc[y][e];
    order();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int id = lane + 64 * i;
        const int64_t t = (int64_t)(rb + (id >> 3)) * ld_along + cb + 8 * (id & 7);
        const float4 a = *reinterpret_cast<const float4*>(f + id * 8), b = *reinterpret_cast<const float4*>(f + id * 8 + 4);
        const float c[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            _Float16 u, w;
            split(c[e] * c_new + (OLD ? c_old * (((float)hi[i][e] + (float)lo[i][e]) * INV_SCALE) : 0.f), u, w);
            hi[i][e] = u;
            lo[i][e] = w;
        }
        if (both) {
            *reinterpret_cast<half8*>(along + t) = hi[i];
            *reinterpret_cast<half8*>(along + plane + t) = lo[i];
        }
    }
    order();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int id = lane + 64 * i, r = id >> 3, at = r * 64 + (((id & 7) ^ ((r >> 3) << 1)) << 3);
        *reinterpret_cast<half8*>(hh + at) = hi[i];
        *reinterpret_cast<half8*>(hh + 2048 + at) = lo[i];
    }
    order();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int c = (lane >> 2) + 16 * i, q = lane & 3, at = q * 512 + (((c >> 3) ^ (q << 1)) << 3) + (c & 7);
        half8 u, w;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            u[e] = hh[at + 64 * e];
            w[e] = hh[2048 + at + 64 * e];
        }
        const int64_t t = (int64_t)(cb + c) * ld_across + rb + 8 * q;
        *reinterpret_cast<half8*>(across + t) = u;
        *reinterpret_cast<half8*>(across + plane + t) = w;
    }
    order();
}

// D: stages of K in flight from memory to registers (the LDS holds two): a workgroup of 64-tiles has little arithmetic per stage to
// cover a load's latency with.
template <int T, int KIND, int D>
__global__ __launch_bounds__(256, T == 64 ? 3 : 2) void k_ns_gemm(Mats M, Part part) {
    constexpr int W = T / 64;             // 32 x 32 tiles per wave and side
    constexpr int LD = T * 4 / 256;       // 16-byte chunks per thread, operand and plane
    __shared__ GemmShared<T> sm;
    const int odd = part.odd, last = part.last;
    int wg = xcd_order(blockIdx.x, gridDim.x), quarter = 0;
    if (part.quarters) {
        quarter = wg & 3;
        wg >>= 2;
    }
    wg += part.base;
    const int i = find_mat(M, wg);
    const Mat& m = M.m[i];
    wg -= M.start[i];
    const int K = KIND == KIND_GRAM ? m.lp : m.sp;
    int ks = 0, ke = K / BK;
    const int slot = wg;
    if (part.kc) {
        const int pieces = pieces_of(ke, part.kc), piece = wg % pieces, len = (ke + pieces - 1) / pieces;
        wg /= pieces;
        ks = piece * len;
        if (ks + len < ke) ke = ks + len;
    }
    const int side = part.quarters ? 2 * T : T;
    int ti, tj;  // tile of P rows, of Q rows
    if (KIND == KIND_APPLY) tile_full(wg, m.lp / side, m.sp / side, ti, tj);
    else tile_lower(wg, m.sp / side, ti, tj);
    if (part.quarters) {
        ti = 2 * ti + (quarter >> 1);
        tj = 2 * tj + (quarter & 1);
        if (KIND != KIND_APPLY && tj > ti) return;  // above the diagonal
    }
    const _Float16* P = KIND == KIND_GRAM ? m.x : KIND == KIND_POLY ? m.a : (odd ? m.xt1 : m.xt0);
    const _Float16* Q = KIND == KIND_GRAM ? m.x : KIND == KIND_POLY ? m.a : m.b;
    const int64_t p_plane = KIND == KIND_POLY ? (int64_t)m.sp * m.sp : (int64_t)m.sp * m.lp;
    const int64_t q_plane = KIND == KIND_GRAM ? (int64_t)m.sp * m.lp : (int64_t)m.sp * m.sp;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave >> 1) * (T / 2), wn = (wave & 1) * (T / 2);
    const int r32 = lane & 31, h = lane >> 5;

    half8 rp[D][2][LD], rq[D][2][LD];
    auto fetch = [&](half8 (&fp)[2][LD], half8 (&fq)[2][LD], int k0) {
#pragma unroll
        for (int pl = 0; pl < 2; pl++)
#pragma unroll
            for (int t = 0; t < LD; t++) {
                const int c = tid + 256 * t, row = c >> 2, q = c & 3;
                fp[pl][t] = *reinterpret_cast<const half8*>(P + pl * p_plane + (int64_t)(ti * T + row) * K + k0 + q * 8);
                fq[pl][t] = *reinterpret_cast<const half8*>(Q + pl * q_plane + (int64_t)(tj * T + row) * K + k0 + q * 8);
            }
    };
    auto place = [&](int st, half8 (&fp)[2][LD], half8 (&fq)[2][LD]) {
#pragma unroll
        for (int pl = 0; pl < 2; pl++)
#pragma unroll
            for (int t = 0; t < LD; t++) {
                const int c = tid + 256 * t, row = c >> 2, q = c & 3;
                sm.p[st][pl][row * 4 + (q ^ ((row >> 2) & 3))] = fp[pl][t];
                sm.q[st][pl][row * 4 + (q ^ ((row >> 2) & 3))] = fq[pl][t];
            }
    };
    floatx16 acc[W][W];
#pragma unroll
    for (int x = 0; x < W; x++)
#pragma unroll
        for (int y = 0; y < W; y++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[x][y][e] = 0.f;

#pragma unroll
    for (int d = 0; d < D; d++)
        fetch(rp[d], rq[d], (ks + d < ke ? ks + d : ke - 1) * BK);
    place(0, rp[0], rq[0]);
    __syncthreads();
    for (int k0 = ks; k0 < ke; k0 += D)
#pragma unroll
    for (int d = 0; d < D; d++) {
        const int k = k0 + d, st = d & 1;  // D is even
        if (k >= ke) break;
        // unconditional (past the end: the last stage once more), so that the loads in flight are the same on every path and the
        // compiler waits for the oldest only
        fetch(rp[d], rq[d], (k + D < ke ? k + D : ke - 1) * BK);
        // all fragments of the stage are asked for at once, and the next stage is written between the two halves of the products (no
        // faster than half by half with two workgroups on a CU)
        half8 fp[2][2][W], fq[2][2][W];
#pragma unroll
        for (int kk = 0; kk < 2; kk++)  // 16 of K each
#pragma unroll
            for (int pl = 0; pl < 2; pl++)
#pragma unroll
                for (int x = 0; x < W; x++) {
                    const int rp_ = wm + 32 * x + r32, rq_ = wn + 32 * x + r32, q = 2 * kk + h;
                    fp[kk][pl][x] = sm.p[st][pl][rp_ * 4 + (q ^ ((rp_ >> 2) & 3))];
                    fq[kk][pl][x] = sm.q[st][pl][rq_ * 4 + (q ^ ((rq_ >> 2) & 3))];
                }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
            __builtin_amdgcn_s_setprio(1);  // the wave that multiplies goes first: 3 % of a 4096 x 4096 product
#pragma unroll
            for (int pr = 0; pr < 3; pr++)  // lo hi, hi lo, hi hi; the same accumulator again only after W W others
#pragma unroll
                for (int x = 0; x < W; x++)
#pragma unroll
                    for (int y = 0; y < W; y++)
                        acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[kk][pr == 0][x], fq[kk][pr == 1][y], acc[x][y], 0, 0, 0);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            if (kk == 0) place(st ^ 1, rp[(d + 1) % D], rq[(d + 1) % D]);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
    }

    if (KIND != KIND_APPLY && part.kc) {
        float4* dst = reinterpret_cast<float4*>(part.partial + (int64_t)(m.pbase + slot) * T * T) + tid;
#pragma unroll
        for (int x = 0; x < W; x++)
#pragma unroll
            for (int y = 0; y < W; y++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    dst[((x * W + y) * 4 + g) * 256] = make_float4(acc[x][y][4 * g], acc[x][y][4 * g + 1], acc[x][y][4 * g + 2], acc[x][y][4 * g + 3]);
        return;
    }
    if constexpr (T == 128) if (KIND != KIND_APPLY || !last) {
        constexpr bool SYM = KIND != KIND_APPLY;
        const int64_t plane = (int64_t)m.sp * (SYM ? m.sp : m.lp);
        const _Float16* old = KIND == KIND_GRAM ? nullptr : KIND == KIND_POLY ? m.a : odd ? m.xt1 : m.xt0;
        _Float16* along = KIND == KIND_GRAM ? m.a : KIND == KIND_POLY ? m.b : odd ? m.xt0 : m.xt1;
        _Float16* across = SYM ? along : m.x;
        const float c_old = KIND == KIND_POLY ? NS_B : NS_A, c_new = KIND == KIND_POLY ? NS_C * INV_SCALE2 : INV_SCALE2;
#pragma unroll
        for (int x = 0; x < W; x++)
            store_both<KIND != KIND_GRAM>(acc[x], reinterpret_cast<char*>(&sm) + wave * 8192, ti * T + wm + 32 * x, tj * T + wn, old, along, across, plane, m.sp,
                                          SYM ? m.sp : m.lp, c_old, c_new, !SYM || ti != tj);
        return;
    }
    // lane holds C[row0 + 8 (e >> 2) + (e & 3)][col]: four consecutive rows at a time
    const float lr = M.o.muon ? (M.o.lr_dev ? *M.o.lr_dev : M.o.lr) : 0.f;
#pragma unroll
    for (int x = 0; x < W; x++)
#pragma unroll
        for (int y = 0; y < W; y++) {
            const int col = tj * T + wn + 32 * y + r32, row0 = ti * T + wm + 32 * x + 4 * h;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int row = row0 + 8 * g;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = acc[x][y][4 * g + e] * INV_SCALE2;
                if (KIND != KIND_APPLY) {
                    store_symmetric<KIND>(m, ti != tj, row, col, v);
                } else {  // C[l][s]
                    const int64_t plane = (int64_t)m.sp * m.lp;
                    const _Float16* old = odd ? m.xt1 : m.xt0;
                    _Float16* nxt = odd ? m.xt0 : m.xt1;
                    half4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int64_t t = (int64_t)(row + e) * m.sp + col;
                        v[e] += NS_A * (((float)old[t] + (float)old[plane + t]) * INV_SCALE);
                    }
                    if (!last) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            _Float16 a, b;
                            split(v[e], a, b);
                            hi[e] = a;
                            lo[e] = b;
                            nxt[(int64_t)(row + e) * m.sp + col] = a;
                            nxt[plane + (int64_t)(row + e) * m.sp + col] = b;
                        }
                        *reinterpret_cast<half4*>(m.x + (int64_t)col * m.lp + row) = hi;
                        *reinterpret_cast<half4*>(m.x + plane + (int64_t)col * m.lp + row) = lo;
                    } else {
                        const bool tall = m.rows > m.cols;
                        const int smax = tall ? m.cols : m.rows, lmax = tall ? m.rows : m.cols;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (col < smax && row + e < lmax) {
                                const int64_t r = tall ? row + e : col, c = tall ? col : row + e;
                                if (M.o.muon) {
                                    float* w = m.param + r * m.cols + c;
                                    *w = *w * (1.f - lr * M.o.weight_decay) - lr * m.scale * v[e];
                                } else {
                                    store_elem(m.out, r * m.out_ld + c, M.o.dtype, v[e]);
                                }
                            }
                    }
                }
            }
        }
}

// The pieces of a split product summed in order; workgroup (tile, group of four rows per lane), lanes as in k_ns_gemm.
template <int T, int KIND>
__global__ __launch_bounds__(256) void k_ns_join(Mats M, Part part) {
    constexpr int W = T / 64;
    const int i = find_mat(M, blockIdx.x);
    const Mat& m = M.m[i];
    const int wg = blockIdx.x - M.start[i], x = blockIdx.y / (4 * W), y = blockIdx.y / 4 % W, g = blockIdx.y % 4;
    int ti, tj;
    tile_lower(wg, m.sp / T, ti, tj);
    const int stages = (KIND == KIND_GRAM ? m.lp : m.sp) / BK, pieces = pieces_of(stages, part.kc);
    const float4* src = reinterpret_cast<const float4*>(part.partial + (int64_t)(m.pbase + wg * pieces) * T * T) + blockIdx.y * 256 + threadIdx.x;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < pieces; p++) {
        const float4 t = src[(int64_t)p * (T * T / 4)];
        v[0] += t.x;
        v[1] += t.y;
        v[2] += t.z;
        v[3] += t.w;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] *= INV_SCALE2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = tj * T + (wave & 1) * (T / 2) + 32 * y + (lane & 31), row = ti * T + (wave >> 1) * (T / 2) + 32 * x + 4 * (lane >> 5) + 8 * g;
    store_symmetric<KIND>(m, ti != tj, row, col, v);
}

// ================================================================ shorter side up to 128: one launch per step
// A workgroup of eight waves owns a strip of 128 entries of the longer side through all steps, with the whole shorter side (S = 64 or
// 128, zero padded).  Strips share nothing but A: every launch ends with each strip's part of the next A = X X^T (float32), and
// begins with every workgroup summing the parts (in order) and forming B = b A + c A A for itself -- a 64^3 product done nine times
// over costs less than the launches it replaces.  Then X' = a X + B X on its strip, from registers, and X' X'^T through LDS.
// Bound by latencies one after the other (descriptor, parts from memory, LDS round trips), not by arithmetic.
constexpr int STRIP = 128, STRIP_THREADS = 512;
constexpr int STRIP_SUM = 65536;  // most floats of parts that a workgroup sums: 16 strips of 64 x 64, 4 of 128 x 128 (256 KB, ~2 us)
constexpr int TINY = 16, TINY_LONG = 8192;

struct StripShared {
    union {
        half8 a[2][128 * 128 / 8];     // A: [hi | lo][row, chunk of 8]
        half8 xs[2][128 * STRIP / 8];  // then X': [hi | lo][row of the shorter side, chunk of 8 of the strip]
        float out[128 * STRIP];        // or the result, [row of the shorter side][entry of the strip ^ row & 31]
        double sum[STRIP_THREADS];
        struct {
            double red[STRIP_THREADS / 64][TINY * TINY], A[TINY][TINY + 1], B[TINY][TINY + 1], P[TINY][TINY + 1], Q[TINY][TINY + 1];
        } tiny;
    };
    half8 b[2][128 * 128 / 8];         // B
};
template <int S>
__device__ __forceinline__ int ab_at(int row, int chunk) {  // sixteen consecutive rows fall on sixteen bank groups
    return row * (S / 8) + (chunk ^ (S == 64 ? (row >> 1) & 7 : row & 15));
}
__device__ __forceinline__ int xs_at(int row, int chunk) { return row * (STRIP / 8) + (chunk ^ (row & 15)); }
// P Q^T with hi / lo operands: one accumulator per product, so that a wave is not bound by the latency of adding to the same
// registers again
struct Acc3 {
    floatx16 a, b, c;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < 16; e++) a[e] = b[e] = c[e] = 0.f;
    }
    __device__ __forceinline__ void add(const half8& ph, const half8& pl, const half8& qh, const half8& ql) {
        a = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, a, 0, 0, 0);
        b = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, b, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, c, 0, 0, 0);
    }
    __device__ __forceinline__ float get(int e) const { return (a[e] + b[e]) + c[e]; }
};
// lanes r | r + 32 hold chunks c | c + 1 of eight values each -> lane r: the lower halves of both, lane r + 32: the upper halves
__device__ __forceinline__ void halves(const half8& v, half4& even, half4& odd) {
    typedef uint32_t uint4_ __attribute__((ext_vector_type(4)));
    typedef uint32_t uint2_ __attribute__((ext_vector_type(2)));
    const uint4_ w = __builtin_bit_cast(uint4_, v);
    const uint2_ a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    even = __builtin_bit_cast(half4, (uint2_){a[0], b[0]});
    odd = __builtin_bit_cast(half4, (uint2_){a[1], b[1]});
}
// The parts of A: its lower tiles of 32 x 32 only (3 of 4, 10 of 16: a CU reads what other workgroups wrote at some 40 GB/s, and this is
// most of what it reads), each [column][row].
template <int S>
constexpr int part_tiles() {
    return S == 64 ? 3 : 10;
}
template <int S>
constexpr int part_floats() {
    return part_tiles<S>() * 1024;
}
__device__ __forceinline__ void part_tile(int t, int& ti, int& tj) {
    ti = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
    tj = t - ti * (ti + 1) / 2;
}
// this strip's part of X X^T, scaled by SCALE^2; a tile per wave, then two more
template <int S>
__device__ __forceinline__ void strip_gram(const StripShared& sm, float* __restrict__ part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, h = lane >> 5;
#pragma unroll 1
    for (int t = wave; t < part_tiles<S>(); t += STRIP_THREADS / 64) {
        int ti, tj;
        part_tile(t, ti, tj);
        Acc3 acc;
        acc.clear();
#pragma unroll
        for (int kk = 0; kk < STRIP / 16; kk++) {
            const int p = xs_at(32 * ti + r32, 2 * kk + h), q = xs_at(32 * tj + r32, 2 * kk + h);
            acc.add(sm.xs[0][p], sm.xs[1][p], sm.xs[0][q], sm.xs[1][q]);
        }
#pragma unroll
        for (int g = 0; g < 4; g++)
            *reinterpret_cast<float4*>(part + t * 1024 + r32 * 32 + 8 * g + 4 * h) = make_float4(acc.get(4 * g), acc.get(4 * g + 1), acc.get(4 * g + 2), acc.get(4 * g + 3));
    }
}
// four entries of the shorter side (s0 ..) of one entry l of the longer side: to X^T in memory and to X in LDS
template <int S>
__device__ __forceinline__ void strip_keep(StripShared& sm, _Float16* xt, int64_t plane, int l0, int l, int s0, const float (&v)[4]) {
    half4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        _Float16 a, b;
        split(v[e], a, b);
        hi[e] = a;
        lo[e] = b;
        const int at = xs_at(s0 + e, l >> 3) * 8 + (l & 7);
        reinterpret_cast<_Float16*>(sm.xs[0])[at] = a;
        reinterpret_cast<_Float16*>(sm.xs[1])[at] = b;
    }
    *reinterpret_cast<half4*>(xt + (int64_t)(l0 + l) * S + s0) = hi;
    *reinterpret_cast<half4*>(xt + plane + (int64_t)(l0 + l) * S + s0) = lo;
}

template <int S>
__device__ __forceinline__ void strip_first(const Mats& M, const Mat& m, int strip, StripShared& sm) {
    double s = 0.0;
    for (int k = threadIdx.x; k < m.nparts; k += STRIP_THREADS) s += m.parts[k];
    sm.sum[threadIdx.x] = s;
    __syncthreads();
    for (int o = STRIP_THREADS / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) sm.sum[threadIdx.x] += sm.sum[threadIdx.x + o];
        __syncthreads();
    }
    const double norm = sqrt(sm.sum[0]);
    const double inv = 1.0 / (norm < (double)NORM_FLOOR ? (double)NORM_FLOOR : norm);
    __syncthreads();
    const bool tall = m.rows > m.cols;
    const void* src = M.o.muon ? (const void*)m.xt1 : m.update;
    const int64_t ld = M.o.muon ? m.cols : m.ld, plane = (int64_t)S * m.lp;
    const int dtype = M.o.muon ? 0 : M.o.dtype, smax = tall ? m.cols : m.rows, lmax = tall ? m.rows : m.cols;
    const int l0 = strip * STRIP, l = threadIdx.x & 127;
#pragma unroll 1
    for (int s0 = (threadIdx.x >> 7) * 4; s0 < S; s0 += 64) {  // sixteen loads in flight per thread
        float v[4][4];
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int si = s0 + 16 * q + e;
                v[q][e] = 0.f;
                if (si < smax && l0 + l < lmax) v[q][e] = (float)((double)load_elem(src, tall ? (int64_t)(l0 + l) * ld + si : (int64_t)si * ld + l0 + l, dtype) * inv);
            }
#pragma unroll
        for (int q = 0; q < 4; q++) strip_keep<S>(sm, m.xt0, plane, l0, l, s0 + 16 * q, v[q]);
    }
    __syncthreads();
    strip_gram<S>(sm, reinterpret_cast<float*>(m.a) + (int64_t)strip * part_floats<S>());
}

template <int S>
__device__ __forceinline__ void strip_step(const Mats& M, const Mat& m, int strip, int odd, int last, StripShared& sm) {
    constexpr int NK = S / 16, NJ = (part_floats<S>() / 4 + STRIP_THREADS - 1) / STRIP_THREADS, NP = S == 64 ? 8 : 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r32 = lane & 31, h = lane >> 5;
    const int l0 = strip * STRIP, lw = (wave & 3) * 32 + r32, strips = m.lp / STRIP;
    const int64_t plane = (int64_t)S * m.lp;
    const _Float16* xt = (odd ? m.xt1 : m.xt0) + (int64_t)(l0 + lw) * S;
    half8 xh[NK], xl[NK];
#pragma unroll
    for (int k = 0; k < NK; k++) {
        xh[k] = *reinterpret_cast<const half8*>(xt + 16 * k + 8 * h);
        xl[k] = *reinterpret_cast<const half8*>(xt + plane + 16 * k + 8 * h);
    }
    {  // A, from the strips' parts: 16 (20) 16-byte loads in flight per thread
        const float4* part = reinterpret_cast<const float4*>(odd ? m.b : m.a);
        float sum[NJ][4] = {};
#pragma unroll 1
        for (int p = 0; p < strips; p += NP) {
            float4 u[NP][NJ];
#pragma unroll
            for (int q = 0; q < NP; q++)
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const int e0 = threadIdx.x + STRIP_THREADS * j;
                    u[q][j] = part[(int64_t)(p + q < strips ? p + q : p) * (part_floats<S>() / 4) + (e0 < part_floats<S>() / 4 ? e0 : 0)];
                }
#pragma unroll
            for (int q = 0; q < NP; q++) {
                if (p + q < strips) {
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        sum[j][0] += u[q][j].x;
                        sum[j][1] += u[q][j].y;
                        sum[j][2] += u[q][j].z;
                        sum[j][3] += u[q][j].w;
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            const int e0 = threadIdx.x + STRIP_THREADS * j;
            if (e0 >= part_floats<S>() / 4) continue;
            int ti, tj;
            part_tile(e0 >> 8, ti, tj);
            const int row = 32 * ti + (e0 & 7) * 4, col = 32 * tj + ((e0 & 255) >> 3);  // four rows of a column
            half4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                _Float16 a, b;
                split(sum[j][e] * INV_SCALE2, a, b);
                hi[e] = a;
                lo[e] = b;
                if (ti != tj) {
                    const int at = ab_at<S>(row + e, col >> 3) * 8 + (col & 7);
                    reinterpret_cast<_Float16*>(sm.a[0])[at] = a;
                    reinterpret_cast<_Float16*>(sm.a[1])[at] = b;
                }
            }
            const int at = ab_at<S>(col, row >> 3) * 2 + ((row >> 2) & 1);
            reinterpret_cast<half4*>(sm.a[0])[at] = hi;
            reinterpret_cast<half4*>(sm.a[1])[at] = lo;
        }
    }
    __syncthreads();
    // B = b A + c A A, all tiles (S = 64: one for each of four waves; S = 128: two per wave)
    if (S == 128 || wave < 4) {
        const int ti = wave >> 1;
#pragma unroll 1
        for (int y = 0; y < (S == 64 ? 1 : 2); y++) {
            const int tj = S == 64 ? wave & 1 : 2 * (wave & 1) + y;
            Acc3 acc;
            acc.clear();
#pragma unroll
            for (int k = 0; k < NK; k++) {
                const int p = ab_at<S>(32 * ti + r32, 2 * k + h), q = ab_at<S>(32 * tj + r32, 2 * k + h);
                acc.add(sm.a[0][p], sm.a[1][p], sm.a[0][q], sm.a[1][q]);
            }
#pragma unroll
            for (int g = 0; g < 4; g++) {  // rows 32 ti + 8 g + 4 h .. of column 32 tj + r32; A is symmetric
                const int at = ab_at<S>(32 * tj + r32, 4 * ti + g) * 2 + h;
                const half4 ah = reinterpret_cast<const half4*>(sm.a[0])[at], al = reinterpret_cast<const half4*>(sm.a[1])[at];
                half4 hi, lo;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    _Float16 a, b;
                    split(NS_B * (((float)ah[e] + (float)al[e]) * INV_SCALE) + NS_C * (acc.get(4 * g + e) * INV_SCALE2), a, b);
                    hi[e] = a;
                    lo[e] = b;
                }
                reinterpret_cast<half4*>(sm.b[0])[at] = hi;
                reinterpret_cast<half4*>(sm.b[1])[at] = lo;
            }
        }
    }
    __syncthreads();
    // X' = a X + B X: rows = the shorter side (waves 4 .. 7 its upper half), columns = 32 entries of the longer one
#pragma unroll
    for (int t = 0; t < S / 64; t++) {
        const int y = t + (wave >> 2) * (S / 64);
        // This lane's entries of the old X: of each chunk of eight, the half that its results lie in.  Lanes r and r + 32 hold chunk
        // 2 k and 2 k + 1; swapping the one's upper with the other's lower half gives both what they need.
        half4 oh[4], ol[4];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            half8 vh = xh[2 * t + k], vl = xl[2 * t + k];
            const half8 uh = xh[2 * (t + S / 64) + k], ul = xl[2 * (t + S / 64) + k];
            if (wave >> 2) {
                vh = uh;
                vl = ul;
            }
            halves(vh, oh[2 * k], oh[2 * k + 1]);
            halves(vl, ol[2 * k], ol[2 * k + 1]);
        }
        Acc3 c;
        c.clear();
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const int p = ab_at<S>(32 * y + r32, 2 * k + h);
            c.add(sm.b[0][p], sm.b[1][p], xh[k], xl[k]);
        }
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int s0 = 32 * y + 8 * g + 4 * h;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = NS_A * (((float)oh[g][e] + (float)ol[g][e]) * INV_SCALE) + c.get(4 * g + e) * INV_SCALE2;
            if (!last) {
                strip_keep<S>(sm, odd ? m.xt0 : m.xt1, plane, l0, lw, s0, v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) sm.out[(s0 + e) * STRIP + (lw ^ ((s0 + e) & 31))] = v[e];
            }
        }
    }
    __syncthreads();
    if (!last) {
        strip_gram<S>(sm, reinterpret_cast<float*>(odd ? m.a : m.b) + (int64_t)strip * part_floats<S>());
        return;
    }
    const bool tall = m.rows > m.cols;
    const int smax = tall ? m.cols : m.rows, lmax = tall ? m.rows : m.cols;
    const float lr = M.o.muon ? (M.o.lr_dev ? *M.o.lr_dev : M.o.lr) : 0.f;
#pragma unroll 1
    for (int e0 = threadIdx.x; e0 < S * STRIP; e0 += 8 * STRIP_THREADS) {  // along the rows of the result, eight weights in flight
        float w[8], v[8];
        int64_t at[8];
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const int e = e0 + q * STRIP_THREADS, si = tall ? e % S : e / STRIP, l = tall ? e / S : e % STRIP;
            const int64_t r = tall ? l0 + l : si, c = tall ? si : l0 + l;
            const bool in = si < smax && l0 + l < lmax;
            v[q] = sm.out[si * STRIP + (l ^ (si & 31))];
            at[q] = in ? r * (M.o.muon ? m.cols : m.out_ld) + c : -1;
            w[q] = M.o.muon && in ? m.param[at[q]] : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 8; q++) {
            if (at[q] < 0) continue;
            if (M.o.muon) m.param[at[q]] = w[q] * (1.f - lr * M.o.weight_decay) - lr * m.scale * v[q];
            else store_elem(m.out, at[q], M.o.dtype, v[q]);
        }
    }
}

// ---- shorter side up to 16: everything in one workgroup, float64
// With X_k = P_k U / |U| only the s x s matrices move: A = U U^T / |U|^2 once, then A <- Q A Q, P <- Q P with Q = a + b A + c A A, and
// X = P U / |U| at the end: 2 s^2 l products instead of 15 s^2 l.  In float32 this loses the small singular values (A holds their
// squares, and its rounding error is carried by a^2 a step); in float64 it is more exact than the products on X.  The sum over l
// runs on the float64 matrix instruction (16 x 16 x 4, both operands the same register; row (lane >> 4) + 4 e of column lane & 15),
// bound by the latency of reading U.
__device__ __forceinline__ void tiny_all(const Mats& M, const Mat& m, StripShared& shared) {
    typedef double double4_ __attribute__((ext_vector_type(4)));
    auto& sm = shared.tiny;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool tall = m.rows > m.cols;
    const int s = tall ? m.cols : m.rows, l = tall ? m.rows : m.cols, size = s * l;
    float* u = reinterpret_cast<float*>(m.xt1);  // [s][l]
#pragma unroll 1
    for (int e0 = tid; e0 < size; e0 += 4 * STRIP_THREADS) {  // four elements' loads in flight per thread
        float v[4], old[4];
        int at[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int e = e0 + STRIP_THREADS * q < size ? e0 + STRIP_THREADS * q : e0, r = e / m.cols, c = e - r * m.cols;
            v[q] = load_elem(m.update, r * m.ld + c, M.o.dtype);
            old[q] = M.o.muon ? m.momentum[e] : 0.f;
            at[q] = tall ? c * l + r : e;
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (e0 + STRIP_THREADS * q >= size) continue;
            if (M.o.muon) {
                const float mom = old[q] + (v[q] - old[q]) * (1.f - M.o.momentum);
                m.momentum[e0 + STRIP_THREADS * q] = mom;
                v[q] = M.o.nesterov ? v[q] + (mom - v[q]) * M.o.momentum : mom;
            }
            u[at[q]] = v[q];
        }
    }
    __syncthreads();
    const int row = lane & 15, kq = lane >> 4;
    double4_ acc = {0.0, 0.0, 0.0, 0.0};
    for (int k0 = __builtin_amdgcn_readfirstlane(wave) * 32; k0 < l; k0 += STRIP_THREADS / 2) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = row < s && k0 + 4 * k + kq < l ? u[row * l + k0 + 4 * k + kq] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)v[k], (double)v[k], acc, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) sm.red[wave][((lane >> 4) + 4 * e) * TINY + row] = acc[e];
    __syncthreads();
    const int i = (tid >> 4) & 15, j = tid & 15;  // (both halves of the workgroup compute, the first writes)
    const bool mine = tid < TINY * TINY;
    double g = 0.0;
#pragma unroll
    for (int w = 0; w < STRIP_THREADS / 64; w++) g += sm.red[w][i * TINY + j];
    if (mine) sm.A[i][j] = g;
    __syncthreads();
    double norm2 = 0.0;
    for (int k = 0; k < s; k++) norm2 += sm.A[k][k];
    const double norm = sqrt(norm2), inv = 1.0 / (norm < (double)NORM_FLOOR ? (double)NORM_FLOOR : norm);
    __syncthreads();
    if (mine) {
        sm.A[i][j] = g * inv * inv;
        sm.P[i][j] = i == j ? inv : 0.0;
    }
    __syncthreads();
    auto product = [&](const double (&x)[TINY][TINY + 1], const double (&y)[TINY][TINY + 1]) {
        double t = 0.0;
        for (int k = 0; k < s; k++) t += x[i][k] * y[k][j];
        return t;
    };
    for (int step = 0; step < M.o.steps; step++) {
        const double q = (i == j ? NS_A_64 : 0.0) + NS_B_64 * sm.A[i][j] + NS_C_64 * product(sm.A, sm.A);
        if (mine) sm.Q[i][j] = q;
        __syncthreads();
        const double p = product(sm.Q, sm.P), t = product(sm.Q, sm.A);
        if (mine) sm.B[i][j] = t;
        __syncthreads();
        const double a = product(sm.B, sm.Q);
        if (mine) {
            sm.P[i][j] = p;
            sm.A[i][j] = a;
        }
        __syncthreads();
    }
    const float lr = M.o.muon ? (M.o.lr_dev ? *M.o.lr_dev : M.o.lr) : 0.f;
#pragma unroll 1
    for (int e0 = tid; e0 < size; e0 += 4 * STRIP_THREADS) {
        double t[4] = {0.0, 0.0, 0.0, 0.0};
        int ss[4], ll[4];
        float w[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int e = e0 + STRIP_THREADS * q < size ? e0 + STRIP_THREADS * q : e0, r = e / m.cols, c = e - r * m.cols;
            ss[q] = tall ? c : r;
            ll[q] = tall ? r : c;
            w[q] = M.o.muon ? m.param[e] : 0.f;
        }
        for (int k = 0; k < s; k++)
#pragma unroll
            for (int q = 0; q < 4; q++) t[q] += sm.P[ss[q]][k] * (double)u[k * l + ll[q]];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int e = e0 + STRIP_THREADS * q;
            if (e >= size) continue;
            if (M.o.muon) m.param[e] = w[q] * (1.f - lr * M.o.weight_decay) - lr * m.scale * (float)t[q];
            else store_elem(m.out, (int64_t)(e / m.cols) * m.out_ld + e % m.cols, M.o.dtype, (float)t[q]);
        }
    }
}

// first: X_0 and the parts of A, and the tiny matrices from beginning to end; else one step of the strips
// Workgroup b runs on XCD b mod 8.  All strips of a matrix are given to one XCD, so that the parts one workgroup wrote are in the L2
// that the others read them from: place (b mod 8) cap + b / 8, where each XCD has cap places; the tiny matrices come behind them.
__global__ __launch_bounds__(STRIP_THREADS) void k_ns_strip(Mats M, int first, int odd, int last, int cap) {
    __shared__ StripShared sm;
    const int b = blockIdx.x, place = b < 8 * cap ? (b & 7) * cap + (b >> 3) : b;
    if (place < M.start[0]) return;
    const int i = find_mat(M, place);
    const Mat& m = M.m[i];
    const int strip = place - M.start[i];
    if (strip >= (m.sp == TINY ? 1 : m.lp / STRIP)) return;  // an empty place
    if (m.sp == TINY) {
        tiny_all(M, m, sm);
    } else if (m.sp == 64) {
        if (first) strip_first<64>(M, m, strip, sm);
        else strip_step<64>(M, m, strip, odd, last, sm);
    } else {
        if (first) strip_first<128>(M, m, strip, sm);
        else strip_step<128>(M, m, strip, odd, last, sm);
    }
}

// ================================================================ host side
int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// How a matrix is worked on, by its sides alone.
enum { PATH_TINY = 0, PATH_STRIP = 1, PATH_TILES = 2 };
int path_of(int64_t rows, int64_t cols) {
    const int64_t s = rows < cols ? rows : cols, l = rows < cols ? cols : rows;
    if (s <= TINY && l <= TINY_LONG) return PATH_TINY;
    const int64_t sp = s <= 64 ? 64 : 128;
    return s <= 128 && (l + STRIP - 1) / STRIP * sp * sp <= STRIP_SUM ? PATH_STRIP : PATH_TILES;
}
// Matrices whose shorter side is 512 or more are padded so that tiles of 128 may be used.
int pad_of(int64_t rows, int64_t cols) { return (rows < cols ? rows : cols) >= 512 ? 128 : 64; }

int64_t layout(const OrthoMatrix& q, char* base, Mat* m) {
    const int64_t s = q.rows < q.cols ? q.rows : q.cols, l = q.rows < q.cols ? q.cols : q.rows;
    const int path = path_of(q.rows, q.cols), T = path == PATH_TINY ? TINY : path == PATH_STRIP ? (s <= 64 ? 64 : 128) : pad_of(q.rows, q.cols);
    const int64_t sp = align_up(s, T), lp = align_up(l, path == PATH_STRIP ? STRIP : T);
    // planes of X, and of A and B: (strips) X^T twice, U in the second's place, and two sets of parts of A; (tiny) U alone
    const int64_t xb = path == PATH_TINY ? align_up(s * l * 4, 256) : align_up(sp * lp * 4, 256);
    const int64_t ab = path == PATH_TINY ? 0 : align_up(sp * sp * 4 * (path == PATH_STRIP ? lp / STRIP : 1), 256), pb = MAX_PARTS * 8;
    const int64_t xs = path == PATH_TINY ? 1 : path == PATH_STRIP ? 2 : 3;
    if (m) {
        const int64_t parts = (q.rows * q.cols + 4095) / 4096;
        m->update = q.update;
        m->out = q.out;
        m->momentum = q.momentum;
        m->param = q.param;
        m->x = reinterpret_cast<_Float16*>(base);
        m->xt0 = reinterpret_cast<_Float16*>(base + (path == PATH_TILES ? xb : 0));
        m->xt1 = reinterpret_cast<_Float16*>(base + (xs - 1) * xb);
        m->a = reinterpret_cast<_Float16*>(base + xs * xb);
        m->b = reinterpret_cast<_Float16*>(base + xs * xb + ab);
        m->parts = reinterpret_cast<double*>(base + xs * xb + 2 * ab);
        m->pbase = 0;
        m->ld = q.ld;
        m->out_ld = q.out_ld;
        m->scale = q.scale;
        m->rows = (int32_t)q.rows;
        m->cols = (int32_t)q.cols;
        m->sp = (int32_t)sp;
        m->lp = (int32_t)lp;
        m->nparts = (int32_t)(parts < MAX_PARTS ? parts : MAX_PARTS);
    }
    return xs * xb + 2 * ab + pb;
}

// A symmetric product of fewer tiles than this is split along K, into about SPLIT_GOAL workgroups of at least SPLIT_MIN stages: alone
// on its CU a workgroup of four waves waits for its own LDS reads most of the time, two or three of them fill the gaps.
// (480 pieces, so that all of them run at once: of 768, a third ran in a second round.)
constexpr int SPLIT_BELOW = 384, SPLIT_GOAL = 480, SPLIT_MIN = 16;
constexpr int SLOTS = 512;  // workgroups of 128-tiles that run at once: two on each of 256 CUs

// -> workgroups; M.start (and pbase) set for tiles of T, split into pieces of kc stages if kc > 0
template <int KIND>
int set_starts(Mats& M, int T, int kc) {
    int wgs = 0;
    for (int i = 0; i < M.count; i++) {
        M.start[i] = wgs;
        const int t = M.m[i].sp / T, nk = (KIND == KIND_GRAM ? M.m[i].lp : M.m[i].sp) / BK;
        wgs += KIND == KIND_APPLY ? t * (M.m[i].lp / T) : t * (t + 1) / 2 * (kc ? pieces_of(nk, kc) : 1);
        if (kc) M.m[i].pbase = M.start[i];
    }
    return wgs;
}
template <int KIND, int T>
void run_symmetric(Mats& M, int tiles, float* partial, int odd, int last, hipStream_t s) {
    constexpr int D = T == 64 ? 4 : 2;
    int64_t stages = 0;
    int longest = 0;
    for (int i = 0; i < M.count; i++) {
        const int t = M.m[i].sp / T, nk = (KIND == KIND_GRAM ? M.m[i].lp : M.m[i].sp) / BK;
        stages += (int64_t)t * (t + 1) / 2 * nk;
        longest = nk > longest ? nk : longest;
    }
    int kc = (int)((stages + SPLIT_GOAL - 1) / SPLIT_GOAL);
    if (kc < SPLIT_MIN) kc = SPLIT_MIN;
    if (tiles >= SPLIT_BELOW || longest < 3 * kc) {
        hipLaunchKernelGGL((k_ns_gemm<T, KIND, D>), dim3(tiles), dim3(256), 0, s, M, Part{0, 0, odd, last, 0, nullptr});
        return;
    }
    const Part part = {0, 0, odd, last, kc, partial};
    const int wgs = set_starts<KIND>(M, T, kc);
    hipLaunchKernelGGL((k_ns_gemm<T, KIND, D>), dim3(wgs), dim3(256), 0, s, M, part);
    set_starts<KIND>(M, T, 0);
    hipLaunchKernelGGL((k_ns_join<T, KIND>), dim3(tiles, T * T / 1024), dim3(256), 0, s, M, part);
}
template <int KIND>
void run_gemm(Mats& M, bool may128, float* partial, int odd, int last, hipStream_t s) {
    int tiles = may128 ? set_starts<KIND>(M, 128, 0) : 0;
    // Tiles of 128 read half as much through LDS per product, tiles of 64 give four times the workgroups.  B = b A + c A A, whose sum is
    // short, takes the larger ones where there is one for every other CU (two 1024 x 1024 products, 72 tiles: 27 us in tiles of 64, 39 us
    // in tiles of 128; six, 216 tiles: 52 us and 45 us); the others, unless there would be next to none (A of two 1024 x 4096: 78 us in
    // tiles of 64, 59 us in tiles of 128 split along the sum; of two 1024 x 1024, whose sum is too short to split, 23 and 32 us).
    if (tiles < (KIND == KIND_POLY ? 128 : 32)) {
        tiles = set_starts<KIND>(M, 64, 0);
        if constexpr (KIND == KIND_APPLY) hipLaunchKernelGGL((k_ns_gemm<64, KIND, 4>), dim3(tiles), dim3(256), 0, s, M, Part{0, 0, odd, last, 0, nullptr});
        else run_symmetric<KIND, 64>(M, tiles, partial, odd, last, s);
        return;
    }
    if constexpr (KIND != KIND_APPLY) {
        if (tiles <= SLOTS) {
            run_symmetric<KIND, 128>(M, tiles, partial, odd, last, s);
            return;
        }
    }
    // what is left over a multiple of the slots runs in quarters, if it is less than half a round
    const int rest = tiles % SLOTS, head = tiles > SLOTS && rest * 2 < SLOTS ? tiles - rest : tiles;
    hipLaunchKernelGGL((k_ns_gemm<128, KIND, 2>), dim3(head), dim3(256), 0, s, M, Part{0, 0, odd, last, 0, nullptr});
    if (head < tiles) hipLaunchKernelGGL((k_ns_gemm<64, KIND, 4>), dim3(4 * (tiles - head)), dim3(256), 0, s, M, Part{head, 1, odd, last, 0, nullptr});
}
hipError_t run_steps(Mats& M, bool may128, float* partial, hipStream_t s) {
    for (int step = 0; step < M.o.steps; step++) {
        run_gemm<KIND_GRAM>(M, may128, partial, step & 1, 0, s);
        run_gemm<KIND_POLY>(M, may128, partial, step & 1, 0, s);
        run_gemm<KIND_APPLY>(M, may128, partial, step & 1, step + 1 == M.o.steps, s);
    }
    return hipGetLastError();
}

// strips and tiny matrices, the tiny ones (shortest: lp is theirs too) behind the strips
hipError_t run_strips(Mats& M, hipStream_t s) {
    const int all = M.count;
    int strips = 0, wgs = 0;
    while (strips < all && M.m[strips].sp != TINY) strips++;
    M.count = strips;
    for (int i = 0; i < strips; i++) {
        M.start[i] = wgs;
        wgs += M.m[i].nparts;
    }
    if (strips) hipLaunchKernelGGL(k_ns_prepare, dim3(wgs), dim3(256), 0, s, M);
    // the longest matrix first, to the XCD with the fewest strips; then in order of place
    int load[8] = {}, xcd[MAX_MATS], cap = 0, n = 0;
    for (int i = 0; i < strips; i++) {
        int x = 0;
        for (int k = 1; k < 8; k++)
            if (load[k] < load[x]) x = k;
        xcd[i] = x;
        load[x] += M.m[i].lp / STRIP;
        cap = load[x] > cap ? load[x] : cap;
    }
    Mats R = M;
    for (int x = 0; x < 8; x++) {
        int at = x * cap;
        for (int i = 0; i < strips; i++)
            if (xcd[i] == x) {
                R.m[n] = M.m[i];
                R.start[n++] = at;
                at += M.m[i].lp / STRIP;
            }
    }
    for (int i = strips; i < all; i++) R.start[i] = 8 * cap + (i - strips);
    R.count = all;
    hipLaunchKernelGGL(k_ns_strip, dim3(8 * cap + (all - strips)), dim3(STRIP_THREADS), 0, s, R, 1, 0, 0, cap);
    R.count = strips;
    for (int step = 0; step < M.o.steps && strips; step++)
        hipLaunchKernelGGL(k_ns_strip, dim3(8 * cap), dim3(STRIP_THREADS), 0, s, R, 0, step & 1, step + 1 == M.o.steps, cap);
    M.count = all;
    return hipGetLastError();
}

hipError_t run_group(Mats& M, int pad, float* partial, hipStream_t s) {
    int wgs = 0;
    for (int i = 0; i < M.count; i++) {
        M.start[i] = wgs;
        wgs += M.m[i].nparts;
    }
    hipLaunchKernelGGL(k_ns_prepare, dim3(wgs), dim3(256), 0, s, M);
    wgs = 0;
    for (int i = 0; i < M.count; i++) {
        M.start[i] = wgs;
        wgs += (M.m[i].sp >> 6) * (M.m[i].lp >> 6);
    }
    hipLaunchKernelGGL(k_ns_split, dim3(wgs), dim3(256), 0, s, M);
    return run_steps(M, pad == 128, partial, s);
}

// Room for the partial sums of split products: a launch has at most SPLIT_GOAL pieces and one more per tile (the last of each), and no
// more pieces than stages / SPLIT_MIN + 1 per tile.
int64_t partial_bytes(const OrthoMatrix* q, int count) {
    int64_t small = 0, most = 0;
    for (int i = 0; i < count; i++) {
        if (q[i].rows <= 0 || q[i].cols <= 0) continue;
        const int64_t s = q[i].rows < q[i].cols ? q[i].rows : q[i].cols, l = q[i].rows < q[i].cols ? q[i].cols : q[i].rows;
        if (path_of(q[i].rows, q[i].cols) != PATH_TILES) continue;
        const int64_t pad = pad_of(q[i].rows, q[i].cols);
        if (pad == 128) most = (int64_t)(SPLIT_GOAL + SLOTS) * 128 * 128 * 4;
        const int64_t t = align_up(s, pad) / 64, nk = align_up(l, pad) / BK;
        small += t * (t + 1) / 2 * (nk / SPLIT_MIN + 1) * 64 * 64 * 4;
    }
    const int64_t top = (int64_t)(SPLIT_GOAL + SPLIT_BELOW) * 64 * 64 * 4;
    if (small > top) small = top;
    return most > small ? most : small;
}

}  // namespace

namespace qzl {
int64_t ortho_workspace_bytes(const OrthoMatrix* q, int count, const OrthoStep&) {
    int64_t n = 0;
    for (int i = 0; i < count; i++)
        if (q[i].rows > 0 && q[i].cols > 0) n += layout(q[i], nullptr, nullptr);
    return n + partial_bytes(q, count);
}

hipError_t orthogonalize(const OrthoMatrix* q, int count, const OrthoStep& o, void* ws, hipStream_t s) {
    // groups that share their launches: strips and tiny ones, and tiles of either padding
    float* partial = static_cast<float*>(ws);
    for (int group = 0; group < 3; group++) {
        const bool tiles = group > 0;
        const int pad = group == 1 ? 64 : 128;
        Mats M;
        M.o = o;
        M.count = 0;
        char* base = static_cast<char*>(ws) + partial_bytes(q, count);
        auto run = [&]() -> hipError_t {
            const hipError_t e = tiles ? run_group(M, pad, partial, s) : run_strips(M, s);
            M.count = 0;
            return e;
        };
        for (int i = 0; i < count; i++) {
            if (q[i].rows <= 0 || q[i].cols <= 0) continue;
            const bool in_tiles = path_of(q[i].rows, q[i].cols) == PATH_TILES;
            if (in_tiles == tiles && (!tiles || pad_of(q[i].rows, q[i].cols) == pad)) {
                Mat m;
                layout(q[i], base, &m);
                // longest first: their workgroups run longest; tiny ones at the end
                const int64_t key = m.sp == TINY ? 0 : m.lp;
                int at = M.count++;
                for (; at > 0 && (M.m[at - 1].sp == TINY ? 0 : M.m[at - 1].lp) < key; at--) M.m[at] = M.m[at - 1];
                M.m[at] = m;
                if (M.count == MAX_MATS) {
                    const hipError_t e = run();
                    if (e != hipSuccess) return e;
                }
            }
            base += layout(q[i], nullptr, nullptr);
        }
        if (M.count) {
            const hipError_t e = run();
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}
}  // namespace qzl
