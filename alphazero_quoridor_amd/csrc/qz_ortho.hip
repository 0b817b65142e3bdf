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
// significand; all entries are below 4 in magnitude, so 4096 keeps hi in range and lo out of the subnormals down to 2^-15), and a
// product is hi hi + hi lo + lo hi with float32 accumulation.  Where the result is rounded to bfloat16 and the shorter side is
// 256 or more, ONE product (hi hi) is enough: the term a X, which carries the small singular values through the steps, is still
// taken from hi + lo, and the error of one product is 1.4e-3 of the result, next to the output's own rounding of 1.7e-3.
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

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f, NORM_FLOOR = 1e-7f;
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
// kc > 0: every tile's sum is split into pieces of kc stages, whose partial sums go to `partial`, one tile's worth per workgroup.
struct Part {
    int32_t base, quarters, odd, last, kc;
    float* partial;
};
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
    const float inv = (float)(1.0 / (norm < (double)NORM_FLOOR ? (double)NORM_FLOOR : norm));
    const bool tall = m.rows > m.cols;
    const void* src = M.o.muon ? (const void*)m.xt1 : m.update;
    const int64_t ld = M.o.muon ? m.cols : m.ld;
    const int dtype = M.o.muon ? 0 : M.o.dtype;
    const int rr0 = tall ? l0 : s0, cc0 = tall ? s0 : l0;
    const int c = threadIdx.x & 63;
    for (int r = threadIdx.x >> 6; r < 64; r += 4) {
        float v = 0.f;
        if (rr0 + r < m.rows && cc0 + c < m.cols) v = load_elem(src, (int64_t)(rr0 + r) * ld + cc0 + c, dtype) * inv;
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
// LDS rows are 64 bytes = four 16-byte chunks; chunk q of row r sits at q ^ ((r >> 2) & 3), so that the sixteen lanes that one
// pass of a 16-byte read serves fall on sixteen different bank groups.
enum { KIND_GRAM = 0, KIND_POLY = 1, KIND_APPLY = 2 };
constexpr int BK = 32;

template <int T, int NPL>
struct GemmShared {
    half8 p[2][NPL][T * 4];  // [stage][hi | lo][row, chunk]
    half8 q[2][NPL][T * 4];
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
// mirrored tile (a tile on the diagonal holds both halves already, equal bit for bit).
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

// D: stages of K in flight from memory to registers (the LDS holds two): a workgroup of 64-tiles has little arithmetic per stage to
// cover a load's latency with.
template <int T, int NP, int KIND, int D>
__global__ __launch_bounds__(256, T == 64 ? 3 : 2) void k_ns_gemm(Mats M, Part part) {
    constexpr int NPL = NP == 3 ? 2 : 1;  // planes read
    constexpr int W = T / 64;             // 32 x 32 tiles per wave and side
    constexpr int LD = T * 4 / 256;       // 16-byte chunks per thread, operand and plane
    __shared__ GemmShared<T, NPL> sm;
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
        const int pieces = (ke + part.kc - 1) / part.kc, piece = wg % pieces;
        wg /= pieces;
        ks = piece * part.kc;
        if (ks + part.kc < ke) ke = ks + part.kc;
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

    half8 rp[D][NPL][LD], rq[D][NPL][LD];
    auto fetch = [&](half8 (&fp)[NPL][LD], half8 (&fq)[NPL][LD], int k0) {
#pragma unroll
        for (int pl = 0; pl < NPL; pl++)
#pragma unroll
            for (int t = 0; t < LD; t++) {
                const int c = tid + 256 * t, row = c >> 2, q = c & 3;
                fp[pl][t] = *reinterpret_cast<const half8*>(P + pl * p_plane + (int64_t)(ti * T + row) * K + k0 + q * 8);
                fq[pl][t] = *reinterpret_cast<const half8*>(Q + pl * q_plane + (int64_t)(tj * T + row) * K + k0 + q * 8);
            }
    };
    auto place = [&](int st, half8 (&fp)[NPL][LD], half8 (&fq)[NPL][LD]) {
#pragma unroll
        for (int pl = 0; pl < NPL; pl++)
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
        // all fragments of the stage are asked for at once, and the next stage is written between the two halves of the products: a
        // workgroup alone on its CU then waits for one LDS round trip per stage instead of three
        half8 fp[2][NPL][W], fq[2][NPL][W];
#pragma unroll
        for (int kk = 0; kk < 2; kk++)  // 16 of K each
#pragma unroll
            for (int pl = 0; pl < NPL; pl++)
#pragma unroll
                for (int x = 0; x < W; x++) {
                    const int rp_ = wm + 32 * x + r32, rq_ = wn + 32 * x + r32, q = 2 * kk + h;
                    fp[kk][pl][x] = sm.p[st][pl][rp_ * 4 + (q ^ ((rp_ >> 2) & 3))];
                    fq[kk][pl][x] = sm.q[st][pl][rq_ * 4 + (q ^ ((rq_ >> 2) & 3))];
                }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
#pragma unroll
            for (int pr = NP == 3 ? 0 : 2; pr < 3; pr++)  // lo hi, hi lo, hi hi; the same accumulator again only after W W others
#pragma unroll
                for (int x = 0; x < W; x++)
#pragma unroll
                    for (int y = 0; y < W; y++)
                        acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[kk][pr == 0 ? NPL - 1 : 0][x], fq[kk][pr == 1 ? NPL - 1 : 0][y], acc[x][y], 0, 0, 0);
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
    const int stages = (KIND == KIND_GRAM ? m.lp : m.sp) / BK, pieces = (stages + part.kc - 1) / part.kc;
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

// ================================================================ host side
int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// Matrices whose shorter side is 512 or more are padded so that tiles of 128 may be used.
int pad_of(int64_t rows, int64_t cols) { return (rows < cols ? rows : cols) >= 512 ? 128 : 64; }
bool one_product(const OrthoMatrix& q, const OrthoStep& o) { return !o.muon && o.dtype == 1 && (q.rows < q.cols ? q.rows : q.cols) >= 256; }

int64_t layout(const OrthoMatrix& q, char* base, Mat* m) {
    const int64_t s = q.rows < q.cols ? q.rows : q.cols, l = q.rows < q.cols ? q.cols : q.rows;
    const int T = pad_of(q.rows, q.cols);
    const int64_t sp = align_up(s, T), lp = align_up(l, T);
    const int64_t xb = align_up(sp * lp * 4, 256), ab = align_up(sp * sp * 4, 256), pb = MAX_PARTS * 8;
    if (m) {
        const int64_t parts = (q.rows * q.cols + 4095) / 4096;
        m->update = q.update;
        m->out = q.out;
        m->momentum = q.momentum;
        m->param = q.param;
        m->x = reinterpret_cast<_Float16*>(base);
        m->xt0 = reinterpret_cast<_Float16*>(base + xb);
        m->xt1 = reinterpret_cast<_Float16*>(base + 2 * xb);
        m->a = reinterpret_cast<_Float16*>(base + 3 * xb);
        m->b = reinterpret_cast<_Float16*>(base + 3 * xb + ab);
        m->parts = reinterpret_cast<double*>(base + 3 * xb + 2 * ab);
        m->ld = q.ld;
        m->out_ld = q.out_ld;
        m->scale = q.scale;
        m->rows = (int32_t)q.rows;
        m->cols = (int32_t)q.cols;
        m->sp = (int32_t)sp;
        m->lp = (int32_t)lp;
        m->nparts = (int32_t)(parts < MAX_PARTS ? parts : MAX_PARTS);
    }
    return 3 * xb + 2 * ab + pb;
}

// A symmetric product of fewer tiles than this is split along K, into about SPLIT_GOAL workgroups of at least SPLIT_MIN stages: alone
// on its CU a workgroup of four waves waits for its own LDS reads most of the time, two or three of them fill the gaps.
constexpr int SPLIT_BELOW = 384, SPLIT_GOAL = 768, SPLIT_MIN = 16;
constexpr int SLOTS = 512;  // workgroups of 128-tiles that run at once: two on each of 256 CUs

// -> workgroups; M.start (and pbase) set for tiles of T, split into pieces of kc stages if kc > 0
template <int KIND>
int set_starts(Mats& M, int T, int kc) {
    int wgs = 0;
    for (int i = 0; i < M.count; i++) {
        M.start[i] = wgs;
        const int t = M.m[i].sp / T, nk = (KIND == KIND_GRAM ? M.m[i].lp : M.m[i].sp) / BK;
        wgs += KIND == KIND_APPLY ? t * (M.m[i].lp / T) : t * (t + 1) / 2 * (kc ? (nk + kc - 1) / kc : 1);
        if (kc) M.m[i].pbase = M.start[i];
    }
    return wgs;
}
template <int NP, int KIND, int T>
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
        hipLaunchKernelGGL((k_ns_gemm<T, NP, KIND, D>), dim3(tiles), dim3(256), 0, s, M, Part{0, 0, odd, last, 0, nullptr});
        return;
    }
    const Part part = {0, 0, odd, last, kc, partial};
    const int wgs = set_starts<KIND>(M, T, kc);
    hipLaunchKernelGGL((k_ns_gemm<T, NP, KIND, D>), dim3(wgs), dim3(256), 0, s, M, part);
    set_starts<KIND>(M, T, 0);
    hipLaunchKernelGGL((k_ns_join<T, KIND>), dim3(tiles, T * T / 1024), dim3(256), 0, s, M, part);
}
template <int NP, int KIND>
void run_gemm(Mats& M, bool may128, float* partial, int odd, int last, hipStream_t s) {
    int tiles = may128 ? set_starts<KIND>(M, 128, 0) : 0;
    // Tiles of 128 read half as much through LDS per product, tiles of 64 give four times the workgroups: the larger ones unless
    // there would be next to none.
    if (tiles < 32) {
        tiles = set_starts<KIND>(M, 64, 0);
        if (KIND == KIND_APPLY) hipLaunchKernelGGL((k_ns_gemm<64, NP, KIND, 4>), dim3(tiles), dim3(256), 0, s, M, Part{0, 0, odd, last, 0, nullptr});
        else run_symmetric<NP, KIND, 64>(M, tiles, partial, odd, last, s);
        return;
    }
    if (KIND != KIND_APPLY && tiles <= SLOTS) {
        run_symmetric<NP, KIND, 128>(M, tiles, partial, odd, last, s);
        return;
    }
    // what is left over a multiple of the slots runs in quarters, if it is less than half a round
    const int rest = tiles % SLOTS, head = tiles > SLOTS && rest * 2 < SLOTS ? tiles - rest : tiles;
    hipLaunchKernelGGL((k_ns_gemm<128, NP, KIND, 2>), dim3(head), dim3(256), 0, s, M, Part{0, 0, odd, last, 0, nullptr});
    if (head < tiles) hipLaunchKernelGGL((k_ns_gemm<64, NP, KIND, 4>), dim3(4 * (tiles - head)), dim3(256), 0, s, M, Part{head, 1, odd, last, 0, nullptr});
}
template <int NP>
hipError_t run_steps(Mats& M, bool may128, float* partial, hipStream_t s) {
    for (int step = 0; step < M.o.steps; step++) {
        run_gemm<NP, KIND_GRAM>(M, may128, partial, step & 1, 0, s);
        run_gemm<NP, KIND_POLY>(M, may128, partial, step & 1, 0, s);
        run_gemm<NP, KIND_APPLY>(M, may128, partial, step & 1, step + 1 == M.o.steps, s);
    }
    return hipGetLastError();
}

hipError_t run_group(Mats& M, int pad, bool one, float* partial, hipStream_t s) {
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
    return one ? run_steps<1>(M, pad == 128, partial, s) : run_steps<3>(M, pad == 128, partial, s);
}

// Room for the partial sums of split products: a launch has at most SPLIT_GOAL pieces and one more per tile (the last of each), and no
// more pieces than stages / SPLIT_MIN + 1 per tile.
int64_t partial_bytes(const OrthoMatrix* q, int count) {
    int64_t small = 0, most = 0;
    for (int i = 0; i < count; i++) {
        if (q[i].rows <= 0 || q[i].cols <= 0) continue;
        const int64_t s = q[i].rows < q[i].cols ? q[i].rows : q[i].cols, l = q[i].rows < q[i].cols ? q[i].cols : q[i].rows;
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
    // matrices of one padding and precision share their launches
    for (int pad = 64; pad <= 128; pad += 64)
        for (int one = 0; one < 2; one++) {
            Mats M;
            M.o = o;
            M.count = 0;
            float* partial = static_cast<float*>(ws);
            char* base = static_cast<char*>(ws) + partial_bytes(q, count);
            for (int i = 0; i < count; i++) {
                if (q[i].rows <= 0 || q[i].cols <= 0) continue;
                if (pad_of(q[i].rows, q[i].cols) == pad && one_product(q[i], o) == (one != 0)) {
                    Mat m;
                    layout(q[i], base, &m);
                    int at = M.count++;  // longest first: their workgroups run longest
                    for (; at > 0 && M.m[at - 1].lp < m.lp; at--) M.m[at] = M.m[at - 1];
                    M.m[at] = m;
                    if (M.count == MAX_MATS) {
                        const hipError_t e = run_group(M, pad, one != 0, partial, s);
                        if (e != hipSuccess) return e;
                        M.count = 0;
                    }
                }
                base += layout(q[i], nullptr, nullptr);
            }
            if (M.count) {
                const hipError_t e = run_group(M, pad, one != 0, partial, s);
                if (e != hipSuccess) return e;
            }
        }
    return hipSuccess;
}
}  // namespace qzl
