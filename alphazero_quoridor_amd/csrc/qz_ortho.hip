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
constexpr int MAX_PARTS = 512;    // partial sums of |U|^2 per matrix

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
};
struct Mats {
    Mat m[MAX_MATS];
    int32_t start[MAX_MATS + 1];  // first workgroup of each matrix in this launch
    int32_t count;
    OrthoStep o;
};
static_assert(sizeof(Mats) + 64 <= 4096, "kernel arguments");

__device__ __forceinline__ int find_mat(const Mats& M, int wg) {
    int i = 0;
    while (i + 1 < M.count && wg >= M.start[i + 1]) i++;
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
    const int64_t size = (int64_t)m.rows * m.cols;
    float* u = reinterpret_cast<float*>(m.xt1);
    double s = 0.0;
    for (int64_t e = (int64_t)wg * 256 + threadIdx.x; e < size; e += (int64_t)m.nparts * 256) {
        const int64_t r = e / m.cols, c = e - r * m.cols;
        float v = load_elem(m.update, r * m.ld + c, M.o.dtype);
        if (M.o.muon) {
            const float old = m.momentum[e], mom = old + (v - old) * (1.f - M.o.momentum);
            m.momentum[e] = mom;
            v = M.o.nesterov ? v + (mom - v) * M.o.momentum : mom;
            u[e] = v;
        }
        s += (double)v * (double)v;
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

template <int T>
struct GemmShared {
    half8 p[2][2][T * 4];  // [stage][hi | lo][row, chunk]
    half8 q[2][2][T * 4];
};

template <int T, int NP, int KIND>
__global__ __launch_bounds__(256, 2) void k_ns_gemm(Mats M, int odd, int last) {
    constexpr int NPL = NP == 3 ? 2 : 1;  // planes read
    constexpr int W = T / 64;             // 32 x 32 tiles per wave and side
    constexpr int LD = T * 4 / 256;       // 16-byte chunks per thread, operand and plane
    __shared__ GemmShared<T> sm;
    const int i = find_mat(M, blockIdx.x);
    const Mat& m = M.m[i];
    int wg = blockIdx.x - M.start[i];
    int ti, tj;  // tile of P rows, of Q rows
    if (KIND == KIND_APPLY) {
        const int tn = m.sp / T;
        ti = wg / tn;
        tj = wg % tn;
    } else {  // lower triangle, row by row
        ti = (int)((sqrtf(8.f * (float)wg + 1.f) - 1.f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= wg) ti++;
        while (ti * (ti + 1) / 2 > wg) ti--;
        tj = wg - ti * (ti + 1) / 2;
    }
    const int K = KIND == KIND_GRAM ? m.lp : m.sp;
    const _Float16* P = KIND == KIND_GRAM ? m.x : KIND == KIND_POLY ? m.a : (odd ? m.xt1 : m.xt0);
    const _Float16* Q = KIND == KIND_GRAM ? m.x : KIND == KIND_POLY ? m.a : m.b;
    const int64_t p_plane = KIND == KIND_POLY ? (int64_t)m.sp * m.sp : (int64_t)m.sp * m.lp;
    const int64_t q_plane = KIND == KIND_GRAM ? (int64_t)m.sp * m.lp : (int64_t)m.sp * m.sp;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave >> 1) * (T / 2), wn = (wave & 1) * (T / 2);
    const int r32 = lane & 31, h = lane >> 5;

    half8 rp[NPL][LD], rq[NPL][LD];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int pl = 0; pl < NPL; pl++)
#pragma unroll
            for (int t = 0; t < LD; t++) {
                const int c = tid + 256 * t, row = c >> 2, q = c & 3;
                rp[pl][t] = *reinterpret_cast<const half8*>(P + pl * p_plane + (int64_t)(ti * T + row) * K + k0 + q * 8);
                rq[pl][t] = *reinterpret_cast<const half8*>(Q + pl * q_plane + (int64_t)(tj * T + row) * K + k0 + q * 8);
            }
    };
    auto place = [&](int st) {
#pragma unroll
        for (int pl = 0; pl < NPL; pl++)
#pragma unroll
            for (int t = 0; t < LD; t++) {
                const int c = tid + 256 * t, row = c >> 2, q = c & 3;
                sm.p[st][pl][row * 4 + (q ^ ((row >> 2) & 3))] = rp[pl][t];
                sm.q[st][pl][row * 4 + (q ^ ((row >> 2) & 3))] = rq[pl][t];
            }
    };
    floatx16 acc[W][W];
#pragma unroll
    for (int x = 0; x < W; x++)
#pragma unroll
        for (int y = 0; y < W; y++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[x][y][e] = 0.f;

    fetch(0);
    place(0);
    __syncthreads();
    const int nk = K / BK;
    for (int k = 0; k < nk; k++) {
        const int st = k & 1;
        if (k + 1 < nk) fetch((k + 1) * BK);
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {  // 16 of K each
            half8 fp[NPL][W], fq[NPL][W];
#pragma unroll
            for (int pl = 0; pl < NPL; pl++)
#pragma unroll
                for (int x = 0; x < W; x++) {
                    const int rp_ = wm + 32 * x + r32, rq_ = wn + 32 * x + r32, q = 2 * kk + h;
                    fp[pl][x] = sm.p[st][pl][rp_ * 4 + (q ^ ((rp_ >> 2) & 3))];
                    fq[pl][x] = sm.q[st][pl][rq_ * 4 + (q ^ ((rq_ >> 2) & 3))];
                }
#pragma unroll
            for (int x = 0; x < W; x++)
#pragma unroll
                for (int y = 0; y < W; y++) {
                    if (NP == 3) {
                        acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[NPL - 1][x], fq[0][y], acc[x][y], 0, 0, 0);
                        acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][x], fq[NPL - 1][y], acc[x][y], 0, 0, 0);
                    }
                    acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][x], fq[0][y], acc[x][y], 0, 0, 0);
                }
        }
        if (k + 1 < nk) place(st ^ 1);
        __syncthreads();
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
                    const int64_t plane = (int64_t)m.sp * m.sp;
                    _Float16* dst = KIND == KIND_GRAM ? m.a : m.b;
                    half4 hi, lo;
                    if (KIND == KIND_POLY) {  // b A + c A A; A[row][col] = A[col][row]
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
                    if (ti != tj) {  // the mirrored tile (a tile on the diagonal holds both halves already, equal bit for bit)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            dst[(int64_t)(row + e) * m.sp + col] = hi[e];
                            dst[plane + (int64_t)(row + e) * m.sp + col] = lo[e];
                        }
                    }
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

// ================================================================ host side
int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// Tiles of 128 for shorter sides from 512 on (a 512 x 512 product is then 16 tiles: small ones rather spread over more CUs).
int tile_of(int64_t rows, int64_t cols) { return (rows < cols ? rows : cols) >= 512 ? 128 : 64; }
bool one_product(const OrthoMatrix& q, const OrthoStep& o) { return !o.muon && o.dtype == 1 && (q.rows < q.cols ? q.rows : q.cols) >= 256; }

int64_t layout(const OrthoMatrix& q, char* base, Mat* m) {
    const int64_t s = q.rows < q.cols ? q.rows : q.cols, l = q.rows < q.cols ? q.cols : q.rows;
    const int T = tile_of(q.rows, q.cols);
    const int64_t sp = align_up(s, T), lp = align_up(l, T);
    const int64_t xb = align_up(sp * lp * 4, 256), ab = align_up(sp * sp * 4, 256), pb = MAX_PARTS * 8;
    if (m) {
        int64_t parts = (q.rows * q.cols + 4095) / 4096;
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

template <int T, int NP>
hipError_t run_steps(Mats& M, hipStream_t s) {
    for (int step = 0; step < M.o.steps; step++) {
        int wgs = 0;
        for (int i = 0; i < M.count; i++) {
            M.start[i] = wgs;
            const int t = M.m[i].sp / T;
            wgs += t * (t + 1) / 2;
        }
        hipLaunchKernelGGL((k_ns_gemm<T, NP, KIND_GRAM>), dim3(wgs), dim3(256), 0, s, M, step & 1, 0);
        hipLaunchKernelGGL((k_ns_gemm<T, NP, KIND_POLY>), dim3(wgs), dim3(256), 0, s, M, step & 1, 0);
        wgs = 0;
        for (int i = 0; i < M.count; i++) {
            M.start[i] = wgs;
            wgs += (M.m[i].sp / T) * (M.m[i].lp / T);
        }
        hipLaunchKernelGGL((k_ns_gemm<T, NP, KIND_APPLY>), dim3(wgs), dim3(256), 0, s, M, step & 1, step + 1 == M.o.steps);
    }
    return hipGetLastError();
}

hipError_t run_group(Mats& M, int tile, bool one, hipStream_t s) {
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
    if (tile == 128) return one ? run_steps<128, 1>(M, s) : run_steps<128, 3>(M, s);
    return one ? run_steps<64, 1>(M, s) : run_steps<64, 3>(M, s);
}

}  // namespace

namespace qzl {
int64_t ortho_workspace_bytes(const OrthoMatrix* q, int count, const OrthoStep&) {
    int64_t n = 0;
    for (int i = 0; i < count; i++)
        if (q[i].rows > 0 && q[i].cols > 0) n += layout(q[i], nullptr, nullptr);
    return n;
}

hipError_t orthogonalize(const OrthoMatrix* q, int count, const OrthoStep& o, void* ws, hipStream_t s) {
    // matrices of one tile size and precision share their launches
    for (int tile = 64; tile <= 128; tile += 64)
        for (int one = 0; one < 2; one++) {
            Mats M;
            M.o = o;
            M.count = 0;
            char* base = static_cast<char*>(ws);
            for (int i = 0; i < count; i++) {
                if (q[i].rows <= 0 || q[i].cols <= 0) continue;
                if (tile_of(q[i].rows, q[i].cols) == tile && one_product(q[i], o) == (one != 0)) {
                    layout(q[i], base, &M.m[M.count++]);
                    if (M.count == MAX_MATS) {
                        const hipError_t e = run_group(M, tile, one != 0, s);
                        if (e != hipSuccess) return e;
                        M.count = 0;
                    }
                }
                base += layout(q[i], nullptr, nullptr);
            }
            if (M.count) {
                const hipError_t e = run_group(M, tile, one != 0, s);
                if (e != hipSuccess) return e;
            }
        }
    return hipSuccess;
}
}  // namespace qzl
