// qz_policy.hip -- log-probabilities of actions and the clipped policy loss, forward and backward.
//
// A row is one decision: n_actions logits z, a legal set, the action a that was taken.
//   p_j = exp(z_j - lse) over the legal columns, lse = log sum_legal exp z_j,
//   log pi(a) = z_a - lse, taken as (z_a - m) - log s (m may be a mask's lowest value, next to which log s would vanish),
//   H = lse - sum p_j z_j = log s - t / s with s = sum e^(z-m), t = sum e^(z-m) (z-m), m = max z
//   (both terms of the last form are >= 0: no cancellation).
// The loss of a row (w = its weight, A = its advantage, r = exp(log pi(a) - old)):
//   L = w [ -min(r A, clip(r, 1 - lo, 1 + hi) A) + beta KL - eta H ]
//   KL over a frozen policy's logits: sum q (log q - log p), computed as sum q (e^x - 1 - x), x = log p - log q: every
//   term is >= 0 and an error of lse cancels to first order, where the plain sum loses all digits of a small KL.
//   From the frozen policy's log-probability of a alone: e^x - 1 - x with x = log q(a) - log p(a), whose mean over actions drawn from p is
//   KL(p || q), the other direction.
//   dL/dz_j = w [ c (delta_ja - p_j) + beta (p_j - q_j) + eta p_j (log p_j + H) ],
//   c = -A r where the ratio is not clipped, minus beta (e^x - 1) for the second form of KL.
// A row whose action is negative, out of range, illegal or has a logit of -inf is LEFT OUT: zero loss, gradient, KL and
// entropy.  Illegal columns are never read into arithmetic (they may hold NaN or infinities) and get a zero gradient.
// All sums are float32 (row) and float64 (over rows), in an order fixed by the shape: results repeat bit for bit.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qz_policy.h"

#pragma clang fp contract(fast)

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float NEG_INF = -__builtin_huge_valf();

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log_fast(float x) { return __builtin_amdgcn_logf(x) * LN2; }

// ---- elements: V of them are 16 bytes.  Rows may start at any element (odd widths): the 16-byte accesses are declared with
// the element's alignment, which the hardware serves in one instruction.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int V = 4;
    static __device__ __forceinline__ float get(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void put(void* p, int64_t i, float v) { static_cast<float*>(p)[i] = v; }
};
template <>
struct Elem<__hip_bfloat16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ float get(const void* p, int64_t i) {
        return __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
    }
    static __device__ __forceinline__ void put(void* p, int64_t i, float v) { static_cast<__bf16*>(p)[i] = (__bf16)v; }
};
template <>
struct Elem<__half> {
    static constexpr int V = 8;
    static __device__ __forceinline__ float get(const void* p, int64_t i) { return (float)static_cast<const _Float16*>(p)[i]; }
    static __device__ __forceinline__ void put(void* p, int64_t i, float v) { static_cast<_Float16*>(p)[i] = (_Float16)v; }
};

struct Raw {
    uint32_t w[4];
};
template <typename T>
__device__ __forceinline__ Raw load_chunk(const void* row, int64_t j0, int n) {
    Raw r = {{0u, 0u, 0u, 0u}};
    if (j0 + Elem<T>::V <= n) {
        __builtin_memcpy(&r, static_cast<const T*>(row) + j0, 16);
    } else if (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (j0 + k < n) r.w[k] = static_cast<const uint32_t*>(row)[j0 + k];
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (j0 + k < n) r.w[k >> 1] |= (uint32_t) static_cast<const uint16_t*>(row)[j0 + k] << (16 * (k & 1));
    }
    return r;
}
template <typename T>
__device__ __forceinline__ float chunk_get(const Raw& r, int k);
template <>
__device__ __forceinline__ float chunk_get<float>(const Raw& r, int k) { return __uint_as_float(r.w[k]); }
template <>
__device__ __forceinline__ float chunk_get<__hip_bfloat16>(const Raw& r, int k) {
    return __uint_as_float((k & 1) ? (r.w[k >> 1] & 0xFFFF0000u) : (r.w[k >> 1] << 16));
}
template <>
__device__ __forceinline__ float chunk_get<__half>(const Raw& r, int k) {
    const uint16_t h = (uint16_t)(r.w[k >> 1] >> (16 * (k & 1)));
    return (float)__builtin_bit_cast(_Float16, h);
}
template <typename T>
__device__ __forceinline__ void store_full(T* at, const float* v) {
    Raw r;
    if (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; k++) r.w[k] = __float_as_uint(v[k]);
    } else if (__is_same(T, __half)) {
#pragma unroll
        for (int k = 0; k < 4; k++)
            r.w[k] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * k]) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * k + 1]) << 16;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            r.w[k] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2 * k]) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)v[2 * k + 1]) << 16;
    }
    __builtin_memcpy(at, &r, 16);
}
template <typename T>
__device__ __forceinline__ void store_chunk(void* row, int64_t j0, int n, const float* v) {
    if (j0 + Elem<T>::V <= n) {
        store_full<T>(static_cast<T*>(row) + j0, v);
    } else {
#pragma unroll
        for (int k = 0; k < Elem<T>::V; k++)
            if (j0 + k < n) Elem<T>::put(row, j0 + k, v[k]);
    }
}

// ---- legal sets: bit k of the result <=> column j0 + k exists and is legal
template <int V>
__device__ __forceinline__ uint32_t legal_bits(const PolicyRows& R, int64_t row, int64_t j0) {
    const int64_t left = (int64_t)R.a - j0;
    if (left <= 0) return 0u;
    const uint32_t inside = left >= V ? (1u << V) - 1u : (1u << (int)left) - 1u;
    if (R.legal_kind == 0) return inside;
    if (R.legal_kind == 1) {  // V divides 32 and j0 is a multiple of V: the bits sit in one word
        const uint32_t w = static_cast<const uint32_t*>(R.legal)[row * R.legal_ld + (j0 >> 5)];
        return (w >> (j0 & 31)) & inside;
    }
    const uint8_t* b = static_cast<const uint8_t*>(R.legal) + row * R.legal_ld + j0;
    uint32_t m = 0u;
    if (left >= V) {
        uint8_t t[V];
        __builtin_memcpy(t, b, V);
#pragma unroll
        for (int k = 0; k < V; k++) m |= (t[k] ? 1u : 0u) << k;
    } else {
#pragma unroll
        for (int k = 0; k < V; k++)
            if (k < left) m |= (b[k] ? 1u : 0u) << k;
    }
    return m;
}
__device__ __forceinline__ bool legal_one(const PolicyRows& R, int64_t row, int64_t j) {
    if (R.legal_kind == 0) return true;
    if (R.legal_kind == 1) return (static_cast<const uint32_t*>(R.legal)[row * R.legal_ld + (j >> 5)] >> (j & 31)) & 1u;
    return static_cast<const uint8_t*>(R.legal)[row * R.legal_ld + j] != 0;
}

// ---- one row's statistics
struct Stat {
    float m, s, t;  // max, sum e^(z-m), sum e^(z-m) (z-m)
};
__device__ __forceinline__ Stat stat_empty() { return {NEG_INF, 0.f, 0.f}; }
__device__ __forceinline__ Stat stat_join(const Stat& a, const Stat& b) {
    // an empty side has m = -inf, s = t = 0; a NaN on either side stays (its s is NaN)
    const float m = fmaxf(a.m, b.m);
    const float da = a.m == m ? 0.f : a.m - m, db = b.m == m ? 0.f : b.m - m;
    const float ea = a.s == 0.f ? 0.f : exp2_fast(da * LOG2E), eb = b.s == 0.f ? 0.f : exp2_fast(db * LOG2E);
    Stat r;
    r.m = m;
    r.s = a.s * ea + b.s * eb;
    r.t = (ea != 0.f ? (a.t + a.s * da) * ea : 0.f * a.t) + (eb != 0.f ? (b.t + b.s * db) * eb : 0.f * b.t);
    return r;
}
__device__ __forceinline__ float stat_log(const Stat& s) { return log_fast(s.s); }
__device__ __forceinline__ float stat_entropy(const Stat& s) { return fmaxf(log_fast(s.s), 0.f) - s.t / s.s; }

// the action's row: live = the action is in range, legal and its logit is not -inf
template <typename T>
__device__ __forceinline__ bool row_live(const PolicyRows& R, int64_t row, int64_t& act, float& za) {
    act = R.actions[row];
    za = 0.f;
    if (act < 0 || act >= R.a || !legal_one(R, row, act)) return false;
    za = Elem<T>::get(static_cast<const T*>(R.logits) + row * R.ld, act);
    return za != NEG_INF;
}

struct Coef {      // what the gradient of a row needs
    float m, ls, h, c, beta, eta, mq, lsq;  // max and log of the sum, of pi and the frozen policy; c, beta, eta carry the row's weight
    int64_t act;
    bool on;  // false: weight 0, no gradient whatever the row holds
};
struct RowOut {
    float logp, loss;  // loss without its KL over logits
    Coef g;
};
// (e^x - 1 - x) / x^2 for |x| < 1/2, from the series to x^5 / 7!: what is left out is below 2^-6 / 8! of 0.4 or more, 1e-6, at the
// edge and falls with x^6.  In KL's terms the series goes that far, and not only to where p - q - q x cancels: p and q each carry
// the error of their own lse, x that of the difference, and q (e^x - 1 - x) is consistent in itself, so that a common error of x only
// counts squared.
__device__ __forceinline__ float series2(float x) {
    float r = 1.f / 5040.f;
    r = r * x + 1.f / 720.f;
    r = r * x + 1.f / 120.f;
    r = r * x + 1.f / 24.f;
    r = r * x + 1.f / 6.f;
    return r * x + 0.5f;
}
__device__ __forceinline__ float expm1_minus_x(float x) {  // e^x - 1 - x >= 0
    return fabsf(x) < 0.5f ? series2(x) * x * x : expf(x) - 1.f - x;
}
// e^x - 1, the derivative of that: by itself, since adding x back to it gives inf - inf where x = -inf, and 0 for -1 past 2^24
__device__ __forceinline__ float expm1_near(float x) { return fabsf(x) < 0.5f ? series2(x) * x * x + x : expf(x) - 1.f; }
__device__ __forceinline__ RowOut row_terms(const PolicyTerms& P, int64_t row, int64_t act, float za, const Stat& st, const Stat& sq, float scale) {
    RowOut o;
    const float h = stat_entropy(st);
    o.g.m = st.m;
    o.g.ls = stat_log(st);
    o.g.mq = sq.m;
    o.g.lsq = stat_log(sq);
    o.logp = (za - o.g.m) - o.g.ls;
    const float w = P.weights ? P.weights[row] : P.default_weight;
    const float adv = P.advantages[row], r = expf(o.logp - P.old_logp[row]);
    const float open = r * adv, held = fminf(fmaxf(r, 1.f - P.clip_low), 1.f + P.clip_high) * adv;
    // a NaN ratio or advantage must reach the loss and the gradient: the comparisons are written so that it takes their first branch
    const bool held_wins = held < open;
    float c = held_wins ? 0.f : -open;
    o.loss = held_wins ? -held : -open;
    if (P.ref_logp && P.kl_coef != 0.f) {  // (a factor of 0: an infinite KL takes no part)
        const float x = P.ref_logp[row] - o.logp;
        o.loss += P.kl_coef * expm1_minus_x(x);
        c -= P.kl_coef * expm1_near(x);
    }
    o.loss -= P.entropy_coef * h;
    const bool on = w != 0.f;
    o.loss = on ? w * o.loss : 0.f;
    const float ws = w * scale;
    o.g.h = h;
    o.g.c = on ? ws * c : 0.f;
    o.g.beta = on && P.ref_logits ? ws * P.kl_coef : 0.f;
    o.g.eta = on ? ws * P.entropy_coef : 0.f;
    o.g.act = act;
    o.g.on = on;
    return o;
}
// what KL over the frozen policy's logits adds to the loss: nothing where a factor is 0, infinite or NaN as it may be
__device__ __forceinline__ double kl_part(const PolicyTerms& P, bool live, float w, float kl) {
    return P.ref_logits && live && w != 0.f && P.kl_coef != 0.f ? (double)w * P.kl_coef * kl : 0.0;
}
__device__ __forceinline__ float kl_taken(const PolicyTerms& P, int64_t row, float logp) { return P.ref_logp ? expm1_minus_x(P.ref_logp[row] - logp) : 0.f; }

// one column: gradient, and the column's term of KL over logits.  p = 0 (a logit of -inf) gives 0 log 0 = 0; q = 0 < p has no KL
// term but p; q > 0 = p is an infinite KL, as it should be.
__device__ __forceinline__ float column(const Coef& g, bool has_q, float z, float zq, int64_t j, float& kl) {
    const float dz = z - g.m, lp = dz - g.ls;
    const float p = exp2_fast(lp * LOG2E);
    float d = p * (g.eta * ((p > 0.f || lp != lp ? lp : 0.f) + g.h) - g.c);
    if (has_q) {
        const float dq = zq - g.mq, lq = dq - g.lsq, q = exp2_fast(lq * LOG2E);
        const float x = (dz - dq) - (g.ls - g.lsq);
        const float f = fabsf(x) < 0.5f ? q * (series2(x) * x * x) : q == 0.f ? p : (p - q) - q * x;
        kl += f;
        if (g.beta != 0.f) d += g.beta * (p - q);
    }
    if (j == g.act) d += g.c;
    return g.on ? d : 0.f;
}

// ---- reductions
template <typename F>
__device__ __forceinline__ float wave_reduce(float v, F f) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    return wave_reduce(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
// of 2 FROM neighbouring lanes
template <int FROM>
__device__ __forceinline__ Stat wave_join(Stat s) {
#pragma unroll
    for (int o = FROM; o > 0; o >>= 1) {
        Stat b = {__shfl_xor(s.m, o), __shfl_xor(s.s, o), __shfl_xor(s.t, o)};
        // both lanes of a pair join in the same order, so that all lanes end with the same bits
        s = (threadIdx.x & o) ? stat_join(b, s) : stat_join(s, b);
    }
    return s;
}
template <int NT>
__device__ __forceinline__ Stat block_join(Stat s, float* sh /*[3 * NT / 64]*/) {
    constexpr int NW = NT / 64;
    s = wave_join<32>(s);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        sh[3 * wave] = s.m;
        sh[3 * wave + 1] = s.s;
        sh[3 * wave + 2] = s.t;
    }
    __syncthreads();
    const int w = threadIdx.x & (NW - 1);  // every wave joins all of them, a lane each: one after the other took 1 us of sixteen waves
    const Stat r = wave_join<NW / 2>(Stat{sh[3 * w], sh[3 * w + 1], sh[3 * w + 2]});
    __syncthreads();
    return r;
}
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* sh) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float r = sh[0];
    for (int w = 1; w < NT / 64; w++) r += sh[w];
    __syncthreads();
    return r;
}

// ---- illegal columns as -inf, in the packed words
template <typename T>
struct NegInf {
    static constexpr uint32_t pair = __is_same(T, __half) ? 0xFC00FC00u : __is_same(T, float) ? 0xFF800000u : 0xFF80FF80u;
};
template <typename T>
__device__ __forceinline__ Raw raw_empty() {
    return {{NegInf<T>::pair, NegInf<T>::pair, NegInf<T>::pair, NegInf<T>::pair}};
}
// columns whose bit of ok is clear become -inf
template <typename T>
__device__ __forceinline__ void raw_mask(Raw& raw, uint32_t ok) {
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (sizeof(T) == 4) {
            raw.w[w] = (ok >> w) & 1u ? raw.w[w] : NegInf<T>::pair;
        } else {
            const uint32_t keep = ((ok >> (2 * w)) & 1u ? 0x0000FFFFu : 0u) | ((ok >> (2 * w + 1)) & 1u ? 0xFFFF0000u : 0u);
            raw.w[w] = (raw.w[w] & keep) | (NegInf<T>::pair & ~keep);
        }
    }
}
// the same from a mask of bytes, four at a time: 0xFF in every non-zero byte, spread over its column's bits
template <typename T>
__device__ __forceinline__ void raw_mask_bytes(Raw& raw, const uint8_t* b) {
    uint32_t w[2] = {0u, 0u};
    __builtin_memcpy(w, b, Elem<T>::V);
#pragma unroll
    for (int i = 0; i < Elem<T>::V / 4; i++) {
        uint32_t t = (((w[i] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | w[i]) & 0x80808080u;
        t |= t - (t >> 7);
#pragma unroll
        for (int k = 0; k < (sizeof(T) == 4 ? 4 : 2); k++) {
            const uint32_t keep = __builtin_amdgcn_perm(0u, t, sizeof(T) == 4 ? 0x01010101u * k : k ? 0x03030202u : 0x01010000u);
            uint32_t& v = raw.w[sizeof(T) == 4 ? k : 2 * i + k];
            v = (v & keep) | (NegInf<T>::pair & ~keep);
        }
    }
}
// the legal columns j0 .. j0 + V - 1 of a row, illegal and missing ones as -inf
template <typename T>
__device__ __forceinline__ Raw load_legal(const PolicyRows& R, const void* row, int64_t r, int64_t j0) {
    constexpr int V = Elem<T>::V;
    Raw raw = load_chunk<T>(row, j0, R.a);
    if (R.legal_kind == 2 && j0 + V <= R.a) raw_mask_bytes<T>(raw, static_cast<const uint8_t*>(R.legal) + r * R.legal_ld + j0);
    else if (R.legal_kind != 0 || j0 + V > R.a) raw_mask<T>(raw, legal_bits<V>(R, r, j0));
    return raw;
}

// the statistics of the columns that one thread visits, online: one running (m, s, t), rescaled where a chunk brings a new maximum.
// m starts at the lowest finite value, so that a chunk of -inf only adds exp(-inf) = 0; a NaN reaches s, which keeps it.
constexpr float LOWEST = -3.402823466e38f;
template <typename T>
__device__ __forceinline__ void stat_chunk(Stat& st, const Raw& raw) {
    constexpr int V = Elem<T>::V;
    float cm = chunk_get<T>(raw, 0);
#pragma unroll
    for (int k = 1; k < V; k++) cm = fmaxf(cm, chunk_get<T>(raw, k));
    if (cm > st.m) {
        const float d = fmaxf(st.m - cm, LOWEST), e = exp2_fast(d * LOG2E);
        st.t = e != 0.f ? (st.t + st.s * d) * e : 0.f * st.t;
        st.s *= e;
        st.m = cm;
    }
#pragma unroll
    for (int k = 0; k < V; k++) {
        const float x = chunk_get<T>(raw, k) - st.m, e = exp2_fast(x * LOG2E);
        st.s += e;
        st.t += e * fmaxf(x, -1e30f);
    }
}

// ---- a row's gradient
// One column without branches, for rows whose coefficients are finite: the same values as column().  -inf in both inputs (an illegal
// column) gives 0 and no term of KL; x is held below 1e30 so that q = 0 gives the term p and not 0 inf.
struct FastCoef {
    float m, ls, mq, lsqb, c, eta, eh, beta, shift;  // lsqb = lsq log2 e, eh = eta h - c, shift = ls - lsq
};
template <bool HAS_Q>
__device__ __forceinline__ float column_fast(const FastCoef& g, float z, float zq, float& kl) {
    const float dz = z - g.m, lp = dz - g.ls, p = exp2_fast(lp * LOG2E);
    float d = p * (g.eta * fmaxf(lp, -1e30f) + g.eh);
    if (HAS_Q) {
        const float dq = zq - g.mq, q = exp2_fast(dq * LOG2E - g.lsqb), x = fminf((dz - dq) - g.shift, 1e30f), pq = p - q;
        const float qx = q * x, near = qx * (x * series2(x)), far = pq - qx;
        kl += fabsf(x) < 0.5f ? near : far;
        d += g.beta * pq;
    }
    return d;
}
// a row with an infinite or NaN coefficient: its gradient column by column from memory
template <typename T, int NT>
__device__ __forceinline__ float row_gradient_slow(const PolicyRows& R, const PolicyTerms& P, const PolicyOut& O, int64_t row, const Coef& g, int64_t j0 = 0, int64_t j1 = INT64_MAX) {
    float kl = 0.f;
    const bool has_q = P.ref_logits != nullptr;
#pragma unroll 1
    for (int64_t j = j0 + threadIdx.x; j < (j1 < R.a ? j1 : R.a); j += NT) {
        float d = 0.f;
        if (legal_one(R, row, j))
            d = column(g, has_q, Elem<T>::get(static_cast<const T*>(R.logits) + row * R.ld, j), has_q ? Elem<T>::get(static_cast<const T*>(P.ref_logits) + row * P.ref_ld, j) : 0.f, j, kl);
        if (O.grad) Elem<T>::put(static_cast<T*>(O.grad) + row * O.ld_grad, j, d);
    }
    return kl;
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_huge_valf(); }

__device__ __forceinline__ FastCoef fast_coef(const Coef& g) { return {g.m, g.ls, g.mq, g.lsq * LOG2E, g.c, g.eta, g.eta * g.h - g.c, g.beta, g.ls - g.lsq}; }
__device__ __forceinline__ bool all_finite(const FastCoef& g) {
    return finite(g.eh) && finite(g.eta) && finite(g.c) && finite(g.beta) && finite(g.shift) && finite(g.m);
}

// Measured: log-probabilities of 4,096 x 32,000 bfloat16 82 us (3.2 TB/s), their backward pass 90 us (5.8 TB/s, part of it from the caches).
// columns j0 .. j1 of a row from memory, two chunks in flight; -> this thread's part of KL
template <typename T, int RT, bool HAS_Q>
__device__ __forceinline__ float row_gradient(const PolicyRows& R, const PolicyOut& O, const FastCoef& g, const T* z, const T* zq, T* out, int64_t row, int act,
                                              int64_t j0, int64_t j1) {
    constexpr int V = Elem<T>::V, STEP = RT * V;
    float kl = 0.f;
    for (int64_t j = j0 + (int64_t)threadIdx.x * V; j < j1; j += 2 * STEP) {
        Raw r[2], q[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            r[c] = q[c] = raw_empty<T>();
            if (j + c * STEP < j1) {
                r[c] = load_legal<T>(R, z, row, j + c * STEP);
                if (HAS_Q) q[c] = load_legal<T>(R, zq, row, j + c * STEP);
            }
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int64_t at = j + c * STEP;
            if (at >= j1) break;
            float d[V];
#pragma unroll
            for (int k = 0; k < V; k++) d[k] = column_fast<HAS_Q>(g, chunk_get<T>(r[c], k), HAS_Q ? chunk_get<T>(q[c], k) : 0.f, kl);
            if ((uint64_t)(act - at) < (uint64_t)V) {
#pragma unroll
                for (int k = 0; k < V; k++) d[k] += act - at == k ? g.c : 0.f;
            }
            if (O.grad) store_chunk<T>(out, at, R.a, d);
        }
    }
    return kl;
}

// ================================================================ any width: one workgroup per row, the row read twice

// j0, j1: the columns of this workgroup (j0 a multiple of a chunk)
template <typename T, int RT>
__device__ __forceinline__ Stat row_stat(const PolicyRows& R, const void* base, int64_t ld, int64_t row, int64_t j0, int64_t j1, float* sh) {
    const T* z = static_cast<const T*>(base) + row * ld;
    constexpr int V = Elem<T>::V, STEP = RT * V;
    Stat st = {LOWEST, 0.f, 0.f};
    int64_t j = j0 + (int64_t)threadIdx.x * V;
    for (; j + 3 * STEP + V <= j1; j += 4 * STEP) {  // four chunks' loads in flight
        Raw r[4];
#pragma unroll
        for (int k = 0; k < 4; k++) r[k] = load_legal<T>(R, z, row, j + k * STEP);
#pragma unroll
        for (int k = 0; k < 4; k++) stat_chunk<T>(st, r[k]);
    }
    for (; j < j1; j += STEP) stat_chunk<T>(st, load_legal<T>(R, z, row, j));
    return block_join<RT>(st, sh);
}

template <typename T, int RT>
__global__ __launch_bounds__(RT) void k_action_logp(PolicyRows R, float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ stats) {
    __shared__ float sh[3 * RT / 64];
    const int64_t row = R.row0 + blockIdx.x;
    int64_t act;
    float za;
    const bool live = row_live<T>(R, row, act, za);
    Stat st = stat_empty();
    if (live) st = row_stat<T, RT>(R, R.logits, R.ld, row, 0, R.a, sh);
    if (threadIdx.x == 0) {
        const float ls = stat_log(st);
        logp[row] = live ? (za - st.m) - ls : act < 0 ? 0.f : NEG_INF;
        if (entropy) entropy[row] = live ? stat_entropy(st) : 0.f;
        if (stats) {
            stats[row] = live ? st.m : 0.f;
            stats[R.n + row] = live ? ls : 0.f;
        }
    }
}

constexpr int BT = 256;
template <typename T>
__global__ __launch_bounds__(BT) void k_action_logp_backward(PolicyRows R, const float* __restrict__ stats, const float* __restrict__ entropy,
                                                             const float* __restrict__ dlogp, const float* __restrict__ dentropy, void* __restrict__ grad,
                                                             int64_t ld_grad) {
    constexpr int V = Elem<T>::V;
    const int64_t row = R.row0 + blockIdx.x;
    int64_t act;
    float za;
    const bool live = row_live<T>(R, row, act, za);
    const T* z = static_cast<const T*>(R.logits) + row * R.ld;
    T* out = static_cast<T*>(grad) + row * ld_grad;
    const Coef g = {stats[row], stats[R.n + row], entropy ? entropy[row] : 0.f, dlogp ? dlogp[row] : 0.f, 0.f, dentropy ? -dentropy[row] : 0.f, 0.f, 0.f, act, true};
    for (int64_t j = ((int64_t)blockIdx.y * BT + threadIdx.x) * V; j < R.a; j += (int64_t)gridDim.y * BT * V) {
        const uint32_t ok = live ? legal_bits<V>(R, row, j) : 0u;
        const Raw raw = load_chunk<T>(z, j, R.a);
        float d[V], kl = 0.f;
#pragma unroll
        for (int k = 0; k < V; k++) d[k] = (ok >> k) & 1u ? column(g, false, chunk_get<T>(raw, k), 0.f, j + k, kl) : 0.f;
        store_chunk<T>(out, j, R.a, d);
    }
}

template <typename T, int RT>
__global__ __launch_bounds__(RT) void k_policy_loss(PolicyRows R, PolicyTerms P, PolicyOut O) {
    constexpr int V = Elem<T>::V;
    __shared__ float sh[3 * RT / 64];
    const float scale = O.scale ? *O.scale : 1.f;
    if (O.only_if_scaled && scale == 1.f) return;  // the gradient that the forward pass wrote is the one asked for
    const int64_t row = R.row0 + blockIdx.x;
    int64_t act;
    float za;
    const bool live = row_live<T>(R, row, act, za);
    T* out = static_cast<T*>(O.grad) + row * O.ld_grad;
    float kl = 0.f;
    RowOut o = {act < 0 ? 0.f : NEG_INF, 0.f, {}};
    float h = 0.f;
    if (live) {
        const Stat st = row_stat<T, RT>(R, R.logits, R.ld, row, 0, R.a, sh);
        const bool has_q = P.ref_logits != nullptr;
        const Stat sq = has_q ? row_stat<T, RT>(R, P.ref_logits, P.ref_ld, row, 0, R.a, sh) : Stat{0.f, 1.f, 0.f};
        h = stat_entropy(st);
        o = row_terms(P, row, act, za, st, sq, scale);
        const T* z = static_cast<const T*>(R.logits) + row * R.ld;
        const T* zq = static_cast<const T*>(P.ref_logits) + row * P.ref_ld;
        const FastCoef g = fast_coef(o.g);
        if (!all_finite(g)) {
            kl = row_gradient_slow<T, RT>(R, P, O, row, o.g);
        } else if (has_q) {
            kl = row_gradient<T, RT, true>(R, O, g, z, zq, out, row, (int)act, 0, R.a);
        } else if (O.grad) {
            row_gradient<T, RT, false>(R, O, g, z, zq, out, row, (int)act, 0, R.a);
        }
        kl = has_q ? block_sum<RT>(kl, sh) : kl_taken(P, row, o.logp);
    } else if (O.grad) {
        const float zero[V] = {};
        for (int64_t j = (int64_t)threadIdx.x * V; j < R.a; j += RT * V) store_chunk<T>(out, j, R.a, zero);
    }
    if (threadIdx.x == 0 && O.parts) {
        const float w = P.weights ? P.weights[row] : P.default_weight;
        O.logp[row] = o.logp;
        O.kl[row] = live ? kl : 0.f;
        O.entropy[row] = h;
        O.parts[row] = (double)o.loss + kl_part(P, live, w, kl);
    }
}

// ================================================================ few wide rows: several workgroups per row
// A CU alone draws some 40 GB/s from memory, so a row of 131,072 columns takes 10 us and more; S workgroups take pieces of it.  First
// launch: every piece's (m, s, t) of both inputs.  Second: each workgroup joins the row's S triples (in order, so that all agree bit
// for bit), and does its piece of the gradient and of KL.  Third: one workgroup sums KL and the loss.
constexpr int ST = 256, MAX_SPLIT = 64;
struct Split {
    int32_t s;       // pieces per row
    int32_t piece;   // columns of one, a multiple of ST chunks
    float* stats;    // [n][2][s][3]: logits, frozen policy
    float* kl;       // [n][s]
    float* coef;     // [n]: w kl_coef of rows with a KL over logits, else 0
};
template <typename T>
__global__ __launch_bounds__(ST) void k_split_stats(PolicyRows R, PolicyTerms P, Split S, const float* scale, int only_if_scaled) {
    __shared__ float sh[3 * ST / 64];
    if (only_if_scaled && *scale == 1.f) return;
    const int64_t row = blockIdx.y, j0 = (int64_t)blockIdx.x * S.piece, j1 = j0 + S.piece < R.a ? j0 + S.piece : R.a;
    for (int k = 0; k < (P.ref_logits ? 2 : 1); k++) {
        const Stat st = k == 0 ? row_stat<T, ST>(R, R.logits, R.ld, row, j0, j1, sh) : row_stat<T, ST>(R, P.ref_logits, P.ref_ld, row, j0, j1, sh);
        float* out = S.stats + ((row * 2 + k) * S.s + blockIdx.x) * 3;
        if (threadIdx.x < 3) out[threadIdx.x] = threadIdx.x == 0 ? st.m : threadIdx.x == 1 ? st.s : st.t;
    }
}
__device__ __forceinline__ Stat split_join(const Split& S, int64_t row, int k) {
    const int lane = threadIdx.x & 63;
    const float* in = S.stats + ((row * 2 + k) * S.s + lane) * 3;
    return wave_join<32>(lane < S.s ? Stat{in[0], in[1], in[2]} : Stat{LOWEST, 0.f, 0.f});
}
template <typename T>
__global__ __launch_bounds__(64) void k_split_logp(PolicyRows R, Split S, float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ stats) {
    const int64_t row = blockIdx.x;
    int64_t act;
    float za;
    const bool live = row_live<T>(R, row, act, za);
    const Stat st = split_join(S, row, 0);
    if (threadIdx.x == 0) {
        const float ls = stat_log(st);
        logp[row] = live ? (za - st.m) - ls : act < 0 ? 0.f : NEG_INF;
        if (entropy) entropy[row] = live ? stat_entropy(st) : 0.f;
        if (stats) {
            stats[row] = live ? st.m : 0.f;
            stats[R.n + row] = live ? ls : 0.f;
        }
    }
}
template <typename T>
__global__ __launch_bounds__(ST) void k_split_loss(PolicyRows R, PolicyTerms P, PolicyOut O, Split S) {
    constexpr int V = Elem<T>::V;
    __shared__ float sh[ST / 64];
    const float scale = O.scale ? *O.scale : 1.f;
    if (O.only_if_scaled && scale == 1.f) return;
    const int64_t row = blockIdx.y, j0 = (int64_t)blockIdx.x * S.piece, j1 = j0 + S.piece < R.a ? j0 + S.piece : R.a;
    int64_t act;
    float za;
    const bool live = row_live<T>(R, row, act, za), has_q = P.ref_logits != nullptr;
    T* out = static_cast<T*>(O.grad) + row * O.ld_grad;
    RowOut o = {act < 0 ? 0.f : NEG_INF, 0.f, {}};
    float kl = 0.f;
    if (live) {
        o = row_terms(P, row, act, za, split_join(S, row, 0), has_q ? split_join(S, row, 1) : Stat{0.f, 1.f, 0.f}, scale);
        const T* z = static_cast<const T*>(R.logits) + row * R.ld;
        const T* zq = static_cast<const T*>(P.ref_logits) + row * P.ref_ld;
        const FastCoef g = fast_coef(o.g);
        if (!all_finite(g)) kl = row_gradient_slow<T, ST>(R, P, O, row, o.g, j0, j1);
        else if (has_q) kl = row_gradient<T, ST, true>(R, O, g, z, zq, out, row, (int)act, j0, j1);
        else if (O.grad) row_gradient<T, ST, false>(R, O, g, z, zq, out, row, (int)act, j0, j1);
        if (has_q) kl = block_sum<ST>(kl, sh);
    } else if (O.grad) {
        const float zero[V] = {};
        for (int64_t j = j0 + (int64_t)threadIdx.x * V; j < j1; j += ST * V) store_chunk<T>(out, j, R.a, zero);
    }
    if (threadIdx.x == 0 && O.parts) {
        S.kl[row * S.s + blockIdx.x] = kl;
        if (blockIdx.x == 0) {
            const float w = P.weights ? P.weights[row] : P.default_weight;
            O.logp[row] = o.logp;
            O.entropy[row] = live ? o.g.h : 0.f;
            O.kl[row] = live && !has_q ? kl_taken(P, row, o.logp) : 0.f;
            O.parts[row] = (double)o.loss;
            S.coef[row] = has_q && live ? w * P.kl_coef : 0.f;
        }
    }
}
// rows' KL from their pieces, and the loss (n <= FEW_ROWS)
__global__ __launch_bounds__(256) void k_split_finish(PolicyOut O, Split S, int n, int has_q, float* __restrict__ loss) {
    __shared__ double sh[256];
    double total = 0.0;
    for (int row = threadIdx.x; row < n; row += 256) {
        double part = O.parts[row];
        if (has_q) {
            float kl = 0.f;
            for (int p = 0; p < S.s; p++) kl += S.kl[(int64_t)row * S.s + p];
            O.kl[row] = kl;
            if (S.coef[row] != 0.f) part += (double)S.coef[row] * kl;
        }
        total += part;
    }
    sh[threadIdx.x] = total;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = (float)sh[0];
}

// ================================================================ narrow rows: a wave per row, the row in registers
// Bound by launch and memory latency at the sizes that boards have (13,312 rows of 140: 7 us, 1.1 TB/s); four rows per workgroup.
template <typename T>
__device__ __forceinline__ float masked(const PolicyRows& R, int64_t row, const void* base, int64_t ld, int64_t j) {
    if (j >= R.a || !legal_one(R, row, j)) return NEG_INF;
    return Elem<T>::get(static_cast<const T*>(base) + row * ld, j);
}
// (m, s, t) of a row whose E values per lane are in registers (-inf: no such column, or an illegal one)
template <int E>
__device__ __forceinline__ Stat wave_stat(const float (&z)[E]) {
    float m = z[0];
#pragma unroll
    for (int e = 1; e < E; e++) m = fmaxf(m, z[e]);
    Stat st;
    st.m = wave_max(m);
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float x = z[e] - st.m, p = exp2_fast(x * LOG2E);
        s += p;
        t += p * fmaxf(x, -1e30f);  // (p = 0 where x is -inf)
    }
    st.s = wave_sum(s);
    st.t = wave_sum(t);
    return st;
}
template <typename T, int E>
__global__ __launch_bounds__(256) void k_wave_logp(PolicyRows R, float* __restrict__ logp, float* __restrict__ entropy, float* __restrict__ stats) {
    const int lane = threadIdx.x & 63;
    const int64_t row = R.row0 + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= R.n) return;
    float z[E];
#pragma unroll
    for (int e = 0; e < E; e++) z[e] = masked<T>(R, row, R.logits, R.ld, lane + 64 * e);
    int64_t act;
    float za;
    const bool live = row_live<T>(R, row, act, za);
    const Stat st = wave_stat<E>(z);
    if (lane == 0) {
        const float ls = stat_log(st);
        logp[row] = live ? (za - st.m) - ls : act < 0 ? 0.f : NEG_INF;
        if (entropy) entropy[row] = live ? stat_entropy(st) : 0.f;
        if (stats) {
            stats[row] = live ? st.m : 0.f;
            stats[R.n + row] = live ? ls : 0.f;
        }
    }
}
template <typename T, int E>
__global__ __launch_bounds__(256) void k_wave_loss(PolicyRows R, PolicyTerms P, PolicyOut O) {
    const float scale = O.scale ? *O.scale : 1.f;
    if (O.only_if_scaled && scale == 1.f) return;
    const int lane = threadIdx.x & 63;
    const int64_t row = R.row0 + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= R.n) return;
    const bool has_q = P.ref_logits != nullptr;
    float z[E], zq[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        z[e] = masked<T>(R, row, R.logits, R.ld, lane + 64 * e);
        zq[e] = has_q ? masked<T>(R, row, P.ref_logits, P.ref_ld, lane + 64 * e) : NEG_INF;
    }
    int64_t act;
    float za;
    const bool live = row_live<T>(R, row, act, za);
    RowOut o = {act < 0 ? 0.f : NEG_INF, 0.f, {}};
    float kl = 0.f, h = 0.f;
    if (live) {
        const Stat st = wave_stat<E>(z);
        const Stat sq = has_q ? wave_stat<E>(zq) : Stat{0.f, 1.f, 0.f};
        o = row_terms(P, row, act, za, st, sq, scale);
        h = o.g.h;
#pragma unroll
        for (int e = 0; e < E; e++) {
            // an illegal column is -inf in both: p = q = 0, its terms 0 (an infinite coefficient is kept out below)
            const float d = column(o.g, has_q, z[e], zq[e], lane + 64 * e, kl);
            z[e] = z[e] == NEG_INF && zq[e] == NEG_INF ? 0.f : d;
        }
        kl = has_q ? wave_sum(kl) : kl_taken(P, row, o.logp);
    }
    if (O.grad) {
        T* out = static_cast<T*>(O.grad) + row * O.ld_grad;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (lane + 64 * e < R.a) Elem<T>::put(out, lane + 64 * e, live ? z[e] : 0.f);
    }
    if (lane == 0 && O.parts) {
        const float w = P.weights ? P.weights[row] : P.default_weight;
        O.logp[row] = o.logp;
        O.kl[row] = live ? kl : 0.f;
        O.entropy[row] = h;
        O.parts[row] = (double)o.loss + kl_part(P, live, w, kl);
    }
}

// ================================================================ wide rows: a workgroup per row, the row in registers
// (8,192 x 32,768 bfloat16 with a frozen policy's logits, 1.6 GB: 410 us, 3.9 TB/s; a copy reaches 4.6.)
// One pass over memory: logits (and the frozen policy's) are read once, into registers as they are stored, illegal columns replaced by
// -inf on the way; then the maximum, the sums and the gradient come from the registers.  Bound by memory where there is one input, by
// vector instructions (~50 per column with two inputs) close behind it otherwise; two workgroups of 512 share a CU, so that one's
// arithmetic covers the other's loads.
template <typename T, int CH>
__device__ __forceinline__ float chunks_max(const Raw (&z)[CH]) {
    float m = NEG_INF;
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
        for (int k = 0; k < Elem<T>::V; k++) m = fmaxf(m, chunk_get<T>(z[c], k));
    return m;
}
// The compiler must not keep the unpacked values of one pass for the next (twice the registers, and spills): to it, the packed ones
// change between the passes.
template <int CH>
__device__ __forceinline__ void forget(Raw (&z)[CH]) {
#pragma unroll
    for (int c = 0; c < CH; c++) asm volatile("" : "+v"(z[c].w[0]), "+v"(z[c].w[1]), "+v"(z[c].w[2]), "+v"(z[c].w[3]));
}
template <int NT>
__device__ __forceinline__ void block_max2(float& a, float& b, float* sh) {
    a = wave_max(a);
    b = wave_max(b);
    if ((threadIdx.x & 63) == 0) {
        sh[threadIdx.x >> 6] = a;
        sh[16 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        a = fmaxf(a, sh[w]);
        b = fmaxf(b, sh[16 + w]);
    }
}
template <int NT>
__device__ __forceinline__ void block_sum3(float& a, float& b, float& c, float* sh) {
    a = wave_sum(a);
    b = wave_sum(b);
    c = wave_sum(c);
    if ((threadIdx.x & 63) == 0) {
        sh[threadIdx.x >> 6] = a;
        sh[16 + (threadIdx.x >> 6)] = b;
        sh[32 + (threadIdx.x >> 6)] = c;
    }
    __syncthreads();
    a = b = c = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        a += sh[w];
        b += sh[16 + w];
        c += sh[32 + w];
    }
}
// A thread holds CH chunks of 16 bytes, and the first few threads one column each of what is left over of the row.
template <typename T, int NT, int CH, bool HAS_Q, bool MASK>
__global__ __launch_bounds__(NT, 4) void k_row_loss(PolicyRows R, PolicyTerms P, PolicyOut O) {
    constexpr int V = Elem<T>::V;
    __shared__ float sh[3][48];
    const float scale = O.scale ? *O.scale : 1.f;
    if (O.only_if_scaled && scale == 1.f) return;
    const int64_t row = R.row0 + blockIdx.x;
    const T* zrow = static_cast<const T*>(R.logits) + row * R.ld;
    const T* qrow = static_cast<const T*>(P.ref_logits) + row * P.ref_ld;
    const int j0 = threadIdx.x * V, full = R.a / V * V, jt = full + threadIdx.x;
    Raw z[CH], q[HAS_Q ? CH : 1] = {};
#pragma unroll
    for (int c = 0; c < CH; c++) {
        z[c] = raw_empty<T>();
        if (HAS_Q) q[c] = raw_empty<T>();
        const int j = j0 + c * NT * V;
        if (j < full) {
            __builtin_memcpy(&z[c], zrow + j, 16);
            if (HAS_Q) __builtin_memcpy(&q[c], qrow + j, 16);
        }
    }
    if (MASK && R.legal_kind == 2) {
        const uint8_t* b = static_cast<const uint8_t*>(R.legal) + row * R.legal_ld;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int j = j0 + c * NT * V;
            if (j < full) {
                raw_mask_bytes<T>(z[c], b + j);
                if (HAS_Q) raw_mask_bytes<T>(q[c], b + j);
            }
        }
    } else if (MASK) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int j = j0 + c * NT * V;
            if (j < full) {
                const uint32_t ok = legal_bits<V>(R, row, j);
                raw_mask<T>(z[c], ok);
                if (HAS_Q) raw_mask<T>(q[c], ok);
            }
        }
    }
    const float zt = masked<T>(R, row, R.logits, R.ld, jt), qt = HAS_Q ? masked<T>(R, row, P.ref_logits, P.ref_ld, jt) : NEG_INF;
    int64_t act;
    float za;
    const bool live = row_live<T>(R, row, act, za);
    T* out = static_cast<T*>(O.grad) + row * O.ld_grad;
    RowOut o = {act < 0 ? 0.f : NEG_INF, 0.f, {}};
    float kl = 0.f, h = 0.f;
    if (live) {
        float m = fmaxf(chunks_max<T, CH>(z), zt), mq = 0.f;
        if (HAS_Q) mq = fmaxf(chunks_max<T, HAS_Q ? CH : 1>(q), qt);
        block_max2<NT>(m, mq, sh[0]);
        forget(z);
        forget(q);
        // sums in powers of two: y = (z - m) log2 e; t is turned back to natural units at the end
        float s = 0.f, t = 0.f, sq = 0.f;
        auto add = [&](float v, float u) {
            const float y = (v - m) * LOG2E, e = exp2_fast(y);
            s += e;
            t += e * fmaxf(y, -1e30f);
            if (HAS_Q) sq += exp2_fast((u - mq) * LOG2E);
        };
        add(zt, qt);
#pragma unroll
        for (int c = 0; c < CH; c++) {
#pragma unroll
            for (int k = 0; k < V; k++) add(chunk_get<T>(z[c], k), HAS_Q ? chunk_get<T>(q[c], k) : 0.f);
            __builtin_amdgcn_sched_barrier(0);  // (a chunk at a time: interleaved further, the values in between spill)
        }
        block_sum3<NT>(s, t, sq, sh[1]);
        forget(z);
        forget(q);
        o = row_terms(P, row, act, za, Stat{m, s, t * LN2}, HAS_Q ? Stat{mq, sq, 0.f} : Stat{0.f, 1.f, 0.f}, scale);
        h = o.g.h;
        const FastCoef g = fast_coef(o.g);
        if (!all_finite(g)) {
            kl = row_gradient_slow<T, NT>(R, P, O, row, o.g);
        } else if (O.grad || HAS_Q) {
            const int a32 = (int)act;
            const float dt = column_fast<HAS_Q>(g, zt, qt, kl) + (jt == a32 ? g.c : 0.f);
            if (O.grad && jt < R.a) Elem<T>::put(out, jt, dt);
#pragma unroll
            for (int c = 0; c < CH; c++) {
                const int j = j0 + c * NT * V;
                float d[V];
#pragma unroll
                for (int k = 0; k < V; k++) d[k] = column_fast<HAS_Q>(g, chunk_get<T>(z[c], k), HAS_Q ? chunk_get<T>(q[c], k) : 0.f, kl);
                asm volatile("" : "+v"(kl));  // (or the terms of KL are put off to the last chunk, with all their inputs kept)
                if ((unsigned)(a32 - j) < (unsigned)V) {
#pragma unroll
                    for (int k = 0; k < V; k++) d[k] += a32 - j == k ? g.c : 0.f;
                }
                if (O.grad && j < full) store_full<T>(out + j, d);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (HAS_Q) {
            float a = 0.f, b = 0.f;
            block_sum3<NT>(kl, a, b, sh[2]);
        } else {
            kl = kl_taken(P, row, o.logp);
        }
    } else if (O.grad) {
        const float zero[V] = {};
        for (int j = j0; j < full; j += NT * V) store_full<T>(out + j, zero);
        if (jt < R.a) Elem<T>::put(out, jt, 0.f);
    }
    if (threadIdx.x == 0 && O.parts) {
        const float w = P.weights ? P.weights[row] : P.default_weight;
        O.logp[row] = o.logp;
        O.kl[row] = live ? kl : 0.f;
        O.entropy[row] = h;
        O.parts[row] = (double)o.loss + kl_part(P, live, w, kl);
    }
}

__global__ __launch_bounds__(1024) void k_sum_parts(const double* __restrict__ parts, int64_t n, float* __restrict__ loss) {
    __shared__ double sh[1024];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += parts[i];
    sh[threadIdx.x] = s;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = (float)sh[0];
}

}  // namespace

#define BY_TYPE(dtype, ...)                                        \
    switch (dtype) {                                               \
        case 0: { using T = float; __VA_ARGS__; break; }           \
        case 1: { using T = __hip_bfloat16; __VA_ARGS__; break; }  \
        default: { using T = __half; __VA_ARGS__; break; }         \
    }

namespace {
// Narrow rows stay with one wave (140 columns take 3 registers of values per lane): log-probabilities of 8,192 x 1,000 float32 8 us, and
// 26 us with a workgroup per row; the loss of 32,768 x 512 56 and 85 us, of 8,192 x 1,000 33 and 30 us.
constexpr int WAVE_WIDEST = 1024, WAVE_WIDEST_LOSS = 512;
#define BY_WIDTH(a, ...)                                       \
    if ((a) <= 64) { constexpr int E = 1; __VA_ARGS__; }       \
    else if ((a) <= 192) { constexpr int E = 3; __VA_ARGS__; } \
    else { constexpr int E = 8; __VA_ARGS__; }

// launch(rows from R.row0 on, workgroups) for all rows, `per` of them to a workgroup.  A launch takes fewer than 2^32 work-items a
// dimension, so 2^21 workgroups of up to 1,024; more rows (17 million of two columns are 134 MB) go to further launches.
template <typename F>
void by_rows(PolicyRows R, int per, F launch) {
    const int64_t most = (int64_t)(1 << 21) * per;
    for (R.row0 = 0; R.row0 < R.n; R.row0 += most) launch(R, (unsigned)(((R.n - R.row0 < most ? R.n - R.row0 : most) + per - 1) / per));
}
template <typename T, int NT, int CH>
void row_loss(const PolicyRows& R, const PolicyTerms& P, const PolicyOut& O, unsigned wgs, hipStream_t s) {
    const dim3 grid(wgs), block(NT);
    if (P.ref_logits && R.legal_kind) hipLaunchKernelGGL((k_row_loss<T, NT, CH, true, true>), grid, block, 0, s, R, P, O);
    else if (P.ref_logits) hipLaunchKernelGGL((k_row_loss<T, NT, CH, true, false>), grid, block, 0, s, R, P, O);
    else if (R.legal_kind) hipLaunchKernelGGL((k_row_loss<T, NT, CH, false, true>), grid, block, 0, s, R, P, O);
    else hipLaunchKernelGGL((k_row_loss<T, NT, CH, false, false>), grid, block, 0, s, R, P, O);
}
// Rows read from memory twice: with one row per CU or fewer, sixteen waves draw more from memory than four (100 x 100,000 bfloat16 with a
// frozen policy: 51 us, and 82 us with four); with more rows, four on each of several rows (600 x 100,000: 145 us, and 161 us).
bool few(int64_t n) { return n <= 256; }
// The smallest workgroup whose registers hold the row: 8,192 x 32,768 bfloat16 with a frozen policy 410 us, 452 us read twice; without
// one 206 and 250 us; 2,048 x 4,000 23 and 32 us.  Past 512 threads of 8 chunks the row is read twice: a workgroup of 1,024 would have
// a CU to itself, and nothing to cover its loads with (2,048 x 50,001: 315 us, 226 us read twice) -- but for one input with a mask, whose
// second reading costs more (2,047 x 50,001 with a byte mask: 180 us, 191 us read twice).  A mask and a frozen policy together at 2,049 to
// 4,096 chunks need 80 bytes a lane of scratch: 8,192 x 32,768 bfloat16 669 us.
template <typename T>
void wide_loss(const PolicyRows& R, const PolicyTerms& P, const PolicyOut& O, unsigned wgs, hipStream_t s) {
    const int chunks = (R.a + Elem<T>::V - 1) / Elem<T>::V;
    if (chunks <= 256) row_loss<T, 256, 1>(R, P, O, wgs, s);
    else if (chunks <= 512) row_loss<T, 256, 2>(R, P, O, wgs, s);
    else if (chunks <= 1024) row_loss<T, 256, 4>(R, P, O, wgs, s);
    else if (chunks <= 2048) row_loss<T, 512, 4>(R, P, O, wgs, s);
    else if (chunks <= 4096) row_loss<T, 512, 8>(R, P, O, wgs, s);
    else if (chunks <= 8192 && R.legal_kind && !P.ref_logits) hipLaunchKernelGGL((k_row_loss<T, 1024, 8, false, true>), dim3(wgs), dim3(1024), 0, s, R, P, O);
    else if (few(R.n)) hipLaunchKernelGGL((k_policy_loss<T, 1024>), dim3(wgs), dim3(1024), 0, s, R, P, O);
    else hipLaunchKernelGGL((k_policy_loss<T, 256>), dim3(wgs), dim3(256), 0, s, R, P, O);
}
}  // namespace

namespace {
// Rows are split where a workgroup each would leave most CUs idle and a row is long enough to be worth three launches: 1 x 131,072
// bfloat16 with a frozen policy 20 us, and 60 us in one workgroup; 32 x 32,768 18 and 19 us; 64 x 32,768 21 and 19 us.
constexpr int FEW_ROWS = 64, SPLIT_WIDTH = 32768;
bool few_wide(int64_t n, int a) { return n <= FEW_ROWS && a >= SPLIT_WIDTH && a >= 1024 * n; }
Split make_split(int64_t n, int a, int v, void* ws) {
    Split S;
    const int unit = ST * v;  // columns that one pass of a workgroup covers
    int pieces = (int)(256 / n);
    if (pieces > MAX_SPLIT) pieces = MAX_SPLIT;
    if (pieces < 1) pieces = 1;
    S.piece = (a + pieces - 1) / pieces;
    S.piece = (S.piece + unit - 1) / unit * unit;
    S.s = (a + S.piece - 1) / S.piece;
    S.stats = reinterpret_cast<float*>(static_cast<char*>(ws) + n * 8);
    S.kl = S.stats + n * 2 * MAX_SPLIT * 3;
    S.coef = S.kl + n * MAX_SPLIT;
    return S;
}
}  // namespace

namespace qzl {
int64_t policy_workspace_bytes(int64_t n, int a) { return n * 8 + (few_wide(n, a) ? n * 4 * (7 * MAX_SPLIT + 1) : 0); }

hipError_t action_logp(const PolicyRows& R, float* logp, float* entropy, float* stats, void* ws, hipStream_t s) {
    if (R.n <= 0) return hipSuccess;
    if (R.a > 512 && R.a <= WAVE_WIDEST) {
        BY_TYPE(R.dtype, by_rows(R, 4, [&](const PolicyRows& Q, unsigned wgs) { hipLaunchKernelGGL((k_wave_logp<T, 16>), dim3(wgs), dim3(256), 0, s, Q, logp, entropy, stats); }));
    } else if (R.a <= 512) {
        BY_TYPE(R.dtype, BY_WIDTH(R.a, by_rows(R, 4, [&](const PolicyRows& Q, unsigned wgs) {
                    hipLaunchKernelGGL((k_wave_logp<T, E>), dim3(wgs), dim3(256), 0, s, Q, logp, entropy, stats); })));
    } else if (few_wide(R.n, R.a)) {
        const PolicyTerms none = {};
        BY_TYPE(R.dtype, const Split S = make_split(R.n, R.a, Elem<T>::V, ws);
                hipLaunchKernelGGL((k_split_stats<T>), dim3(S.s, (unsigned)R.n), dim3(ST), 0, s, R, none, S, nullptr, 0);
                hipLaunchKernelGGL((k_split_logp<T>), dim3((unsigned)R.n), dim3(64), 0, s, R, S, logp, entropy, stats));
    } else if (few(R.n) && R.a >= 65536) {  // (shorter rows: four waves, 1,024 x 8,192 8 us, and 22 us with sixteen)
        BY_TYPE(R.dtype, hipLaunchKernelGGL((k_action_logp<T, 1024>), dim3((unsigned)R.n), dim3(1024), 0, s, R, logp, entropy, stats));
    } else {
        BY_TYPE(R.dtype, by_rows(R, 1, [&](const PolicyRows& Q, unsigned wgs) { hipLaunchKernelGGL((k_action_logp<T, 256>), dim3(wgs), dim3(256), 0, s, Q, logp, entropy, stats); }));
    }
    return hipGetLastError();
}
hipError_t action_logp_backward(const PolicyRows& R, const float* stats, const float* entropy, const float* dlogp, const float* dentropy, void* grad,
                                int64_t ld_grad, hipStream_t s) {
    if (R.n <= 0) return hipSuccess;
    // few rows: several workgroups for each, up to one per pass over BT chunks
    BY_TYPE(R.dtype, const int most = (R.a + BT * Elem<T>::V - 1) / (BT * Elem<T>::V); int y = (int)((1024 + R.n - 1) / R.n); y = y < most ? y : most;
            by_rows(R, 1, [&](const PolicyRows& Q, unsigned wgs) {
                hipLaunchKernelGGL((k_action_logp_backward<T>), dim3(wgs, y), dim3(BT), 0, s, Q, stats, entropy, dlogp, dentropy, grad, ld_grad); }));
    return hipGetLastError();
}
hipError_t policy_loss(const PolicyRows& R, const PolicyTerms& P, PolicyOut O, float* loss, void* ws, hipStream_t s) {
    O.parts = loss ? static_cast<double*>(ws) : nullptr;
    if (R.n > 0) {
        if (R.a <= WAVE_WIDEST_LOSS) {
            BY_TYPE(R.dtype, BY_WIDTH(R.a, by_rows(R, 4, [&](const PolicyRows& Q, unsigned wgs) { hipLaunchKernelGGL((k_wave_loss<T, E>), dim3(wgs), dim3(256), 0, s, Q, P, O); })));
        } else if (few_wide(R.n, R.a)) {
            BY_TYPE(R.dtype, const Split S = make_split(R.n, R.a, Elem<T>::V, ws); const dim3 grid(S.s, (unsigned)R.n);
                    hipLaunchKernelGGL((k_split_stats<T>), grid, dim3(ST), 0, s, R, P, S, O.scale, O.only_if_scaled);
                    hipLaunchKernelGGL((k_split_loss<T>), grid, dim3(ST), 0, s, R, P, O, S);
                    if (loss) hipLaunchKernelGGL(k_split_finish, dim3(1), dim3(256), 0, s, O, S, (int)R.n, P.ref_logits != nullptr, loss));
            return hipGetLastError();
        } else {
            BY_TYPE(R.dtype, by_rows(R, 1, [&](const PolicyRows& Q, unsigned wgs) { wide_loss<T>(Q, P, O, wgs, s); }));
        }
    }
    if (loss) hipLaunchKernelGGL(k_sum_parts, dim3(1), dim3(1024), 0, s, O.parts, R.n, loss);
    return hipGetLastError();
}
}  // namespace qzl
