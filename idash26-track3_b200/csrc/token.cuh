// Building blocks of a secure token model: fully connected layers with 4-bit
// public weights (fc_q4.cu) and linear attention with a decay per head
// (linattn.cu).  One party's local arithmetic over Z_2^bw; the openings and
// the truncation gates between them are the executors' (graph.cuh).
#pragma once
#include "common.cuh"
#include "q4_plan.cuh"

namespace ddg {

// ------------------------------------------------------------------ 4-bit weights
//
// W[k][n] = step[k / group][n] * (nibble(n, k) - 8): 12-bit steps and 4-bit
// codes, so every weight fits 16 bits signed.  Output n's codes are one row of
// q4_row_bytes(K) bytes, code k in the low (k even) or high half of byte k/2.
struct Q4 {
    int K = 0, N = 0, group = 32;
    const uint8_t *q = nullptr;
    const uint16_t *step = nullptr;
};
inline uint64_t q4_row_bytes(int K) { return 16ull * ((uint64_t(K) + 31) / 32); }
constexpr int Q4_STEP_MAX = 4095;
// what one call covers: Q4_MAX_K, and grid rows of 64 (32 over Z_2^64) rows of x
constexpr int q4_max_rows(int bw) { return 65535 * (2048 / bw); }

// out[m][n] = sign * (x . W)[m][n] + bias[n] + Add[m][n] (bias, Add may be null)
template <typename T>
struct Q4Args {
    Q4 w;
    int M = 0;
    const T *x = nullptr;
    int64_t ldx = 0;
    T sign = 1;
    const T *bias = nullptr, *Add = nullptr;
    T *out = nullptr;
};
template <typename T>
int fc_q4(const Q4Args<T> &a, cudaStream_t st);
// codes and steps of an int64 weight matrix w (K x N)
int q4_quantize(int K, int N, int group, const int64_t *w, uint8_t *q, uint16_t *step, cudaStream_t st);

// ------------------------------------------------------------------ linear attention
//
// Sizes and array layouts.  The q|k|v rows are token-major, (batch, tokens) of
// row stride ld, each row heads x dk | heads x dk | heads x dv.  Everything
// else is head-major, head index bh = batch * heads + head:
//   decayed operands  Qd (bh, T, dk), then Kd (bh, T, dk)
//   score/state array P  (bh, tri), then states (chunk, bh, dk, dv);
//                     tri: per chunk the rows i = 0, 1, .. of its causal
//                     triangle, i + 1 entries each
// pow[h][n], n = 0..pn: lambda_h^n at the fixed-point scale.
constexpr int LA_MAX_CHUNKS = 2048;  // chunks of one prompt call
struct LaShape {
    int B = 0, H = 0, T = 0, dk = 0, dv = 0, C = 128, pn = 0;
    __host__ __device__ int64_t bh() const { return int64_t(B) * H; }
    __host__ __device__ int chunks() const { return (T + C - 1) / C; }
    __host__ __device__ int len(int c) const { return T - c * C < C ? T - c * C : C; }
    __host__ __device__ int end(int c) const { return c * C + len(c); }
    __host__ __device__ int64_t tri_at(int c) const { return int64_t(c) * (int64_t(C) * (C + 1) / 2); }
    __host__ __device__ int64_t tri() const
    {
        const int64_t r = T % C;
        return tri_at(T / C) + r * (r + 1) / 2;
    }
    // (pn may be the largest int; one 32 x 32-bit multiply)
    __host__ __device__ int64_t pow_at(uint32_t h) const { return int64_t(uint64_t(h) * (uint32_t(pn) + 1u)); }
    __host__ __device__ int64_t width() const { return int64_t(H) * (2 * int64_t(dk) + dv); }
    __host__ __device__ int64_t n_qkv() const { return int64_t(B) * T * width(); }
    __host__ __device__ int64_t n_decayed() const { return bh() * T * dk; }  // of each of Qd, Kd
    __host__ __device__ int64_t n_scores() const { return bh() * tri(); }
    __host__ __device__ int64_t n_state() const { return bh() * dk * dv; }
    __host__ __device__ int64_t n_ps() const { return n_scores() + chunks() * n_state(); }
    __host__ __device__ int64_t n_out() const { return bh() * T * dv; }
    __host__ __device__ int64_t n_step() const { return n_state() + bh() * (dv + 1); }
};

// out = [pow[i+1] q | pow[len-1-i] k] of token i of its chunk (scale 2s)
template <typename T>
int la_decay(const LaShape &s, int64_t ld, const T *pow, const T *x, T *out, cudaStream_t st);

// out = [causal q . k^T per chunk | Kd^T . V per chunk] + z: party's share.
// *_ms are the party's mask shares; qkv_ms null stands for all of them zero,
// so that the dealer's word (the product of the masks plus the output mask, as
// z) is the same call on the masks with p0 = 1.
template <typename T>
struct LaChunkArgs {
    int64_t ld = 0;
    const T *qkv = nullptr, *qkv_ms = nullptr, *kd = nullptr, *kd_ms = nullptr, *z = nullptr;
    T *out = nullptr;
    T p0 = 1;
};
template <typename T>
int la_chunk(const LaShape &s, const LaChunkArgs<T> &a, cudaStream_t st);

// out = [pow[i-j] P | per chunk c: sum_{c' <= c} pow[end(c)-end(c')] dS[c'] + pow[end(c)] S0]
// (s0 may be null)
template <typename T>
int la_carry(const LaShape &s, const T *pow, const T *ps, const T *s0, T *out, cudaStream_t st);

// out (B, T, H, dv) = P . V + Qd . S[chunk - 1] + z: party's share (S[-1] = s0, or nothing when null)
template <typename T>
struct LaOutArgs {
    int64_t ld = 0;
    const T *qkv = nullptr, *qkv_ms = nullptr, *qd = nullptr, *qd_ms = nullptr, *ps = nullptr, *ps_ms = nullptr,
            *s0 = nullptr, *s0_ms = nullptr, *z = nullptr;
    T *out = nullptr;
    T p0 = 1;
};
template <typename T>
int la_output(const LaShape &s, const LaOutArgs<T> &a, cudaStream_t st);

// one token: out = [lambda S + k (x) v | q . S | q . k] + z: party's share
template <typename T>
struct LaStepArgs {
    int64_t ld = 0;
    const T *pow = nullptr, *qkv = nullptr, *qkv_ms = nullptr, *s = nullptr, *s_ms = nullptr, *z = nullptr;
    T *out = nullptr;
    T p0 = 1;   // 1 for party 0 and for the dealer, 0 for party 1
    T lam = 1;  // factor of the public term lambda * (masked value): p0 for a party, -1 for the dealer's word
};
template <typename T>
int la_step(const LaShape &s, const LaStepArgs<T> &a, cudaStream_t st);
// out (bh, dv) = lambda y + w v + z: party's share; yw = [y (bh, dv) | w (bh)]
template <typename T>
struct LaStepOutArgs {
    int64_t ld = 0;
    const T *pow = nullptr, *qkv = nullptr, *qkv_ms = nullptr, *yw = nullptr, *yw_ms = nullptr, *z = nullptr;
    T *out = nullptr;
    T p0 = 1;   // 1 for party 0 and for the dealer, 0 for party 1
    T lam = 1;  // factor of the public term lambda * (masked value): p0 for a party, -1 for the dealer's word
};
template <typename T>
int la_step_output(const LaShape &s, const LaStepOutArgs<T> &a, cudaStream_t st);

// argument checks of the C ABI's structs (capi_token.cu)
int check_q4(const ddg_q4_weights *w);
int check_q4_call(const ddg_q4_weights *w, int bw, int M);
int check_linattn(const ddg_linattn_shape *p, LaShape *s);

}  // namespace ddg
