// Fully connected layers with 4-bit public weights and group steps:
//
//   out[m][n] = sign * sum_k x[m][k] W[k][n] + bias[n] + Add[m][n]   modulo 2^bw
//   W[k][n]   = step[k / group][n] * (code(n, k) - 8)
//
// The ring sum is exact in any order, so the result does not depend on how K is split.
#include "token.cuh"

namespace ddg {

namespace {

__device__ __forceinline__ int q4_code(const uint8_t *row, int k) { return (row[k >> 1] >> (4 * (k & 1))) & 15; }

// one output element per thread
template <typename T>
__global__ void __launch_bounds__(256) k_fc_q4(const __grid_constant__ Q4Args<T> a, int64_t row_bytes)
{
    const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (e >= int64_t(a.M) * a.w.N) return;
    const int64_t m = e / a.w.N, n = e % a.w.N;
    const uint8_t *row = a.w.q + n * row_bytes;
    const T *x = a.x + m * a.ldx;
    T sum = 0;
    for (int k0 = 0, g = 0; k0 < a.w.K; k0 += a.w.group, g++) {
        const int k1 = a.w.K - k0 < a.w.group ? a.w.K : k0 + a.w.group;
        T part = 0;
        for (int k = k0; k < k1; k++) part += x[k] * T(int64_t(q4_code(row, k) - 8));
        sum += part * T(a.w.step[int64_t(g) * a.w.N + n] & Q4_STEP_MAX);
    }
    T v = a.sign * sum;
    if (a.bias) v += a.bias[n];
    if (a.Add) v += a.Add[e];
    a.out[e] = v;
}

// one group of one output per thread: the smallest step whose codes -7..7
// reach the group's largest weight (at most 4095, beyond which codes saturate),
// codes rounded to nearest
__global__ void __launch_bounds__(256)
    k_q4_quantize(int K, int N, int group, const int64_t *w, uint8_t *q, uint16_t *step, int64_t row_bytes)
{
    const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int ng = (K + group - 1) / group;
    if (e >= int64_t(ng) * N) return;
    const int64_t n = e % N;
    const int k0 = int(e / N) * group, k1 = K - k0 < group ? K : k0 + group;
    auto mag = [](int64_t v) { return v < 0 ? uint64_t(0) - uint64_t(v) : uint64_t(v); };
    uint64_t top = 0;
    for (int k = k0; k < k1; k++) {
        const uint64_t a = mag(w[int64_t(k) * N + n]);
        top = a > top ? a : top;
    }
    const uint64_t fit = top / 7 + (top % 7 ? 1 : 0);
    const uint64_t s = fit < 1 ? 1 : fit > uint64_t(Q4_STEP_MAX) ? uint64_t(Q4_STEP_MAX) : fit;
    step[e] = uint16_t(s);
    const int kend = k1 == K ? int(2 * row_bytes) : k1;  // the row's padding holds zero weights
    for (int k = k0; k < kend; k += 2) {
        uint32_t byte = 0;
        for (int i = 0; i < 2; i++) {
            uint32_t code = 8;
            if (k + i < K) {
                const int64_t v = w[int64_t(k + i) * N + n];
                const uint64_t a = mag(v);
                const uint32_t r = a >= 8 * s ? 8 : uint32_t((2 * a + s) / (2 * s));
                code = v < 0 ? 8 - r : 8 + (r > 7 ? 7 : r);
            }
            byte |= code << (4 * i);
        }
        q[n * row_bytes + (k >> 1)] = uint8_t(byte);
    }
}

}  // namespace

template <typename T>
int fc_q4(const Q4Args<T> &a, cudaStream_t st)
{
    const int64_t n = int64_t(a.M) * a.w.N, blocks = (n + 255) / 256;
    if (!n) return DDG_OK;
    DDG_CHECK(blocks <= 0x7fffffff, DDG_ERR_ARG, "fc_q4: %d x %d outputs are too many for one call", a.M, a.w.N);
    k_fc_q4<T><<<int(blocks), 256, 0, st>>>(a, int64_t(q4_row_bytes(a.w.K)));
    note_launch();
    DDG_CUDA(cudaGetLastError());
    return DDG_OK;
}
template int fc_q4<uint32_t>(const Q4Args<uint32_t> &, cudaStream_t);
template int fc_q4<uint64_t>(const Q4Args<uint64_t> &, cudaStream_t);

int q4_quantize(int K, int N, int group, const int64_t *w, uint8_t *q, uint16_t *step, cudaStream_t st)
{
    const int64_t n = (int64_t(K) + group - 1) / group * N, blocks = (n + 255) / 256;
    if (!n) return DDG_OK;
    DDG_CHECK(blocks <= 0x7fffffff, DDG_ERR_ARG, "q4_quantize: %d x %d weights are too many for one call", K, N);
    k_q4_quantize<<<int(blocks), 256, 0, st>>>(K, N, group, w, q, step, int64_t(q4_row_bytes(K)));
    note_launch();
    DDG_CUDA(cudaGetLastError());
    return DDG_OK;
}

}  // namespace ddg
