// extern "C" share-level entry points of the token-model operators
// (include/ddg_fss.h): argument checks and dispatch on the ring, one party's
// local computation, no communication.
#include <cmath>

#include "token.cuh"

using namespace ddg;

namespace ddg {

int check_q4(const ddg_q4_weights *w)
{
    DDG_CHECK(w, DDG_ERR_ARG, "null 4-bit weights");
    DDG_CHECK(w->K >= 0 && w->N >= 0, DDG_ERR_ARG, "negative size");
    DDG_CHECK(w->group > 0 && w->group % 32 == 0, DDG_ERR_ARG, "group must be a multiple of 32 (got %d)", w->group);
    DDG_CHECK(w->K == 0 || w->N == 0 || (w->d_q && w->d_step), DDG_ERR_ARG, "null pointer");
    DDG_CHECK((reinterpret_cast<uintptr_t>(w->d_q) & 15) == 0, DDG_ERR_ARG, "4-bit codes must be 16-byte aligned");
    DDG_CHECK((reinterpret_cast<uintptr_t>(w->d_step) & 1) == 0, DDG_ERR_ARG, "4-bit steps must be 2-byte aligned");
    return DDG_OK;
}

// the same answer on the dealer and both parties, although party 1 multiplies nothing
int check_q4_call(const ddg_q4_weights *w, int bw, int M)
{
    DDG_TRY(check_q4(w));
    DDG_CHECK(M >= 0, DDG_ERR_ARG, "negative size");
    DDG_CHECK(w->K <= Q4_MAX_K, DDG_ERR_ARG, "K = %d is too long (at most %d)", w->K, Q4_MAX_K);
    DDG_CHECK(M <= q4_max_rows(bw), DDG_ERR_ARG, "%d rows are too many for one call (at most %d)", M, q4_max_rows(bw));
    return DDG_OK;
}

int check_linattn(const ddg_linattn_shape *p, LaShape *s)
{
    DDG_CHECK(p, DDG_ERR_ARG, "null linear attention shape");
    DDG_CHECK(p->batch >= 0 && p->tokens >= 0 && p->heads >= 1, DDG_ERR_ARG, "bad batch, heads or tokens");
    DDG_CHECK(p->dk >= 1 && p->dk <= 128 && p->dv >= 1 && p->dv <= 128 && p->chunk >= 1 && p->chunk <= 128,
              DDG_ERR_ARG, "dk, dv and chunk must be 1..128 (got %d, %d, %d)", p->dk, p->dv, p->chunk);
    DDG_CHECK(p->pow_n >= 1 && p->pow_n >= p->tokens, DDG_ERR_ARG, "%d powers of the decay for %d tokens", p->pow_n,
              p->tokens);
    s->B = p->batch, s->H = p->heads, s->T = p->tokens, s->dk = p->dk, s->dv = p->dv, s->C = p->chunk;
    s->pn = p->pow_n;
    const double tokens = double(p->tokens < 128 ? 128 : p->tokens);
    // the carry's sums grow with the square of the chunks; a longer prompt goes on from the state
    DDG_CHECK((int64_t(p->tokens) + p->chunk - 1) / p->chunk <= LA_MAX_CHUNKS, DDG_ERR_ARG,
              "%d tokens are more than %d chunks of %d", p->tokens, LA_MAX_CHUNKS, p->chunk);
    DDG_CHECK(double(p->batch) * p->heads * tokens * 512.0 * 128.0 < 9e18 && double(p->heads) * 384.0 < 2e9,
              DDG_ERR_ARG, "linear attention sizes overflow");
    return DDG_OK;
}

}  // namespace ddg

namespace {

int check_ring(int bw, int party)
{
    DDG_CHECK(bw == 32 || bw == 64, DDG_ERR_ARG, "bw must be 32 or 64 (got %d)", bw);
    DDG_CHECK(party == 0 || party == 1, DDG_ERR_ARG, "party must be 0 or 1");
    return DDG_OK;
}

int check_la(int bw, int party, const ddg_linattn_shape *p, int64_t ld, LaShape *s)
{
    DDG_TRY(check_ring(bw, party));
    DDG_TRY(check_linattn(p, s));
    DDG_CHECK(ld >= s->width(), DDG_ERR_ARG, "row stride %lld below the row's %lld elements", (long long)ld,
              (long long)s->width());
    return DDG_OK;
}

// ring arrays: there, and on element boundaries
int check_ptrs(int bw, std::initializer_list<const void *> ptrs)
{
    for (const void *p : ptrs) {
        DDG_CHECK(p, DDG_ERR_ARG, "null pointer");
        DDG_CHECK(reinterpret_cast<uintptr_t>(p) % uintptr_t(bw / 8) == 0, DDG_ERR_ARG, "misaligned ring array");
    }
    return DDG_OK;
}

template <typename T>
const T *in(const void *p)
{
    return static_cast<const T *>(p);
}

template <typename T>
int fc_q4_t(int M, const ddg_q4_weights *w, const void *x, int64_t ldx, const void *c, void *out, cudaStream_t st)
{
    Q4Args<T> a;
    a.w.K = w->K, a.w.N = w->N, a.w.group = w->group;
    a.w.q = in<uint8_t>(w->d_q), a.w.step = in<uint16_t>(w->d_step);
    a.M = M, a.x = in<T>(x), a.ldx = ldx, a.bias = in<T>(w->d_bias2s), a.Add = in<T>(c);
    a.out = static_cast<T *>(out);
    return fc_q4<T>(a, st);
}

template <typename T>
int chunk_t(int party, const LaShape &s, int64_t ld, const void *qkv, const void *qkv_ms, const void *kd,
            const void *kd_ms, const void *z, void *out, cudaStream_t st)
{
    LaChunkArgs<T> a;
    a.ld = ld, a.qkv = in<T>(qkv), a.qkv_ms = in<T>(qkv_ms), a.kd = in<T>(kd), a.kd_ms = in<T>(kd_ms);
    a.z = in<T>(z), a.out = static_cast<T *>(out), a.p0 = party == 0 ? T(1) : T(0);
    return la_chunk<T>(s, a, st);
}

template <typename T>
int output_t(int party, const LaShape &s, int64_t ld, const void *qkv, const void *qkv_ms, const void *qd,
             const void *qd_ms, const void *ps, const void *ps_ms, const void *s0, const void *s0_ms, const void *z,
             void *out, cudaStream_t st)
{
    LaOutArgs<T> a;
    a.ld = ld, a.qkv = in<T>(qkv), a.qkv_ms = in<T>(qkv_ms), a.qd = in<T>(qd), a.qd_ms = in<T>(qd_ms);
    a.ps = in<T>(ps), a.ps_ms = in<T>(ps_ms), a.s0 = in<T>(s0), a.s0_ms = in<T>(s0_ms);
    a.z = in<T>(z), a.out = static_cast<T *>(out), a.p0 = party == 0 ? T(1) : T(0);
    return la_output<T>(s, a, st);
}

template <typename T>
int step_t(int party, const LaShape &s, int64_t ld, const void *pow, const void *qkv, const void *qkv_ms,
           const void *S, const void *S_ms, const void *z, void *out, cudaStream_t st)
{
    LaStepArgs<T> a;
    a.ld = ld, a.pow = in<T>(pow), a.qkv = in<T>(qkv), a.qkv_ms = in<T>(qkv_ms), a.s = in<T>(S), a.s_ms = in<T>(S_ms);
    a.z = in<T>(z), a.out = static_cast<T *>(out), a.p0 = a.lam = party == 0 ? T(1) : T(0);
    return la_step<T>(s, a, st);
}

template <typename T>
int step_output_t(int party, const LaShape &s, int64_t ld, const void *pow, const void *qkv, const void *qkv_ms,
                  const void *yw, const void *yw_ms, const void *z, void *out, cudaStream_t st)
{
    LaStepOutArgs<T> a;
    a.ld = ld, a.pow = in<T>(pow), a.qkv = in<T>(qkv), a.qkv_ms = in<T>(qkv_ms);
    a.yw = in<T>(yw), a.yw_ms = in<T>(yw_ms);
    a.z = in<T>(z), a.out = static_cast<T *>(out), a.p0 = a.lam = party == 0 ? T(1) : T(0);
    return la_step_output<T>(s, a, st);
}

}  // namespace

extern "C" {

uint64_t ddg_q4_row_bytes(int K) { return K < 1 ? 0 : q4_row_bytes(K); }

int ddg_q4_quantize(int K, int N, int group, const int64_t *d_w, void *d_q, void *d_step, void *stream)
{
    ddg_q4_weights w = {K, N, group, d_q, d_step, nullptr};
    DDG_TRY(check_q4(&w));
    if (K && N) DDG_TRY(check_ptrs(64, {d_w}));
    return q4_quantize(K, N, group, d_w, static_cast<uint8_t *>(d_q), static_cast<uint16_t *>(d_step),
                       static_cast<cudaStream_t>(stream));
}

int ddg_fc_q4_share(int bw, int party, int M, const ddg_q4_weights *w, const void *d_xhat, int64_t ldx,
                    const void *d_c, void *d_out, void *stream)
{
    DDG_TRY(check_ring(bw, party));
    DDG_TRY(check_q4_call(w, bw, M));
    DDG_CHECK(ldx >= w->K, DDG_ERR_ARG, "row stride %lld below K = %d", (long long)ldx, w->K);
    const uint64_t n = uint64_t(M) * w->N;
    if (!n) return DDG_OK;
    DDG_TRY(check_ptrs(bw, {d_c, d_out}));
    auto st = static_cast<cudaStream_t>(stream);
    if (party == 1) {
        if (d_out != d_c)
            DDG_CUDA(cudaMemcpyAsync(d_out, d_c, n * uint64_t(bw / 8), cudaMemcpyDeviceToDevice, st));
        return DDG_OK;
    }
    if (w->K) DDG_TRY(check_ptrs(bw, {d_xhat}));
    if (w->d_bias2s) DDG_TRY(check_ptrs(bw, {w->d_bias2s}));
    return bw == 32 ? fc_q4_t<uint32_t>(M, w, d_xhat, ldx, d_c, d_out, st)
                    : fc_q4_t<uint64_t>(M, w, d_xhat, ldx, d_c, d_out, st);
}

int ddg_decay_table(int bw, int scale, int heads, int n, const double *h_lambda, void *h_pow)
{
    DDG_TRY(check_ring(bw, 0));
    DDG_CHECK(scale >= 0 && scale < bw - 1, DDG_ERR_ARG, "scale %d out of range for bw %d", scale, bw);
    DDG_CHECK(heads >= 0 && n >= 0, DDG_ERR_ARG, "negative size");
    DDG_CHECK(heads == 0 || (h_lambda && h_pow), DDG_ERR_ARG, "null pointer");
    for (int h = 0; h < heads; h++)
        DDG_CHECK(h_lambda[h] >= 0.0 && h_lambda[h] <= 1.0, DDG_ERR_ARG, "decay %d is not in [0, 1]", h);
    for (int h = 0; h < heads; h++) {
        double p = std::ldexp(1.0, scale);
        for (int64_t i = 0; i <= n; i++, p *= h_lambda[h]) {  // n may be the largest int
            const uint64_t v = uint64_t(std::llround(p));
            const int64_t at = int64_t(h) * (int64_t(n) + 1) + i;
            if (bw == 32)
                static_cast<uint32_t *>(h_pow)[at] = uint32_t(v);
            else
                static_cast<uint64_t *>(h_pow)[at] = v;
        }
    }
    return DDG_OK;
}

int ddg_linattn_sizes(const ddg_linattn_shape *shape, int64_t *out6)
{
    LaShape s;
    DDG_TRY(check_linattn(shape, &s));
    DDG_CHECK(out6, DDG_ERR_ARG, "null pointer");
    out6[0] = s.n_qkv(), out6[1] = 2 * s.n_decayed(), out6[2] = s.n_ps(), out6[3] = s.n_state();
    out6[4] = s.n_step(), out6[5] = s.n_out();
    return DDG_OK;
}

int ddg_linattn_decay(int bw, const ddg_linattn_shape *shape, int64_t ld, const void *d_pow, const void *d_qkv,
                      void *d_out, void *stream)
{
    LaShape s;
    DDG_TRY(check_la(bw, 0, shape, ld, &s));
    if (!s.n_qkv()) return DDG_OK;
    DDG_TRY(check_ptrs(bw, {d_pow, d_qkv, d_out}));
    auto st = static_cast<cudaStream_t>(stream);
    return bw == 32 ? la_decay<uint32_t>(s, ld, in<uint32_t>(d_pow), in<uint32_t>(d_qkv),
                                         static_cast<uint32_t *>(d_out), st)
                    : la_decay<uint64_t>(s, ld, in<uint64_t>(d_pow), in<uint64_t>(d_qkv),
                                         static_cast<uint64_t *>(d_out), st);
}

int ddg_linattn_carry(int bw, const ddg_linattn_shape *shape, const void *d_pow, const void *d_ps, const void *d_s0,
                      void *d_out, void *stream)
{
    LaShape s;
    DDG_TRY(check_ring(bw, 0));
    DDG_TRY(check_linattn(shape, &s));
    if (!s.n_ps()) return DDG_OK;
    DDG_TRY(check_ptrs(bw, {d_pow, d_ps, d_out, d_s0 ? d_s0 : d_ps}));
    auto st = static_cast<cudaStream_t>(stream);
    return bw == 32 ? la_carry<uint32_t>(s, in<uint32_t>(d_pow), in<uint32_t>(d_ps), in<uint32_t>(d_s0),
                                         static_cast<uint32_t *>(d_out), st)
                    : la_carry<uint64_t>(s, in<uint64_t>(d_pow), in<uint64_t>(d_ps), in<uint64_t>(d_s0),
                                         static_cast<uint64_t *>(d_out), st);
}

int ddg_linattn_chunk_share(int bw, int party, const ddg_linattn_shape *shape, int64_t ld, const void *d_qkv_hat,
                            const void *d_qkv_ms, const void *d_kd_hat, const void *d_kd_ms, const void *d_z,
                            void *d_out, void *stream)
{
    LaShape s;
    DDG_TRY(check_la(bw, party, shape, ld, &s));
    if (!s.n_ps()) return DDG_OK;
    DDG_TRY(check_ptrs(bw, {d_qkv_hat, d_qkv_ms, d_kd_hat, d_kd_ms, d_z, d_out}));
    auto st = static_cast<cudaStream_t>(stream);
    return bw == 32 ? chunk_t<uint32_t>(party, s, ld, d_qkv_hat, d_qkv_ms, d_kd_hat, d_kd_ms, d_z, d_out, st)
                    : chunk_t<uint64_t>(party, s, ld, d_qkv_hat, d_qkv_ms, d_kd_hat, d_kd_ms, d_z, d_out, st);
}

int ddg_linattn_output_share(int bw, int party, const ddg_linattn_shape *shape, int64_t ld, const void *d_qkv_hat,
                             const void *d_qkv_ms, const void *d_qd_hat, const void *d_qd_ms, const void *d_ps_hat,
                             const void *d_ps_ms, const void *d_s0_hat, const void *d_s0_ms, const void *d_z,
                             void *d_out, void *stream)
{
    LaShape s;
    DDG_TRY(check_la(bw, party, shape, ld, &s));
    DDG_CHECK(!d_s0_hat == !d_s0_ms, DDG_ERR_ARG, "the first state needs its value and its mask share");
    if (!s.n_out()) return DDG_OK;
    DDG_TRY(check_ptrs(bw, {d_qkv_hat, d_qkv_ms, d_qd_hat, d_qd_ms, d_ps_hat, d_ps_ms, d_z, d_out,
                            d_s0_hat ? d_s0_hat : d_z, d_s0_ms ? d_s0_ms : d_z}));
    auto st = static_cast<cudaStream_t>(stream);
    return bw == 32 ? output_t<uint32_t>(party, s, ld, d_qkv_hat, d_qkv_ms, d_qd_hat, d_qd_ms, d_ps_hat, d_ps_ms,
                                         d_s0_hat, d_s0_ms, d_z, d_out, st)
                    : output_t<uint64_t>(party, s, ld, d_qkv_hat, d_qkv_ms, d_qd_hat, d_qd_ms, d_ps_hat, d_ps_ms,
                                         d_s0_hat, d_s0_ms, d_z, d_out, st);
}

int ddg_linattn_step_share(int bw, int party, const ddg_linattn_shape *shape, int64_t ld, const void *d_pow,
                           const void *d_qkv_hat, const void *d_qkv_ms, const void *d_s_hat, const void *d_s_ms,
                           const void *d_z, void *d_out, void *stream)
{
    LaShape s;
    DDG_TRY(check_la(bw, party, shape, ld, &s));
    DDG_CHECK(s.T == 1, DDG_ERR_ARG, "a step takes one token per sequence (got %d)", s.T);
    if (!s.bh()) return DDG_OK;
    DDG_TRY(check_ptrs(bw, {d_pow, d_qkv_hat, d_qkv_ms, d_s_hat, d_s_ms, d_z, d_out}));
    auto st = static_cast<cudaStream_t>(stream);
    return bw == 32 ? step_t<uint32_t>(party, s, ld, d_pow, d_qkv_hat, d_qkv_ms, d_s_hat, d_s_ms, d_z, d_out, st)
                    : step_t<uint64_t>(party, s, ld, d_pow, d_qkv_hat, d_qkv_ms, d_s_hat, d_s_ms, d_z, d_out, st);
}

int ddg_linattn_step_output_share(int bw, int party, const ddg_linattn_shape *shape, int64_t ld, const void *d_pow,
                                  const void *d_qkv_hat, const void *d_qkv_ms, const void *d_yw_hat,
                                  const void *d_yw_ms, const void *d_z, void *d_out, void *stream)
{
    LaShape s;
    DDG_TRY(check_la(bw, party, shape, ld, &s));
    DDG_CHECK(s.T == 1, DDG_ERR_ARG, "a step takes one token per sequence (got %d)", s.T);
    if (!s.bh()) return DDG_OK;
    DDG_TRY(check_ptrs(bw, {d_pow, d_qkv_hat, d_qkv_ms, d_yw_hat, d_yw_ms, d_z, d_out}));
    auto st = static_cast<cudaStream_t>(stream);
    return bw == 32
               ? step_output_t<uint32_t>(party, s, ld, d_pow, d_qkv_hat, d_qkv_ms, d_yw_hat, d_yw_ms, d_z, d_out, st)
               : step_output_t<uint64_t>(party, s, ld, d_pow, d_qkv_hat, d_qkv_ms, d_yw_hat, d_yw_ms, d_z, d_out, st);
}

}  // extern "C"
