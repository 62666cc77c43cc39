// Linear attention with a decay per head, one party's share, over Z_2^bw:
//
//   S_t = lambda_h S_{t-1} + k_t v_t^T,   o_t = q_t S_t
//
// for prompts in chunks of C tokens (la_decay, la_chunk, la_carry, la_output)
// and for one token (la_step, la_step_output); sizes and layouts in token.cuh.
// Products of two masked wires are Beaver products,
//   share of a.b = a^ . (p0 b^ - [r_b]) - [r_a] . b^ + Z ,
// products with the public decays are local on the masked values.
#include "token.cuh"

namespace ddg {

namespace {

constexpr int LA_THREADS = 256;

int la_grid(int64_t n)
{
    const int64_t b = (n + LA_THREADS - 1) / LA_THREADS;
    return int(b < 148 * 64 ? (b ? b : 1) : 148 * 64);
}

#define LA_EACH(e, n) \
    for (int64_t e = int64_t(blockIdx.x) * LA_THREADS + threadIdx.x; e < (n); e += int64_t(gridDim.x) * LA_THREADS)

// chunk and row of entry e of one head's score triangles
__device__ __forceinline__ void tri_find(const LaShape &s, int64_t e, int &c, int &i, int &j)
{
    const int64_t full = int64_t(s.C) * (s.C + 1) / 2;
    c = int(e / full);
    const int r = int(e - c * full);
    i = int((sqrtf(8.f * float(r) + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= r) i++;
    while (i * (i + 1) / 2 > r) i--;
    j = r - i * (i + 1) / 2;
}

template <typename T>
__device__ __forceinline__ const T *qkv_row(const LaShape &s, int64_t ld, const T *x, int64_t b, int64_t t)
{
    return x + (b * s.T + t) * ld;
}

template <typename T>
__global__ void __launch_bounds__(LA_THREADS)
    k_la_decay(const LaShape s, int64_t ld, const T *pow, const T *x, T *out)
{
    const int64_t nd = s.n_decayed();
    LA_EACH(e, 2 * nd)
    {
        const bool key = e >= nd;
        const int64_t r = key ? e - nd : e;
        const int d = int(r % s.dk);
        const int64_t bt = r / s.dk;
        const int t = int(bt % s.T);
        const int64_t bh = bt / s.T, b = bh / s.H;
        const int h = int(bh % s.H), c = t / s.C, i = t - c * s.C;
        const T *row = qkv_row(s, ld, x, b, t) + (key ? int64_t(s.H) * s.dk : 0) + int64_t(h) * s.dk;
        out[e] = pow[int64_t(h) * (s.pn + 1) + (key ? s.len(c) - 1 - i : i + 1)] * row[d];
    }
}

template <typename T>
__global__ void __launch_bounds__(LA_THREADS) k_la_chunk(const LaShape s, const __grid_constant__ LaChunkArgs<T> a)
{
    const int64_t ns = s.n_scores(), tri = s.tri(), kd_off = int64_t(s.H) * s.dk, vo = 2 * kd_off;
    LA_EACH(e, s.n_ps())
    {
        T acc = 0;
        if (e < ns) {
            const int64_t bh = e / tri, b = bh / s.H;
            const int h = int(bh % s.H);
            int c, i, j;
            tri_find(s, e - bh * tri, c, i, j);
            const int64_t oq = (b * s.T + c * s.C + i) * a.ld + int64_t(h) * s.dk;
            const int64_t ok = (b * s.T + c * s.C + j) * a.ld + kd_off + int64_t(h) * s.dk;
            for (int x = 0; x < s.dk; x++) {
                T right = a.p0 * a.qkv[ok + x];
                if (a.qkv_ms) right -= a.qkv_ms[ok + x], acc -= a.qkv_ms[oq + x] * a.qkv[ok + x];
                acc += a.qkv[oq + x] * right;
            }
        } else {
            int64_t r = e - ns;
            const int y = int(r % s.dv);
            r /= s.dv;
            const int x = int(r % s.dk);
            r /= s.dk;
            const int64_t bh = r % s.bh(), b = bh / s.H;
            const int h = int(bh % s.H), c = int(r / s.bh()), len = s.len(c);
            for (int i = 0; i < len; i++) {
                const int64_t t = int64_t(c) * s.C + i;
                const int64_t ok = (bh * s.T + t) * s.dk + x;
                const int64_t ov = (b * s.T + t) * a.ld + vo + int64_t(h) * s.dv + y;
                T right = a.p0 * a.qkv[ov];
                if (a.qkv_ms) right -= a.qkv_ms[ov], acc -= a.kd_ms[ok] * a.qkv[ov];
                acc += a.kd[ok] * right;
            }
        }
        a.out[e] = acc + a.z[e];
    }
}

template <typename T>
__global__ void __launch_bounds__(LA_THREADS)
    k_la_carry(const LaShape s, const T *pow, const T *ps, const T *s0, T *out)
{
    const int64_t ns = s.n_scores(), tri = s.tri(), state = s.n_state(), per = int64_t(s.dk) * s.dv;
    LA_EACH(e, s.n_ps())
    {
        if (e < ns) {
            const int64_t bh = e / tri;
            int c, i, j;
            tri_find(s, e - bh * tri, c, i, j);
            out[e] = pow[(bh % s.H) * (s.pn + 1) + i - j] * ps[e];
        } else {
            const int64_t r = (e - ns) % state;
            const int c = int((e - ns) / state), end = s.end(c);
            const T *pw = pow + (r / per % s.H) * (s.pn + 1);
            T acc = s0 ? pw[end] * s0[r] : T(0);
            for (int j = 0; j <= c; j++) acc += pw[end - s.end(j)] * ps[ns + j * state + r];
            out[e] = acc;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(LA_THREADS) k_la_output(const LaShape s, const __grid_constant__ LaOutArgs<T> a)
{
    const int64_t ns = s.n_scores(), tri = s.tri(), state = s.n_state(), per = int64_t(s.dk) * s.dv;
    LA_EACH(e, s.n_out())
    {
        const int y = int(e % s.dv);
        int64_t r = e / s.dv;
        const int h = int(r % s.H);
        r /= s.H;
        const int t = int(r % s.T), c = t / s.C, i = t - c * s.C;
        const int64_t b = r / s.T, bh = b * s.H + h;
        T acc = 0;
        const int64_t op = bh * tri + s.tri_at(c) + int64_t(i) * (i + 1) / 2;
        for (int j = 0; j <= i; j++) {
            const int64_t ov = (b * s.T + c * s.C + j) * a.ld + 2 * int64_t(s.H) * s.dk + int64_t(h) * s.dv + y;
            T right = a.p0 * a.qkv[ov];
            if (a.qkv_ms) right -= a.qkv_ms[ov], acc -= a.ps_ms[op + j] * a.qkv[ov];
            acc += a.ps[op + j] * right;
        }
        const T *S = c ? a.ps + ns + (c - 1) * state : a.s0, *Sm = c ? a.ps_ms + ns + (c - 1) * state : a.s0_ms;
        if (S) {
            for (int x = 0; x < s.dk; x++) {
                const int64_t oq = (bh * s.T + t) * s.dk + x, os = bh * per + int64_t(x) * s.dv + y;
                T right = a.p0 * S[os];
                if (a.qkv_ms) right -= Sm[os], acc -= a.qd_ms[oq] * S[os];
                acc += a.qd[oq] * right;
            }
        }
        a.out[e] = acc + a.z[e];
    }
}

template <typename T>
__global__ void __launch_bounds__(LA_THREADS) k_la_step(const LaShape s, const __grid_constant__ LaStepArgs<T> a)
{
    const int64_t state = s.n_state(), ny = s.bh() * s.dv, per = int64_t(s.dk) * s.dv;
    LA_EACH(e, s.n_step())
    {
        const bool u = e < state, w = e >= state + ny;
        const int64_t r = u ? e : w ? e - state - ny : e - state;
        const int64_t bh = u ? r / per : w ? r : r / s.dv, b = bh / s.H, h = bh % s.H;
        const int64_t oq = b * a.ld + h * s.dk, ok = oq + int64_t(s.H) * s.dk;
        T acc = 0;
        if (u) {
            const int64_t x = ok + (r - bh * per) / s.dv;
            const int64_t y = b * a.ld + 2 * int64_t(s.H) * s.dk + h * s.dv + r % s.dv;
            T right = a.p0 * a.qkv[y];
            if (a.qkv_ms) right -= a.qkv_ms[y], acc -= a.qkv_ms[x] * a.qkv[y];
            acc += a.qkv[x] * right + a.lam * a.pow[h * (s.pn + 1) + 1] * a.s[r];
        } else {
            for (int x = 0; x < s.dk; x++) {
                const int64_t os = bh * per + int64_t(x) * s.dv + r % s.dv;
                const T b1 = w ? a.qkv[ok + x] : a.s[os];
                T right = a.p0 * b1;
                if (a.qkv_ms) right -= w ? a.qkv_ms[ok + x] : a.s_ms[os], acc -= a.qkv_ms[oq + x] * b1;
                acc += a.qkv[oq + x] * right;
            }
        }
        a.out[e] = acc + a.z[e];
    }
}

template <typename T>
__global__ void __launch_bounds__(LA_THREADS)
    k_la_step_output(const LaShape s, const __grid_constant__ LaStepOutArgs<T> a)
{
    const int64_t ny = s.bh() * s.dv;
    LA_EACH(e, ny)
    {
        const int64_t bh = e / s.dv, b = bh / s.H, h = bh % s.H;
        const int64_t ov = b * a.ld + 2 * int64_t(s.H) * s.dk + h * s.dv + e % s.dv;
        T right = a.p0 * a.qkv[ov], acc = a.lam * a.pow[h * (s.pn + 1) + 1] * a.yw[e];
        if (a.qkv_ms) right -= a.qkv_ms[ov], acc -= a.yw_ms[ny + bh] * a.qkv[ov];
        a.out[e] = acc + a.yw[ny + bh] * right + a.z[e];
    }
}

int launched()
{
    note_launch();
    DDG_CUDA(cudaGetLastError());
    return DDG_OK;
}

}  // namespace

template <typename T>
int la_decay(const LaShape &s, int64_t ld, const T *pow, const T *x, T *out, cudaStream_t st)
{
    if (!s.n_decayed()) return DDG_OK;
    k_la_decay<T><<<la_grid(2 * s.n_decayed()), LA_THREADS, 0, st>>>(s, ld, pow, x, out);
    return launched();
}

template <typename T>
int la_chunk(const LaShape &s, const LaChunkArgs<T> &a, cudaStream_t st)
{
    if (!s.n_ps()) return DDG_OK;
    k_la_chunk<T><<<la_grid(s.n_ps()), LA_THREADS, 0, st>>>(s, a);
    return launched();
}

template <typename T>
int la_carry(const LaShape &s, const T *pow, const T *ps, const T *s0, T *out, cudaStream_t st)
{
    if (!s.n_ps()) return DDG_OK;
    k_la_carry<T><<<la_grid(s.n_ps()), LA_THREADS, 0, st>>>(s, pow, ps, s0, out);
    return launched();
}

template <typename T>
int la_output(const LaShape &s, const LaOutArgs<T> &a, cudaStream_t st)
{
    if (!s.n_out()) return DDG_OK;
    k_la_output<T><<<la_grid(s.n_out()), LA_THREADS, 0, st>>>(s, a);
    return launched();
}

template <typename T>
int la_step(const LaShape &s, const LaStepArgs<T> &a, cudaStream_t st)
{
    if (!s.bh()) return DDG_OK;
    k_la_step<T><<<la_grid(s.n_step()), LA_THREADS, 0, st>>>(s, a);
    return launched();
}

template <typename T>
int la_step_output(const LaShape &s, const LaStepOutArgs<T> &a, cudaStream_t st)
{
    if (!s.bh()) return DDG_OK;
    k_la_step_output<T><<<la_grid(s.bh() * s.dv), LA_THREADS, 0, st>>>(s, a);
    return launched();
}

#define LA_INSTANCES(T)                                                                                  \
    template int la_decay<T>(const LaShape &, int64_t, const T *, const T *, T *, cudaStream_t);         \
    template int la_chunk<T>(const LaShape &, const LaChunkArgs<T> &, cudaStream_t);                     \
    template int la_carry<T>(const LaShape &, const T *, const T *, const T *, T *, cudaStream_t);       \
    template int la_output<T>(const LaShape &, const LaOutArgs<T> &, cudaStream_t);                      \
    template int la_step<T>(const LaShape &, const LaStepArgs<T> &, cudaStream_t);                       \
    template int la_step_output<T>(const LaShape &, const LaStepOutArgs<T> &, cudaStream_t);
LA_INSTANCES(uint32_t)
LA_INSTANCES(uint64_t)

}  // namespace ddg
