// Linear attention with a decay per head, one party's share, over Z_2^bw:
//
//   S_t = lambda_h S_{t-1} + k_t v_t^T,   o_t = q_t S_t
//
// for prompts in chunks of C tokens (la_decay, la_chunk, la_carry, la_output)
// and for one token (la_step, la_step_output); sizes and layouts in token.cuh.
// Products of two masked wires are Beaver products,
//   share of a.b = a^ . (p0 b^ - [r_b]) - [r_a] . b^ + Z ,
// products with the public decays are local on the masked values.
//
// The three matrix stages (scores, chunk states, outputs) run on the tensor
// cores in la_tile: 128 rows x NT columns of sum_p A_p . B_p, ring operands
// split into bytes by the loading threads, limb sums
//   C = sum_s 2^(8s) sum_{i+j=s} A_i . B_j  (u8 x u8 -> s32, exact: K <= 512)
// in tensor memory.  The limbs of B are stacked along N, so one MMA per limb i
// of A covers every j with i + j < P, landing in the columns of s = i .. P-1.
#include "token.cuh"
#include "umma.cuh"

namespace ddg {

namespace {

constexpr int LA_THREADS = 256;

int la_grid(int64_t n)
{
    const int64_t b = (n + LA_THREADS - 1) / LA_THREADS;
    return int(b < 148 * 64 ? (b ? b : 1) : 148 * 64);
}

// blocks of LA_THREADS threads with V of n elements each
inline int64_t la_blocks(int64_t n, int V) { return (n + int64_t(LA_THREADS) * V - 1) / (int64_t(LA_THREADS) * V); }

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

// V elements moved together: 16 bytes, or single elements where rows do not allow it
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
    T e[V];
};
template <typename T>
constexpr int VEC = 16 / int(sizeof(T));

inline bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ------------------------------------------------------------------ public maps (memory-bound)

// One token per block step: its q and k are one contiguous run, written as dk-long runs per head.
template <typename T, int V>
__global__ void __launch_bounds__(LA_THREADS)
    k_la_decay(const LaShape s, int64_t ld, const T *pow, const T *x, T *out)
{
    const int dkv = s.dk / V, half = s.H * dkv;
    const int64_t tokens = int64_t(s.B) * s.T, nd = s.n_decayed();
    for (int64_t bt = blockIdx.x; bt < tokens; bt += gridDim.x) {
        const int64_t b = bt / s.T;
        const int t = int(bt - b * s.T), c = t / s.C, i = t - c * s.C, back = s.len(c) - 1 - i;
        const Pack<T, V> *row = reinterpret_cast<const Pack<T, V> *>(x + bt * ld);
        for (int e = threadIdx.x; e < 2 * half; e += LA_THREADS) {
            const bool key = e >= half;
            const int r = key ? e - half : e, h = r / dkv, d = r - h * dkv;
            const T p = __ldg(pow + int64_t(h) * (s.pn + 1) + (key ? back : i + 1));
            Pack<T, V> v = row[e];
#pragma unroll
            for (int j = 0; j < V; j++) v.e[j] *= p;
            reinterpret_cast<Pack<T, V> *>(out + (key ? nd : 0) + ((b * s.H + h) * s.T + t) * s.dk)[d] = v;
        }
    }
}

// Scores: V consecutive packed entries per thread, the triangle walked from the
// first one's position.  States: V columns of up to LC_OT output chunks per
// thread, every earlier chunk read once per LC_OT outputs; the sums cannot
// be chained from chunk to chunk, because each S_c is floored from exact terms.
constexpr int LC_OT = 16;

template <typename T, int V>
__global__ void __launch_bounds__(LA_THREADS)
    k_la_carry(const LaShape s, const T *pow, const T *ps, const T *s0, T *out, int score_blocks)
{
    const int64_t ns = s.n_scores(), tri = s.tri();
    if (int(blockIdx.x) < score_blocks) {
        for (int64_t e0 = (int64_t(blockIdx.x) * LA_THREADS + threadIdx.x) * V; e0 < ns;
             e0 += int64_t(score_blocks) * LA_THREADS * V) {
            int64_t bh = e0 / tri;
            int c, i, j;
            tri_find(s, e0 - bh * tri, c, i, j);
            const int n = ns - e0 < V ? int(ns - e0) : V;
            Pack<T, V> v;
            if (n == V)
                v = *reinterpret_cast<const Pack<T, V> *>(ps + e0);
            else
                for (int k = 0; k < n; k++) v.e[k] = ps[e0 + k];
            const T *pw = pow + bh % s.H * (s.pn + 1);
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (k >= n) break;
                v.e[k] *= __ldg(pw + i - j);
                if (++j > i) {  // next row, chunk or head
                    j = 0;
                    if (++i >= s.len(c)) {
                        i = 0;
                        if (++c >= s.chunks()) c = 0, bh++, pw = pow + bh % s.H * (s.pn + 1);
                    }
                }
            }
            if (n == V)
                *reinterpret_cast<Pack<T, V> *>(out + e0) = v;
            else
                for (int k = 0; k < n; k++) out[e0 + k] = v.e[k];
        }
        return;
    }
    const int64_t state = s.n_state(), per = int64_t(s.dk) * s.dv;
    const int nc = s.chunks();
    const int64_t r = (int64_t(blockIdx.x - score_blocks) * LA_THREADS + threadIdx.x) * V;
    if (r >= state) return;
    const T *const pw = pow + r / per % s.H * (s.pn + 1);
    const T *const in = ps + ns + r;
    Pack<T, V> first;
#pragma unroll
    for (int k = 0; k < V; k++) first.e[k] = 0;
    if (s0) first = *reinterpret_cast<const Pack<T, V> *>(s0 + r);
    for (int c0 = 0; c0 < nc; c0 += LC_OT) {
        T acc[LC_OT][V];
#pragma unroll
        for (int o = 0; o < LC_OT; o++) {
            const T p = c0 + o < nc ? __ldg(pw + s.end(c0 + o)) : T(0);
#pragma unroll
            for (int k = 0; k < V; k++) acc[o][k] = p * first.e[k];
        }
        const int jn = c0 + LC_OT < nc ? c0 + LC_OT : nc;
        for (int j = 0; j < jn; j++) {
            const Pack<T, V> v = *reinterpret_cast<const Pack<T, V> *>(in + j * state);
            const int at = s.end(j);
#pragma unroll
            for (int o = 0; o < LC_OT; o++) {
                if (c0 + o >= j && c0 + o < nc) {
                    const T p = __ldg(pw + s.end(c0 + o) - at);
#pragma unroll
                    for (int k = 0; k < V; k++) acc[o][k] += p * v.e[k];
                }
            }
        }
#pragma unroll
        for (int o = 0; o < LC_OT; o++) {
            if (c0 + o >= nc) break;
            Pack<T, V> v;
#pragma unroll
            for (int k = 0; k < V; k++) v.e[k] = acc[o][k];
            *reinterpret_cast<Pack<T, V> *>(out + ns + (c0 + o) * state + r) = v;
        }
    }
}

// ------------------------------------------------------------------ matrix stages

template <typename T>
struct LtShape {
    static constexpr int P = int(sizeof(T));
    static constexpr int NT = 256 / P;             // tile columns: P x NT = 256 accumulator columns, two CTAs an SM
    static constexpr int NSTAGE = 2;
    // 8-row groups of the operand planes 272 instead of 256 bytes apart: the
    // transposing loaders store rows 4 apart, which then fall on distinct banks
    static constexpr uint32_t SBO = 272;
    static constexpr uint32_t A_PLANE = TC_BM / 8 * SBO, B_PLANE = NT / 8 * SBO;
    static constexpr uint32_t STAGE = P * (A_PLANE + B_PLANE);
    static constexpr int BI = NT * 8 / LA_THREADS;  // 4-element items of B per thread
    static constexpr uint32_t SMEM = 64 + 1024 + NSTAGE * STAGE + 4096;
    static_assert(TC_BM * (NT + 1) * sizeof(T) <= NSTAGE * STAGE, "the output tile is staged in the operand stages");
};

// n <= 4 elements at p, zeros behind them
template <typename T>
__device__ __forceinline__ void load4(const T *p, int n, bool vec, T (&e)[4])
{
    if (vec && n >= 4) {
        const uint4 *v = reinterpret_cast<const uint4 *>(p);
#pragma unroll
        for (int i = 0; i < int(sizeof(T)) / 4; i++) *reinterpret_cast<uint4 *>(e + i * (16 / int(sizeof(T)))) = __ldg(v + i);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = i < n ? __ldg(p + i) : T(0);
    }
}

template <typename T>
__device__ __forceinline__ bool vec_ok(const T *p, int64_t ld)
{
    return ((reinterpret_cast<uintptr_t>(p) | uintptr_t(ld * int64_t(sizeof(T)))) & 15) == 0;
}

// One K-step's operands.  A: rows of K elements (a_t = 0), K rows of elements
// (1), or packed triangle rows (2, row i at a + i (i + 1) / 2, entries j <= i).
// B: N rows of K elements (b_t = 0) or K rows of N elements (1); its value is
// p0 * b - bm, or -b when neg.
template <typename T>
struct LtStep {
    const T *a, *b, *bm;
    int64_t lda, ldb;
    int k0, K, rows, cols;
    bool a_vec, b_vec, neg;
};

enum { LT_SCORES = 0, LT_STATES = 1, LT_OUTPUT = 2 };

// rows x cols of one output tile: step(s) gives K-step s of `steps`, at(row)
// the index of its first column in out and z (columns up to last(row))
template <typename T, int KIND, class Step, class At, class Last>
__device__ __forceinline__ void la_tile(int steps, T p0, Step step, int rows, At at, Last last, const T *z, T *out,
                                        uint32_t *err)
{
    using S = LtShape<T>;
    constexpr int P = S::P, NT = S::NT, BI = S::BI;
    constexpr bool B_T = KIND != LT_SCORES;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint64_t *const bars = reinterpret_cast<uint64_t *>(smem_raw);
    uint32_t &s_tmem = *reinterpret_cast<uint32_t *>(smem_raw + 32);
    uint8_t *const smem = smem_raw + 64 + ((1024u - ((smem_addr(smem_raw) + 64u) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                     "r"(256)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < S::NSTAGE; i++) mbar_init(bars + i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    // K-contiguous items: 8 rows x 4 quads of k per warp; transposed 4 x 4
    // blocks: 8 row quads x 4 quads of k per warp
    const int kq = 4 * (warp & 1) + (lane & 3), krow = 8 * (warp >> 1) + (lane >> 2);
    const int tkq = 4 * (warp & 1) + (lane >> 3), trow = 4 * (8 * (warp >> 1) + (lane & 7));
    T ra[4][4];
    T rb[B_T ? 4 : BI][4], rm[B_T ? 4 : BI][4];
    bool neg = false;
    const bool b_on = !B_T || trow < NT;

    auto load_stage = [&](int s) {
        const LtStep<T> o = step(s);
        neg = o.neg;
        if constexpr (KIND == LT_STATES) {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int k = o.k0 + 4 * tkq + t;
                load4<T>(o.a + int64_t(k) * o.lda + trow, k < o.K ? o.rows - trow : 0, o.a_vec, ra[t]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int row = krow + 32 * j, k = o.k0 + 4 * kq;
                if (KIND == LT_OUTPUT && o.lda < 0) {  // packed triangle
                    load4<T>(o.a + row * (row + 1) / 2 + k, row < o.rows ? row + 1 - k : 0, false, ra[j]);
                } else {
                    load4<T>(o.a + row * o.lda + k, row < o.rows ? o.K - k : 0, o.a_vec, ra[j]);
                }
            }
        }
        const bool with_m = !o.neg && o.bm;
        if constexpr (B_T) {
            if (b_on) {
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const int k = o.k0 + 4 * tkq + t, n = k < o.K ? o.cols - trow : 0;
                    const int64_t off = int64_t(k) * o.ldb + trow;
                    load4<T>(o.b + off, n, o.b_vec, rb[t]);
                    load4<T>(o.bm + off, with_m ? n : 0, o.b_vec, rm[t]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < BI; j++) {
                const int w = warp + 8 * j, n = 8 * (w >> 1) + (lane >> 2), k = o.k0 + 16 * (w & 1) + 4 * (lane & 3);
                const int cnt = n < o.cols ? o.K - k : 0;
                const int64_t off = int64_t(n) * o.ldb + k;
                load4<T>(o.b + off, cnt, o.b_vec, rb[j]);
                load4<T>(o.bm + off, with_m ? cnt : 0, o.b_vec, rm[j]);
            }
        }
    };
    auto store_stage = [&](int st) {
        uint8_t *const pa = smem + st * S::STAGE, *const pb = pa + P * S::A_PLANE;
        auto at_off = [](int row, int q) -> uint32_t {
            return (row >> 3) * S::SBO + (q >> 2) * 128 + (row & 7) * 16 + (q & 3) * 4;
        };
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (KIND == LT_STATES) {
                const T e[4] = {ra[0][j], ra[1][j], ra[2][j], ra[3][j]};
                store_planes<T>(pa, S::A_PLANE, at_off(trow + j, tkq), e);
            } else {
                store_planes<T>(pa, S::A_PLANE, at_off(krow + 32 * j, kq), ra[j]);
            }
        }
#pragma unroll
        for (int i = 0; i < (B_T ? 4 : BI); i++)
#pragma unroll
            for (int e = 0; e < 4; e++) rb[i][e] = neg ? T(0) - rb[i][e] : p0 * rb[i][e] - rm[i][e];
        if constexpr (B_T) {
            if (b_on) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const T e[4] = {rb[0][j], rb[1][j], rb[2][j], rb[3][j]};
                    store_planes<T>(pb, S::B_PLANE, at_off(trow + j, tkq), e);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < BI; j++) {
                const int w = warp + 8 * j;
                store_planes<T>(pb, S::B_PLANE, at_off(8 * (w >> 1) + (lane >> 2), 4 * (w & 1) + (lane & 3)), rb[j]);
            }
        }
    };

    bool ok = true;
    load_stage(0);
    for (int s = 0; s < steps; s++) {
        const int st = s & 1;
        bool mine = true;
        if (s >= 2) mine = mbar_wait(&bars[st], uint32_t(((s >> 1) - 1) & 1));
        if (mine) store_stage(st);
        if (s + 1 < steps) load_stage(s + 1);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // CTA-uniform: every thread leaves the loop together if any wait gave up
        if (!__syncthreads_and(mine ? 1 : 0)) {
            ok = false;
            break;
        }
        if (tid == 0) {
            tc_fence_after();
            const uint32_t sa = smem_addr(smem + st * S::STAGE);
            const uint64_t db = smem_desc(sa + P * S::A_PLANE, 128, S::SBO);
#pragma unroll
            for (int i = 0; i < P; i++)
                mma_i8(tmem + uint32_t(i * NT), smem_desc(sa + i * S::A_PLANE, 128, S::SBO), db,
                       i8_idesc((P - i) * NT, false), (s > 0 || i > 0) ? 1u : 0u);
            mma_commit(&bars[st]);
        }
    }
    if (ok) ok = mbar_wait(&bars[(steps - 1) & 1], uint32_t(((steps - 1) >> 1) & 1));
    const int all_ok = __syncthreads_and(ok ? 1 : 0);
    tc_fence_after();

    // limb sums -> ring elements, row by row through shared memory for whole-row stores
    T *const tile = reinterpret_cast<T *>(smem);
    if (all_ok) {
        const int q = warp & 3, h = warp >> 2;
#pragma unroll 1
        for (int c = h * (NT / 2); c < (h + 1) * (NT / 2); c += 8) {
            T r[8];
#pragma unroll
            for (int e = 0; e < 8; e++) r[e] = 0;
#pragma unroll
            for (int s = 0; s < P; s++) {
                uint32_t v[8];
                tmem_ld8(tmem + (uint32_t(32 * q) << 16) + uint32_t(s * NT + c), v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 8; e++) r[e] += T(v[e]) << (8 * s);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) tile[(32 * q + lane) * (NT + 1) + c + e] = r[e];
        }
    } else if (tid == 0) {
        atomicOr(err, 8u);
    }
    tc_fence_before();
    __syncthreads();
    if (all_ok) {
        for (int row = warp; row < rows; row += LA_THREADS / 32) {
            const int64_t o = at(row);
            const int n = last(row);
#pragma unroll
            for (int c = lane; c < NT; c += 32)
                if (c < n) out[o + c] = tile[row * (NT + 1) + c] + z[o + c];
        }
    }
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
    }
}

// tiles of chunk c of head bh: score columns 0, NT, .. then state columns 0, NT, ..
template <typename T>
__global__ void __launch_bounds__(LA_THREADS, 2)
    k_la_chunk(const LaShape s, const __grid_constant__ LaChunkArgs<T> a, int score_tiles, int state_tiles, uint32_t *err)
{
    constexpr int NT = LtShape<T>::NT;
    const int per = score_tiles + state_tiles, which = blockIdx.x % per;
    const int64_t bc = blockIdx.x / per, bh = bc / s.chunks();
    const int c = int(bc - bh * s.chunks()), len = s.len(c);
    const int64_t b = bh / s.H, h = bh - b * s.H;
    const int64_t row0 = (b * s.T + int64_t(c) * s.C) * a.ld;
    if (which < score_tiles) {
        const int j0 = which * NT;
        if (j0 >= len) return;
        const int64_t oq = row0 + h * s.dk, ok = oq + int64_t(s.H) * s.dk;
        const bool qv = vec_ok(a.qkv + oq, a.ld) && vec_ok(a.qkv_ms + oq, a.ld);
        const bool kv = vec_ok(a.qkv + ok, a.ld) && vec_ok(a.qkv_ms + ok, a.ld);
        const int nd = (s.dk + 31) / 32;
        const int64_t o = bh * s.tri() + s.tri_at(c) + j0;
        la_tile<T, LT_SCORES>(
            a.qkv_ms ? 2 * nd : nd, a.p0,
            [&](int i) {
                const bool neg = a.qkv_ms && (i & 1);
                LtStep<T> r;
                r.a = (neg ? a.qkv_ms : a.qkv) + oq, r.lda = a.ld, r.a_vec = qv, r.rows = len;
                r.b = a.qkv + ok + j0 * a.ld, r.bm = a.qkv_ms ? a.qkv_ms + ok + j0 * a.ld : nullptr;
                r.ldb = a.ld, r.b_vec = kv, r.cols = len - j0;
                r.k0 = (a.qkv_ms ? i >> 1 : i) * 32, r.K = s.dk, r.neg = neg;
                return r;
            },
            len, [&](int i) { return o + int64_t(i) * (i + 1) / 2; }, [&](int i) { return i + 1 - j0; }, a.z, a.out, err);
    } else {
        const int y0 = (which - score_tiles) * NT;
        const int64_t ok = (bh * s.T + int64_t(c) * s.C) * s.dk;
        const int64_t ov = row0 + 2 * int64_t(s.H) * s.dk + h * s.dv + y0;
        const bool kv = vec_ok(a.kd + ok, s.dk) && vec_ok(a.kd_ms + ok, s.dk);
        const bool vv = vec_ok(a.qkv + ov, a.ld) && vec_ok(a.qkv_ms + ov, a.ld);
        const int nl = (len + 31) / 32;
        const int64_t o = s.n_scores() + ((int64_t(c) * s.bh() + bh) * s.dk) * s.dv + y0;
        la_tile<T, LT_STATES>(
            a.qkv_ms ? 2 * nl : nl, a.p0,
            [&](int i) {
                const bool neg = a.qkv_ms && (i & 1);
                LtStep<T> r;
                r.a = (neg ? a.kd_ms : a.kd) + ok, r.lda = s.dk, r.a_vec = kv, r.rows = s.dk;
                r.b = a.qkv + ov, r.bm = a.qkv_ms ? a.qkv_ms + ov : nullptr, r.ldb = a.ld, r.b_vec = vv;
                r.cols = s.dv - y0, r.k0 = (a.qkv_ms ? i >> 1 : i) * 32, r.K = len, r.neg = neg;
                return r;
            },
            s.dk, [&](int x) { return o + int64_t(x) * s.dv; }, [&](int) { return s.dv - y0; }, a.z, a.out, err);
    }
}

template <typename T>
__global__ void __launch_bounds__(LA_THREADS, 2)
    k_la_output(const LaShape s, const __grid_constant__ LaOutArgs<T> a, int tiles, uint32_t *err)
{
    constexpr int NT = LtShape<T>::NT;
    const int y0 = int(blockIdx.x % tiles) * NT;
    const int64_t bc = blockIdx.x / tiles, bh = bc / s.chunks();
    const int c = int(bc - bh * s.chunks()), len = s.len(c);
    const int64_t b = bh / s.H, h = bh - b * s.H;
    const int64_t op = bh * s.tri() + s.tri_at(c), oq = (bh * s.T + int64_t(c) * s.C) * s.dk;
    const int64_t ov = (b * s.T + int64_t(c) * s.C) * a.ld + 2 * int64_t(s.H) * s.dk + h * s.dv + y0;
    const int64_t os = (c ? s.n_scores() + int64_t(c - 1) * s.n_state() : 0) + bh * s.dk * s.dv + y0;
    const T *const st = c ? a.ps : a.s0, *const st_ms = c ? a.ps_ms : a.s0_ms;
    const bool qv = vec_ok(a.qd + oq, s.dk) && vec_ok(a.qd_ms + oq, s.dk);
    const bool vv = vec_ok(a.qkv + ov, a.ld) && vec_ok(a.qkv_ms + ov, a.ld);
    const bool sv = vec_ok(st + os, s.dv) && vec_ok(st_ms + os, s.dv);
    const int two = a.qkv_ms ? 2 : 1;
    const int nl = two * ((len + 31) / 32), nd = st ? two * ((s.dk + 31) / 32) : 0;
    const int64_t o = ((b * s.T + int64_t(c) * s.C) * s.H + h) * s.dv + y0;
    la_tile<T, LT_OUTPUT>(
        nl + nd, a.p0,
        [&](int i) {
            LtStep<T> r;
            const bool tri = i < nl;
            if (!tri) i -= nl;
            r.neg = two == 2 && (i & 1);
            r.k0 = i / two * 32, r.cols = s.dv - y0, r.rows = len;
            if (tri) {
                r.a = (r.neg ? a.ps_ms : a.ps) + op, r.lda = -1, r.a_vec = false, r.K = len;
                r.b = a.qkv + ov, r.bm = a.qkv_ms ? a.qkv_ms + ov : nullptr, r.ldb = a.ld, r.b_vec = vv;
            } else {
                r.a = (r.neg ? a.qd_ms : a.qd) + oq, r.lda = s.dk, r.a_vec = qv, r.K = s.dk;
                r.b = st + os, r.bm = a.qkv_ms ? st_ms + os : nullptr, r.ldb = s.dv, r.b_vec = sv;
            }
            return r;
        },
        len, [&](int i) { return o + int64_t(i) * s.H * s.dv; }, [&](int) { return s.dv - y0; }, a.z, a.out, err);
}

// ------------------------------------------------------------------ one token
//
// A block takes CX x V columns of one head's state, its 256 / CX thread rows
// stride over dk: S, its mask share and the dealer's word are read once and
// the new state written once (4 words moved and 5 multiply-adds per entry, so
// bound by memory); q . S comes out of the same pass, summed over the thread
// rows in shared memory.
template <typename T, int V>
__global__ void __launch_bounds__(LA_THREADS)
    k_la_step(const LaShape s, const __grid_constant__ LaStepArgs<T> a, int cx, int slabs)
{
    __shared__ T qs[128], ks[128], rq[128], rk[128];
    __shared__ Pack<T, V> red[LA_THREADS];
    using PV = Pack<T, V>;
    const int64_t bh = blockIdx.x / slabs, b = bh / s.H;
    const int slab = int(blockIdx.x - bh * slabs), h = int(bh - b * s.H), tid = threadIdx.x;
    const int ry = LA_THREADS / cx, x = tid % cx, y0 = tid / cx, col = (slab * cx + x) * V;
    const int64_t state = s.n_state(), ny = s.bh() * s.dv, per = int64_t(s.dk) * s.dv;
    const int64_t oq = b * a.ld + int64_t(h) * s.dk, ok = oq + int64_t(s.H) * s.dk;
    const int64_t ov = b * a.ld + 2 * int64_t(s.H) * s.dk + int64_t(h) * s.dv + col;
    const bool on = col < s.dv;
    T v[V], vr[V], acc[V];
#pragma unroll
    for (int k = 0; k < V; k++) {
        v[k] = on ? __ldg(a.qkv + ov + k) : T(0);
        vr[k] = a.p0 * v[k] - (on && a.qkv_ms ? __ldg(a.qkv_ms + ov + k) : T(0));
        acc[k] = 0;
    }
    for (int i = tid; i < s.dk; i += LA_THREADS) {
        qs[i] = __ldg(a.qkv + oq + i), ks[i] = __ldg(a.qkv + ok + i);
        rq[i] = a.qkv_ms ? __ldg(a.qkv_ms + oq + i) : T(0), rk[i] = a.qkv_ms ? __ldg(a.qkv_ms + ok + i) : T(0);
    }
    const T lam = a.lam * __ldg(a.pow + int64_t(h) * (s.pn + 1) + 1);
    __syncthreads();
    if (on) {
        const int64_t at = bh * per + col;
#pragma unroll 4
        for (int i = y0; i < s.dk; i += ry) {
            const int64_t o = at + int64_t(i) * s.dv;
            const PV S = *reinterpret_cast<const PV *>(a.s + o), z = *reinterpret_cast<const PV *>(a.z + o);
            PV m, u;
            if (a.qkv_ms)
                m = *reinterpret_cast<const PV *>(a.s_ms + o);
            else
#pragma unroll
                for (int k = 0; k < V; k++) m.e[k] = 0;
            const T q = qs[i], key = ks[i], mq = rq[i], mk = rk[i];
#pragma unroll
            for (int k = 0; k < V; k++) {
                u.e[k] = z.e[k] + lam * S.e[k] + key * vr[k] - mk * v[k];
                acc[k] += q * (a.p0 * S.e[k] - m.e[k]) - mq * S.e[k];
            }
            *reinterpret_cast<PV *>(a.out + o) = u;
        }
    }
#pragma unroll
    for (int k = 0; k < V; k++) red[tid].e[k] = acc[k];
    for (int half = ry / 2; half; half >>= 1) {
        __syncthreads();
        if (y0 < half)
#pragma unroll
            for (int k = 0; k < V; k++) red[tid].e[k] += red[tid + half * cx].e[k];
    }
    if (y0 == 0 && on)
#pragma unroll
        for (int k = 0; k < V; k++) {
            const int64_t o = state + bh * s.dv + col + k;
            a.out[o] = red[tid].e[k] + a.z[o];
        }
    if (slab == 0 && tid < 32) {
        T w = 0;
        for (int i = tid; i < s.dk; i += 32) w += qs[i] * (a.p0 * ks[i] - rk[i]) - rq[i] * ks[i];
#pragma unroll
        for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        if (tid == 0) a.out[state + ny + bh] = w + a.z[state + ny + bh];
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
    constexpr int V = VEC<T>;
    const int64_t tokens = int64_t(s.B) * s.T;
    const int grid = int(tokens < 148 * 16 ? tokens : 148 * 16);
    if (s.dk % V == 0 && ld % V == 0 && al16(x) && al16(out))
        k_la_decay<T, V><<<grid, LA_THREADS, 0, st>>>(s, ld, pow, x, out);
    else
        k_la_decay<T, 1><<<grid, LA_THREADS, 0, st>>>(s, ld, pow, x, out);
    return launched();
}

template <typename K>
static int la_tile_launch(K kern, uint32_t smem, int64_t blocks, int (&configured)[64], uint32_t **err)
{
    DDG_CHECK(blocks <= 0x7fffffff, DDG_ERR_ARG, "linear attention: %lld tiles are too many for one call",
              (long long)blocks);
    int dev = 0;
    DDG_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        DDG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
        if (dev >= 0 && dev < 64) configured[dev] = 1;
    }
    return ring_gemm_err_word(err);
}

template <typename T>
int la_chunk(const LaShape &s, const LaChunkArgs<T> &a, cudaStream_t st)
{
    if (!s.n_ps()) return DDG_OK;
    using S = LtShape<T>;
    static thread_local int configured[64];
    const int np = (s.len(0) + S::NT - 1) / S::NT, ns = (s.dv + S::NT - 1) / S::NT;
    const int64_t blocks = s.bh() * s.chunks() * (np + ns);
    uint32_t *err = nullptr;
    DDG_TRY(la_tile_launch(k_la_chunk<T>, S::SMEM, blocks, configured, &err));
    k_la_chunk<T><<<unsigned(blocks), LA_THREADS, S::SMEM, st>>>(s, a, np, ns, err);
    return launched();
}

template <typename T, int V>
static int launch_carry(const LaShape &s, const T *pow, const T *ps, const T *s0, T *out, cudaStream_t st)
{
    const int64_t sb = la_blocks(s.n_scores(), V), nb = la_blocks(s.n_state(), V);
    const int score_blocks = int(sb < 148 * 16 ? sb : 148 * 16);
    DDG_CHECK(nb + score_blocks <= 0x7fffffff, DDG_ERR_ARG, "linear attention: %lld state entries are too many",
              (long long)s.n_state());
    k_la_carry<T, V><<<unsigned(score_blocks + nb), LA_THREADS, 0, st>>>(s, pow, ps, s0, out, score_blocks);
    return launched();
}

template <typename T>
int la_carry(const LaShape &s, const T *pow, const T *ps, const T *s0, T *out, cudaStream_t st)
{
    if (!s.n_ps()) return DDG_OK;
    constexpr int V = VEC<T>;
    // 16-byte accesses need both parts of the array and every head's state on 16-byte boundaries
    if (s.n_scores() % V == 0 && int64_t(s.dk) * s.dv % V == 0 && al16(ps) && al16(s0) && al16(out))
        return launch_carry<T, V>(s, pow, ps, s0, out, st);
    return launch_carry<T, 1>(s, pow, ps, s0, out, st);
}

template <typename T>
int la_output(const LaShape &s, const LaOutArgs<T> &a, cudaStream_t st)
{
    if (!s.n_out()) return DDG_OK;
    using S = LtShape<T>;
    static thread_local int configured[64];
    const int tiles = (s.dv + S::NT - 1) / S::NT;
    const int64_t blocks = s.bh() * s.chunks() * tiles;
    uint32_t *err = nullptr;
    DDG_TRY(la_tile_launch(k_la_output<T>, S::SMEM, blocks, configured, &err));
    k_la_output<T><<<unsigned(blocks), LA_THREADS, S::SMEM, st>>>(s, a, tiles, err);
    return launched();
}

template <typename T, int V>
static int launch_step(const LaShape &s, const LaStepArgs<T> &a, cudaStream_t st)
{
    // whole rows of up to 32 x V columns per block; fewer where that leaves SMs idle
    int cx = 32;
    while (cx > 8 && (s.dv <= cx / 2 * V || s.bh() * ((s.dv + cx * V - 1) / (cx * V)) < 2 * 148)) cx /= 2;
    const int slabs = (s.dv + cx * V - 1) / (cx * V);
    DDG_CHECK(s.bh() * slabs <= 0x7fffffff, DDG_ERR_ARG, "linear attention: %lld heads are too many for one call",
              (long long)s.bh());
    k_la_step<T, V><<<unsigned(s.bh() * slabs), LA_THREADS, 0, st>>>(s, a, cx, slabs);
    return launched();
}

template <typename T>
int la_step(const LaShape &s, const LaStepArgs<T> &a, cudaStream_t st)
{
    if (!s.bh()) return DDG_OK;
    constexpr int V = VEC<T>;
    if (s.dv % V == 0 && al16(a.s) && al16(a.s_ms) && al16(a.z) && al16(a.out)) return launch_step<T, V>(s, a, st);
    return launch_step<T, 1>(s, a, st);
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
