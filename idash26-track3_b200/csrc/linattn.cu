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
// cores in la_tiles: 128 rows x NT columns of sum_p A_p . B_p, ring operands
// split into bytes by the loading threads, limb sums
//   C = sum_s 2^(8s) sum_{i+j=s} A_i . B_j  (u8 x u8 -> s32, exact: K <= 512)
// in tensor memory.  The limbs of B are stacked along N, so one MMA per limb i
// of A covers every j with i + j < P, landing in the columns of s = i .. P-1.
//
// Measured on one B200 for 4 x 16 heads x 2048 tokens x 64 x 64 over Z_2^32 (ncu):
// decay 29 us (4.6 TB/s), chunk stage 131 us (2.8 TB/s of 369 MB), carry 28 us
// (3.6 TB/s), output stage 85 us (3.6 TB/s of 302 MB).
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

// chunk, row and column of entry e of one head's score triangles (e < 2^31: LA_MAX_CHUNKS)
__device__ __forceinline__ void tri_find(const LaShape &s, int64_t e, int &c, int &i, int &j)
{
    const uint32_t full = uint32_t(s.C) * uint32_t(s.C + 1) / 2;
    c = int(uint32_t(e) / full);
    const int r = int(uint32_t(e) - uint32_t(c) * full);
    i = int((sqrtf(8.f * float(r) + 1.f) - 1.f) * 0.5f);
    if ((i + 1) * (i + 2) / 2 <= r) i++;
    if (i * (i + 1) / 2 > r) i--;
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
            const T p = __ldg(pow + s.pow_at(uint32_t(h)) + (key ? back : i + 1));
            Pack<T, V> v = row[e];
#pragma unroll
            for (int j = 0; j < V; j++) v.e[j] *= p;
            reinterpret_cast<Pack<T, V> *>(out + (key ? nd : 0) + ((b * s.H + h) * s.T + t) * s.dk)[d] = v;
        }
    }
}

// Blocks take a slice of one head's scores or of one head's states.
// Scores: V packed entries at a time, the triangle walked from the first one's
// position.  States: V entries of LC_OT output chunks per thread; every earlier
// chunk is read once per LC_OT outputs, against a table of decays in shared
// memory.  The sums cannot be chained from chunk to chunk, because each S_c is
// floored from exact terms.
constexpr int LC_OT = 8, LC_SLICE = 4 * LA_THREADS;  // slice: vectors per block, four a thread

template <typename T, int V>
__global__ void __launch_bounds__(LA_THREADS, 3)
    k_la_carry(const LaShape s, const T *pow, const T *ps, const T *s0, T *out, int state_slices, int score_slices,
               int64_t state_blocks)
{
    __shared__ T w[LC_OT][LC_OT];  // [j][o]: decay from chunk j0 + j to chunk c0 + o
    const int64_t ns = s.n_scores(), state = s.n_state();
    const int nc = s.chunks();
    if (blockIdx.x >= state_blocks) {
        const uint32_t block = uint32_t(blockIdx.x - state_blocks), bh = block / uint32_t(score_slices);
        const int64_t tri = s.tri(), base = int64_t(bh) * tri;
        const T *const pw = pow + s.pow_at(bh % uint32_t(s.H));
        // whole vectors start on multiples of V of the array, so the head's first may be cut
        const int64_t lo = (block - bh * uint32_t(score_slices)) * int64_t(LC_SLICE * V) - base % V;
        constexpr int PER = LC_SLICE / LA_THREADS;
        Pack<T, V> v[PER];
        // every load before the first use: what is in flight is what this part's time goes by
#pragma unroll
        for (int p = 0; p < PER; p++) {
            const int64_t r0 = lo + (p * LA_THREADS + int(threadIdx.x)) * V;
            if (r0 >= 0 && r0 + V <= tri)
                v[p] = *reinterpret_cast<const Pack<T, V> *>(ps + base + r0);
            else
#pragma unroll
                for (int k = 0; k < V; k++) v[p].e[k] = r0 + k >= 0 && r0 + k < tri ? ps[base + r0 + k] : T(0);
        }
#pragma unroll
        for (int p = 0; p < PER; p++) {
            const int64_t r0 = lo + (p * LA_THREADS + int(threadIdx.x)) * V;
            if (r0 >= tri) break;
            const int skip = r0 < 0 ? int(-r0) : 0, n = tri - r0 < V ? int(tri - r0) : V;
            if (skip >= n) continue;
            int c, i, j;
            tri_find(s, r0 + skip, c, i, j);
            int len = s.len(c);
#pragma unroll
            for (int k = 0; k < V; k++) {
                if (k < skip || k >= n) continue;
                v[p].e[k] *= __ldg(pw + i - j);
                if (++j > i) {  // next row or chunk
                    j = 0;
                    if (++i >= len && c + 1 < nc) i = 0, len = s.len(++c);
                }
            }
            if (!skip && n == V)
                *reinterpret_cast<Pack<T, V> *>(out + base + r0) = v[p];
            else
#pragma unroll
                for (int k = 0; k < V; k++)
                    if (k >= skip && k < n) out[base + r0 + k] = v[p].e[k];
        }
        return;
    }
    const uint32_t block = blockIdx.x, bh = block / uint32_t(state_slices);
    const int per = s.dk * s.dv, at = int(block - bh * uint32_t(state_slices)) * LA_THREADS * V + threadIdx.x * V;
    const T *const pw = pow + s.pow_at(bh % uint32_t(s.H));
    const bool on = at < per;
    const int64_t r = int64_t(bh) * per + (on ? at : 0);
    const T *const in = ps + ns + r;
    Pack<T, V> first;
#pragma unroll
    for (int k = 0; k < V; k++) first.e[k] = 0;
    if (s0) first = *reinterpret_cast<const Pack<T, V> *>(s0 + r);
    for (int c0 = 0; c0 < nc; c0 += LC_OT) {
        T acc[LC_OT][V];
#pragma unroll
        for (int o = 0; o < LC_OT; o++) {
            const T p = s0 && c0 + o < nc ? __ldg(pw + s.end(c0 + o)) : T(0);
#pragma unroll
            for (int k = 0; k < V; k++) acc[o][k] = p * first.e[k];
        }
        for (int j0 = 0; j0 <= c0; j0 += LC_OT) {
            __syncthreads();
            if (threadIdx.x < LC_OT * LC_OT) {
                const int j = j0 + threadIdx.x / LC_OT, c = c0 + threadIdx.x % LC_OT;
                w[threadIdx.x / LC_OT][threadIdx.x % LC_OT] = c < nc && j <= c ? __ldg(pw + s.end(c) - s.end(j)) : T(0);
            }
            __syncthreads();
            const int jn = nc - j0 < LC_OT ? nc - j0 : LC_OT;
            for (int j = 0; j < jn; j += 4) {
                Pack<T, V> v[4];
#pragma unroll
                for (int q = 0; q < 4; q++)
                    v[q] = *reinterpret_cast<const Pack<T, V> *>(in + int64_t(j0 + (j + q < jn ? j + q : j)) * state);
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int o = 0; o < LC_OT; o++) {
                        const T p = j + q < jn ? w[j + q][o] : T(0);
#pragma unroll
                        for (int k = 0; k < V; k++) acc[o][k] += p * v[q].e[k];
                    }
            }
        }
        if (on)
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

// Persistent kernels, two CTAs per SM over strided lists of tiles.  Eight warps
// load the operands of the next K-step into registers (no detour through shared
// memory, whose bandwidth the planes and the MMAs' own reads take), split the
// present one into planes and hand the stage over by mbarrier; there is no
// CTA-wide barrier in the loop, and loads run on across tiles.  What bounds
// these kernels is the loads' latency against what the registers hold in flight
// (the largest wait of every warp, 2.4 of 8 cycles an instruction, over Z_2^64 6.2
// of 11.5; issue 0.47 and 0.32, tensor pipe 16 to 23 %, DRAM a third), so every load
// covers whole 128-byte lines and whole tiles take loads without bounds.
constexpr int LT_WARPS = 8, LT_THREADS = LT_WARPS * 32;

template <typename T>
struct LtShape {
    static constexpr int P = int(sizeof(T));
    static constexpr int NT = 256 / P;             // tile columns: P x NT = 256 accumulator columns
    static constexpr int NSTAGE = P == 4 ? 3 : 2;
    // 8-row groups of the operand planes 272 instead of 256 bytes apart: the
    // transposing loaders store rows 4 apart, which then fall on distinct banks
    static constexpr uint32_t SBO = 272;
    static constexpr uint32_t A_PLANE = TC_BM / 8 * SBO, B_PLANE = NT / 8 * SBO;
    static constexpr uint32_t STAGE = P * (A_PLANE + B_PLANE);
    // the output tile on its way to whole-row stores lies in the stages, empty between two tiles
    static_assert(TC_BM * (NT + 1) * sizeof(T) <= NSTAGE * STAGE, "output tile");
    static constexpr uint32_t DESC = LT_WARPS * 4 * 192;            // every warp's descriptions of the tiles in hand
    static constexpr uint32_t SMEM = 128 + 1024 + NSTAGE * STAGE + DESC + 1024;
};

template <typename T>
__device__ __forceinline__ bool aligned16(const T *p, int64_t ld)
{
    return ((reinterpret_cast<uintptr_t>(p) | uintptr_t(ld * int64_t(sizeof(T)))) & 15) == 0;
}

// four elements at p as 16-byte accesses
template <typename T>
__device__ __forceinline__ void load4(const T *p, T (&e)[4])
{
#pragma unroll
    for (int i = 0; i < int(sizeof(T)) / 4; i++)
        *reinterpret_cast<uint4 *>(e + i * (16 / int(sizeof(T)))) = __ldg(reinterpret_cast<const uint4 *>(p) + i);
}
// the first n of them, zeros behind; vec: 16-byte accesses where all four are there
template <typename T>
__device__ __forceinline__ void load4(const T *p, int n, bool vec, T (&e)[4])
{
    if (vec && n >= 4) {
        load4<T>(p, e);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = i < n ? __ldg(p + i) : T(0);
    }
}

// Which product a tile belongs to, by how its operands lie.
//   LT_SCORES  A = q (rows of k), B = k (rows of k)
//   LT_STATES  A = Kd, B = V (both k-major: a row per token)
//   LT_OUTPUT  first A = P (packed causal triangle), B = V (k-major), then A = Qd (rows of k), B = S (k-major)
enum { LT_SCORES = 0, LT_STATES = 1, LT_OUTPUT = 2 };
template <typename T>
struct LtPair {
    const T *a, *a_ms, *b, *b_ms;
    int64_t lda, ldb;
    int K;
    bool vec_a, vec_b;      // 16-byte boundaries
    bool whole_a, whole_b;  // and every load inside
};

// A tile: rows x cols valid of 128 x NT, column j of row i at at + stride * i + j
// (scores: at + i (i + 1) / 2 + j, entries with j0 + j <= i)
template <typename T>
struct LtTile {
    LtPair<T> p[2];
    int steps0, steps;  // K-steps of the first pair, of all
    int rows, cols, j0;
    int64_t at, stride;
};

// (bar.sync is .aligned: the lanes of a warp arrive together, whatever rows and columns they have stored)
__device__ __forceinline__ void expander_sync()
{
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(LT_THREADS) : "memory");
}

// Tiles first, first + step, .. below `tiles`; tile_of(index) describes one.
// beaver: with the mask-share products (odd K-steps are -[a] . b), else the
// plain product (the dealer's word).
template <typename T, int KIND, class TileOf>
__device__ __forceinline__ void la_tiles(int64_t first, int64_t step, int64_t tiles, TileOf tile_of, T p0, bool beaver,
                                         const T *z, T *out, uint32_t *err)
{
    using S = LtShape<T>;
    constexpr int P = S::P, NT = S::NT, NST = S::NSTAGE;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint64_t *const empty = reinterpret_cast<uint64_t *>(smem_raw), *const full = empty + NST;
    uint32_t &s_tmem = *reinterpret_cast<uint32_t *>(smem_raw + 96);
    uint8_t *const smem = smem_raw + 128 + ((1024u - ((smem_addr(smem_raw) + 128u) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                     "r"(256)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < NST; i++) mbar_init(empty + i, 1), mbar_init(full + i, LT_WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    // A wait that gave up turns `ok` off: the warp then runs through its remaining
    // arrivals and barriers without waiting or writing, and the launch reports it.
    bool ok = true;

    {
        // Warp 0 also issues the MMAs, a step's at the start of the next one, when the other warps' planes are
        // likely there (a warp of its own for them would leave 96 registers a thread instead of 128).
        const bool leader = elect_one();
        auto multiply = [&](uint32_t g, bool first) {
            const uint32_t st = g % NST;
            if (ok) ok = mbar_wait(&full[st], (g / NST) & 1);
            tc_fence_after();
            if (ok && leader) {
                const uint32_t sa = smem_addr(smem + st * S::STAGE);
                const uint64_t da = smem_desc(sa, 128, S::SBO), db = smem_desc(sa + P * S::A_PLANE, 128, S::SBO);
#pragma unroll
                for (int i = 0; i < P; i++)  // the address field counts 16-byte units
                    mma_i8(tmem + uint32_t(i * NT), da + uint64_t(i * S::A_PLANE >> 4), db, i8_idesc((P - i) * NT, false),
                           (!first || i > 0) ? 1u : 0u);
                mma_commit(&empty[st]);
            }
            __syncwarp();
        };
        // This thread's items of a K-step.  Rows of k: A rows krow + 32 j, B rows (columns of the tile)
        // brow + 32 j, four k from 4 kq.  k-major: 4 x 4 blocks of rows trow.. and k 4 tkq.. .
        constexpr bool A_T = KIND == LT_STATES, B_T = KIND != LT_SCORES;
        // (P = 8: 32 columns; one column and four k a thread, to save registers)
        constexpr bool B_ONE = B_T && P == 8;
        constexpr int BI = B_ONE ? 1 : B_T ? 4 : NT / 32;
        const int kq = 4 * (warp & 1) + (lane & 3), krow = 8 * (warp >> 1) + (lane >> 2);
        const int tkq = 4 * (warp & 1) + (lane >> 3), trow = 4 * (8 * (warp >> 1) + (lane & 7));
        const int bcol = 8 * (warp >> 1) + (lane & 7);
        const bool b_on = !B_T || B_ONE || trow < NT;
        struct Regs {
            T a[4][4], b[BI][4], m[BI][4];
            bool neg;
            int skip;  // scores: rows above the tile's first column have no entry in it, their items stay out
        };

        auto load = [&](const LtTile<T> &t, int s, Regs &r) {
            const bool second = KIND == LT_OUTPUT && s >= t.steps0;
            const LtPair<T> &p = t.p[second ? 1 : 0];
            const int i = second ? s - t.steps0 : s;
            r.skip = KIND == LT_SCORES ? t.j0 >> 5 : 0;
            r.neg = beaver && (i & 1);
            const int k0 = (beaver ? i >> 1 : i) * 32;
            const T *const a = r.neg ? p.a_ms : p.a;
            const int64_t lda = p.lda, ldb = p.ldb;
            if constexpr (A_T) {
                const T *q = a + int64_t(k0 + 4 * tkq) * lda + trow;
                if (p.whole_a) {
#pragma unroll
                    for (int e = 0; e < 4; e++, q += lda) load4<T>(q, r.a[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++, q += lda) load4<T>(q, k0 + 4 * tkq + e < p.K ? t.rows - trow : 0, p.vec_a, r.a[e]);
                }
            } else if (KIND == LT_OUTPUT && !second) {
                const int k = k0 + 4 * kq;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int row = krow + 32 * j;
                    load4<T>(a + row * (row + 1) / 2 + k, row < t.rows ? row + 1 - k : 0, false, r.a[j]);
                }
            } else {
                const T *q = a + krow * lda + k0 + 4 * kq;
                if (p.whole_a) {
#pragma unroll
                    for (int j = 0; j < 4; j++, q += 32 * lda)
                        if (j >= r.skip) load4<T>(q, r.a[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++, q += 32 * lda)
                        if (j >= r.skip) load4<T>(q, krow + 32 * j < t.rows ? p.K - k0 - 4 * kq : 0, p.vec_a, r.a[j]);
                }
            }
            // the second step of a pair takes the B of the first, still in its registers
            if (!b_on || r.neg) return;
            if constexpr (B_ONE) {
                const int64_t o = int64_t(k0 + 4 * tkq) * ldb + bcol;
                const int n = p.whole_b ? 4 : bcol < t.cols ? p.K - k0 - 4 * tkq : 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    r.b[0][e] = e < n ? __ldg(p.b + o + e * ldb) : T(0);
                    r.m[0][e] = beaver && e < n ? __ldg(p.b_ms + o + e * ldb) : T(0);
                }
                return;
            }
            const int64_t o = B_T ? int64_t(k0 + 4 * tkq) * ldb + trow : krow * ldb + k0 + 4 * kq;
            const int64_t inc = B_T ? ldb : 32 * ldb;
            const T *q = p.b + o, *m = p.b_ms + o;
            if (p.whole_b) {
#pragma unroll
                for (int e = 0; e < BI; e++, q += inc) load4<T>(q, r.b[e]);
                if (beaver) {
#pragma unroll
                    for (int e = 0; e < BI; e++, m += inc) load4<T>(m, r.m[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < BI; e++, q += inc, m += inc) {
                    const int n = B_T ? (k0 + 4 * tkq + e < p.K ? t.cols - trow : 0)
                                      : (krow + 32 * e < t.cols ? p.K - k0 - 4 * kq : 0);
                    load4<T>(q, n, p.vec_b, r.b[e]);
                    if (beaver) load4<T>(m, n, p.vec_b, r.m[e]);
                }
            }
        };
        auto at_off = [](int row, int q) -> uint32_t {
            return (row >> 3) * S::SBO + (q >> 2) * 128 + (row & 7) * 16 + (q & 3) * 4;
        };
        const uint32_t a_off = A_T ? at_off(trow, tkq) : at_off(krow, kq), a_inc = A_T ? 16 : 4 * S::SBO;
        const uint32_t b_off = B_ONE ? at_off(bcol, tkq) : B_T ? at_off(trow, tkq) : at_off(krow, kq), b_inc = B_T ? 16 : 4 * S::SBO;
        auto split = [&](Regs &r, uint32_t st) {
            uint8_t *const pa = smem + st * S::STAGE + a_off, *const pb = smem + st * S::STAGE + P * S::A_PLANE + b_off;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const T e[4] = {A_T ? r.a[0][j] : r.a[j][0], A_T ? r.a[1][j] : r.a[j][1], A_T ? r.a[2][j] : r.a[j][2],
                                A_T ? r.a[3][j] : r.a[j][3]};
                if (j >= r.skip) store_planes<T>(pa, S::A_PLANE, j * a_inc, e);
            }
            if (!b_on) return;
            auto planes = [&](auto &&right) {
#pragma unroll
                for (int j = 0; j < BI; j++) {
                    constexpr bool X = B_T && !B_ONE;
                    const T e[4] = {X ? right(0, j) : right(j, 0), X ? right(1 % BI, j) : right(j, 1),
                                    X ? right(2 % BI, j) : right(j, 2), X ? right(3 % BI, j) : right(j, 3)};
                    store_planes<T>(pb, S::B_PLANE, j * b_inc, e);
                }
            };
            if (r.neg)
                planes([&](int i, int e) { return T(0) - r.b[i][e]; });
            else if (beaver)
                planes([&](int i, int e) { return p0 * r.b[i][e] - r.m[i][e]; });
            else
                planes([&](int i, int e) { return r.b[i][e]; });
        };

        T *const tile = reinterpret_cast<T *>(smem);
        // one tile's accumulators (complete with K-step `last`) to memory; the next tile's MMAs wait for
        // planes that every warp hands over only after this
        auto epilogue = [&](const LtTile<T> &t, uint32_t last) {
            constexpr int RW = TC_BM / LT_WARPS, CW = NT / 32, U = 8;  // rows per warp, pieces per row, rows in flight
            if (ok) ok = mbar_wait(&empty[last % NST], (last / NST) & 1);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            const int q = warp & 3;
            if (ok) {
#pragma unroll 2
                for (int c = (warp >> 2) * (NT / 2); c < (warp >> 2) * (NT / 2) + NT / 2; c += 8) {
                    uint32_t v[P][8];
#pragma unroll
                    for (int s = 0; s < P; s++)
                        tmem_ld8(tmem + (uint32_t(32 * q) << 16) + uint32_t(s * NT + c), v[s]);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        T r = 0;
#pragma unroll
                        for (int s = 0; s < P; s++) r += T(v[s][e]) << (8 * s);
                        tile[(32 * q + lane) * (NT + 1) + c + e] = r;
                    }
                }
            }
            tc_fence_before();
            expander_sync();
#pragma unroll 1
            for (int i0 = 0; i0 < RW; i0 += U) {
                if (!ok || warp + LT_WARPS * i0 >= t.rows) break;
                T add[U][CW];
                const T *zr = z + t.at;
                T *const orow = out + t.at;
                auto row_at = [&](int row) {
                    return KIND == LT_SCORES ? int64_t(row * (row + 1) / 2) : t.stride * row;
                };
                auto width = [&](int row) { return row >= t.rows ? 0 : KIND == LT_SCORES ? row + 1 - t.j0 : t.cols; };
#pragma unroll
                for (int i = 0; i < U; i++) {
                    const int row = warp + LT_WARPS * (i0 + i), w = width(row);
                    const T *const zp = zr + row_at(row) + lane;
#pragma unroll
                    for (int c = 0; c < CW; c++) add[i][c] = lane + 32 * c < w ? zp[32 * c] : T(0);
                }
#pragma unroll
                for (int i = 0; i < U; i++) {
                    const int row = warp + LT_WARPS * (i0 + i), w = width(row);
                    T *const op = orow + row_at(row) + lane;
#pragma unroll
                    for (int c = 0; c < CW; c++)
                        if (lane + 32 * c < w) op[32 * c] = tile[row * (NT + 1) + lane + 32 * c] + add[i][c];
                }
            }
            expander_sync();  // the stages may be filled again
        };

        // the K-steps of this CTA's tiles, one list: loads run a step ahead of the splits
        static_assert(sizeof(LtTile<T>) <= 192, "tile descriptions");
        uint8_t *const desc = smem + NST * S::STAGE + warp * 4 * 192;
        auto slot = [&](uint32_t i) -> LtTile<T> & { return *reinterpret_cast<LtTile<T> *>(desc + (i & 3) * 192); };
        auto describe = [&](uint32_t i, int64_t index) {  // tile i of this CTA, for the lanes of this warp
            const LtTile<T> t = tile_of(index);
            __syncwarp();
            if (lane == 0) slot(i) = t;
            __syncwarp();
        };
        Regs r;
        int64_t li = first, ci = first;  // tile being loaded, being split
        int ls = 0, cs = 0;
        uint32_t g = 0, n = 0, ln = 0;
        if (first < tiles) describe(0, first);
        auto load_next = [&]() {
            if (li >= tiles) return;
            load(slot(ln), ls, r);
            if (++ls == slot(ln).steps) {
                ls = 0, li += step;
                if (li < tiles) describe(++ln, li);
            }
        };
        load_next();
        while (ci < tiles) {
            const uint32_t st = g % NST;
            if (warp == 0 && cs > 0) multiply(g - 1, cs == 1);
            if (g >= NST && ok) ok = mbar_wait(&empty[st], (g / NST - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) split(r, st);
            load_next();
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[st]);
            g++;
            if (++cs == slot(n).steps) {
                if (warp == 0) multiply(g - 1, cs == 1);
                epilogue(slot(n), g - 1);
                n++, cs = 0, ci += step;
            }
        }
        if (!ok && lane == 0) atomicOr(err, 8u);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
    }
}

inline __host__ __device__ int steps32(int k) { return (k + 31) / 32; }

// CTAs below score_ctas take score tiles (columns 0, NT, .. of each chunk), the others state tiles
template <typename T>
__global__ void __launch_bounds__(LT_THREADS, 2)
    k_la_chunk(const LaShape s, const __grid_constant__ LaChunkArgs<T> a, int score_tiles, int state_tiles, int score_ctas,
               uint32_t *err)
{
    constexpr int NT = LtShape<T>::NT;
    const int two = a.qkv_ms ? 2 : 1, nc = s.chunks();
    const int64_t chunks = s.bh() * nc, kd0 = int64_t(s.H) * s.dk;
    struct Spot {
        int64_t b, h, bh, row0;
        int c, len, which;
    };
    auto find = [&](int64_t index, int per) {
        Spot f;
        // heads before chunks before sequences: what runs at one time reads whole q|k|v rows
        const int64_t r = index / per, bc = r / s.H;
        f.which = int(index - r * per), f.h = r - bc * s.H, f.b = bc / nc, f.c = int(bc - f.b * nc);
        f.bh = f.b * s.H + f.h, f.len = s.len(f.c);
        f.row0 = (f.b * s.T + int64_t(f.c) * s.C) * a.ld;
        return f;
    };
    if (int(blockIdx.x) < score_ctas) {
        auto tile_of = [&](int64_t index) {
            const Spot f = find(index, score_tiles);
            const int j0 = f.which * NT;
            const int64_t oq = f.row0 + f.h * s.dk, ok = oq + kd0 + int64_t(j0) * a.ld;
            LtTile<T> t;
            LtPair<T> &p = t.p[0];
            p.a = a.qkv + oq, p.a_ms = a.qkv_ms + oq, p.b = a.qkv + ok, p.b_ms = a.qkv_ms + ok;
            p.lda = p.ldb = a.ld, p.K = s.dk;
            // a short chunk's last column tiles may be empty: no rows
            t.rows = j0 < f.len ? f.len : 0, t.cols = j0 < f.len ? f.len - j0 : 0, t.j0 = j0;
            p.vec_a = aligned16(p.a, a.ld) && aligned16(p.a_ms, a.ld);
            p.vec_b = aligned16(p.b, a.ld) && aligned16(p.b_ms, a.ld);
            p.whole_a = p.vec_a && t.rows == TC_BM && s.dk % 32 == 0;
            p.whole_b = p.vec_b && t.cols >= NT && s.dk % 32 == 0;
            t.at = f.bh * s.tri() + s.tri_at(f.c) + j0, t.stride = 0;
            t.steps0 = t.steps = two * steps32(s.dk);
            return t;
        };
        la_tiles<T, LT_SCORES>(blockIdx.x, score_ctas, chunks * score_tiles, tile_of, a.p0, two == 2, a.z, a.out, err);
    } else {
        auto tile_of = [&](int64_t index) {
            const Spot f = find(index, state_tiles);
            const int y0 = f.which * NT;
            const int64_t ok = (f.bh * s.T + int64_t(f.c) * s.C) * s.dk, ov = f.row0 + 2 * kd0 + f.h * s.dv + y0;
            LtTile<T> t;
            LtPair<T> &p = t.p[0];
            p.a = a.kd + ok, p.a_ms = a.kd_ms + ok, p.b = a.qkv + ov, p.b_ms = a.qkv_ms + ov;
            p.lda = s.dk, p.ldb = a.ld, p.K = f.len;
            t.rows = s.dk, t.cols = s.dv - y0, t.j0 = 0;
            p.vec_a = aligned16(p.a, s.dk) && aligned16(p.a_ms, s.dk);
            p.vec_b = aligned16(p.b, a.ld) && aligned16(p.b_ms, a.ld);
            p.whole_a = p.vec_a && s.dk == TC_BM && f.len % 32 == 0;
            p.whole_b = p.vec_b && t.cols >= NT && f.len % 32 == 0;
            t.at = s.n_scores() + (int64_t(f.c) * s.bh() + f.bh) * s.dk * s.dv + y0, t.stride = s.dv;
            t.steps0 = t.steps = two * steps32(f.len);
            return t;
        };
        la_tiles<T, LT_STATES>(blockIdx.x - score_ctas, gridDim.x - score_ctas, chunks * state_tiles, tile_of, a.p0,
                               two == 2, a.z, a.out, err);
    }
}

// tiles of chunk c of head bh: output columns 0, NT, ..
template <typename T>
__global__ void __launch_bounds__(LT_THREADS, 2)
    k_la_output(const LaShape s, const __grid_constant__ LaOutArgs<T> a, int64_t count, int tiles, uint32_t *err)
{
    constexpr int NT = LtShape<T>::NT;
    const int two = a.qkv_ms ? 2 : 1, nc = s.chunks();
    auto tile_of = [&](int64_t index) {
        const int64_t r = index / tiles, bc = r / s.H, h = r - bc * s.H, b = bc / nc, bh = b * s.H + h;
        const int y0 = int(index - r * tiles) * NT, c = int(bc - b * nc), len = s.len(c);
        const int64_t t0 = b * s.T + int64_t(c) * s.C;
        const int64_t op = bh * s.tri() + s.tri_at(c), oq = (bh * s.T + int64_t(c) * s.C) * s.dk;
        const int64_t ov = t0 * a.ld + 2 * int64_t(s.H) * s.dk + h * s.dv + y0;
        const int64_t os = (c ? s.n_scores() + int64_t(c - 1) * s.n_state() : 0) + bh * s.dk * s.dv + y0;
        const T *const st = c ? a.ps : a.s0, *const st_ms = c ? a.ps_ms : a.s0_ms;
        LtTile<T> t;
        LtPair<T> &p = t.p[0], &q = t.p[1];
        t.rows = len, t.cols = s.dv - y0, t.j0 = 0;
        p.a = a.ps + op, p.a_ms = a.ps_ms + op, p.b = a.qkv + ov, p.b_ms = a.qkv_ms + ov;
        p.lda = 0, p.ldb = a.ld, p.K = len, p.vec_a = p.whole_a = false;
        p.vec_b = aligned16(p.b, a.ld) && aligned16(p.b_ms, a.ld);
        p.whole_b = p.vec_b && t.cols >= NT && len % 32 == 0;
        q.a = a.qd + oq, q.a_ms = a.qd_ms + oq, q.b = st + os, q.b_ms = st_ms + os;
        q.lda = s.dk, q.ldb = s.dv, q.K = s.dk;
        q.vec_a = aligned16(q.a, s.dk) && aligned16(q.a_ms, s.dk);
        q.vec_b = aligned16(q.b, s.dv) && aligned16(q.b_ms, s.dv);
        q.whole_a = q.vec_a && len == TC_BM && s.dk % 32 == 0;
        q.whole_b = q.vec_b && t.cols >= NT && s.dk % 32 == 0;
        t.steps0 = two * steps32(len), t.steps = t.steps0 + (st ? two * steps32(s.dk) : 0);
        t.at = (t0 * s.H + h) * s.dv + y0, t.stride = int64_t(s.H) * s.dv;
        return t;
    };
    la_tiles<T, LT_OUTPUT>(blockIdx.x, gridDim.x, count, tile_of, a.p0, two == 2, a.z, a.out, err);
}

// ------------------------------------------------------------------ matrix stages of a few heads
//
// The same products on the CUDA cores, in 32 x 32 tiles, for calls whose few
// 128-row tiles would leave most SMs idle and run at one tile's latency.  256
// threads load 32 k at a time, the next ones on their way in registers; four
// groups of 64 threads take 8 k each, 4 x 4 entries a thread, and their sums meet
// in shared memory.  (4 x 1 entries a thread, all k, read shared memory more often
// than they multiplied: the chunk stage of 8 heads x 128 tokens x 64 took 7.9 us
// instead of 7.0.)
template <typename T>
struct LsTile {
    LtPair<T> p[2];
    int pairs, rows, cols, i0, j0;  // the product's extent, this tile's corner
    int64_t at, stride;             // as LtTile, from row 0 and column 0
};

template <typename T>
constexpr int LS_W = 32 + VEC<T>;  // row pitch: 16-byte reads, off the banks of the next row
template <typename T, int KIND>
__device__ __forceinline__ void ls_tile(T (&sm)[4][32][LS_W<T>], const LsTile<T> &t, T p0, bool beaver, const T *z, T *out)
{
    // A, -[A] (k, row); p0 B - [B], B (k, column)
    auto &as = sm[0], &am = sm[1], &br = sm[2], &bs = sm[3];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int group = threadIdx.x >> 6, ty = 4 * ((threadIdx.x & 63) >> 3), tx = 4 * (threadIdx.x & 7);
    T acc[4][4] = {};
    T ra[4], rm[4], rb[4], rn[4];
    auto load = [&](int which, int k0) {
        LtPair<T> p = t.p[0];  // (indexed by `which` it would lie in local memory)
        if (KIND == LT_OUTPUT && which) p = t.p[1];
        const bool tri = KIND == LT_OUTPUT && which == 0;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int y4 = y + 8 * q;
            {  // A: x runs along what is contiguous
                const int row = t.i0 + (KIND == LT_STATES ? x : y4), k = k0 + (KIND == LT_STATES ? y4 : x);
                const bool in = row < t.rows && k < p.K && (!tri || k <= row);
                const int64_t o = KIND == LT_STATES ? k * p.lda + row : tri ? row * (row + 1) / 2 + k : row * p.lda + k;
                ra[q] = in ? __ldg(p.a + o) : T(0), rm[q] = in && beaver ? __ldg(p.a_ms + o) : T(0);
            }
            {
                const int col = t.j0 + (KIND == LT_SCORES ? y4 : x), k = k0 + (KIND == LT_SCORES ? x : y4);
                const bool in = col < t.cols && k < p.K;
                const int64_t o = KIND == LT_SCORES ? col * p.ldb + k : k * p.ldb + col;
                rb[q] = in ? __ldg(p.b + o) : T(0), rn[q] = in && beaver ? __ldg(p.b_ms + o) : T(0);
            }
        }
    };
    // entries right of a causal tile's last row add nothing
    auto length = [&](int which) {
        if (KIND != LT_OUTPUT) return t.p[0].K;
        return which ? t.p[1].K : t.i0 + 32 < t.p[0].K ? t.i0 + 32 : t.p[0].K;
    };
    int which = 0, k0 = 0;
    load(0, 0);
    while (which < t.pairs) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int y4 = y + 8 * q;
            (KIND == LT_STATES ? as[y4][x] : as[x][y4]) = ra[q], (KIND == LT_STATES ? am[y4][x] : am[x][y4]) = T(0) - rm[q];
            (KIND == LT_SCORES ? br[x][y4] : br[y4][x]) = p0 * rb[q] - rn[q];
            (KIND == LT_SCORES ? bs[x][y4] : bs[y4][x]) = rb[q];
        }
        __syncthreads();
        k0 += 32;
        if (k0 >= length(which)) which++, k0 = 0;
        if (which < t.pairs) load(which, k0);
        auto four = [](const T *p, T (&e)[4]) {
#pragma unroll
            for (int i = 0; i < 4; i += VEC<T>) {
                const Pack<T, VEC<T>> v = *reinterpret_cast<const Pack<T, VEC<T>> *>(p + i);
#pragma unroll
                for (int j = 0; j < VEC<T>; j++) e[i + j] = v.e[j];
            }
        };
#pragma unroll
        for (int k = 8 * group, n = 0; n < 8; n++, k++) {
            T a[4], m[4], r[4], b[4];
            four(&as[k][ty], a), four(&am[k][ty], m), four(&br[k][tx], r), four(&bs[k][tx], b);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] += a[i] * r[j] + m[i] * b[j];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j += VEC<T>) {
            Pack<T, VEC<T>> v;
#pragma unroll
            for (int e = 0; e < VEC<T>; e++) v.e[e] = acc[i][j + e];
            *reinterpret_cast<Pack<T, VEC<T>> *>(&sm[group][ty + i][tx + j]) = v;
        }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int row = t.i0 + y + 8 * q, col = t.j0 + x;
        if (row >= t.rows || col >= t.cols || (KIND == LT_SCORES && col > row)) continue;
        const int64_t o = t.at + (KIND == LT_SCORES ? int64_t(row) * (row + 1) / 2 : t.stride * row) + col;
        const int a = y + 8 * q;
        out[o] = sm[0][a][x] + sm[1][a][x] + sm[2][a][x] + sm[3][a][x] + z[o];
    }
}

// per chunk of a head: score_tiles tiles of the causal triangle, row by row, then the state's tiles
template <typename T>
__global__ void __launch_bounds__(LA_THREADS)
    k_ls_chunk(const LaShape s, const __grid_constant__ LaChunkArgs<T> a, int score_tiles, int state_tiles)
{
    __shared__ alignas(16) T sm[4][32][LS_W<T>];
    const int per = score_tiles + state_tiles, nc = s.chunks();
    const int64_t r = blockIdx.x / per, bc = r / s.H, h = r - bc * s.H, b = bc / nc, bh = b * s.H + h;
    const int which = int(blockIdx.x - r * per), c = int(bc - b * nc), len = s.len(c);
    const int64_t row0 = (b * s.T + int64_t(c) * s.C) * a.ld, kd0 = int64_t(s.H) * s.dk;
    LsTile<T> t;
    LtPair<T> &p = t.p[0];
    t.pairs = 1;
    if (which < score_tiles) {
        int i = 0;
        while ((i + 1) * (i + 2) / 2 <= which) i++;
        t.i0 = 32 * i, t.j0 = 32 * (which - i * (i + 1) / 2);
        if (t.i0 >= len) return;
        const int64_t oq = row0 + h * s.dk, ok = oq + kd0;
        p.a = a.qkv + oq, p.a_ms = a.qkv_ms + oq, p.b = a.qkv + ok, p.b_ms = a.qkv_ms + ok;
        p.lda = p.ldb = a.ld, p.K = s.dk, t.rows = t.cols = len;
        t.at = bh * s.tri() + s.tri_at(c), t.stride = 0;
        ls_tile<T, LT_SCORES>(sm, t, a.p0, a.qkv_ms != nullptr, a.z, a.out);
    } else {
        const int across = (s.dv + 31) / 32, i = (which - score_tiles) / across;
        t.i0 = 32 * i, t.j0 = 32 * (which - score_tiles - i * across);
        const int64_t ok = (bh * s.T + int64_t(c) * s.C) * s.dk, ov = row0 + 2 * kd0 + h * s.dv;
        p.a = a.kd + ok, p.a_ms = a.kd_ms + ok, p.b = a.qkv + ov, p.b_ms = a.qkv_ms + ov;
        p.lda = s.dk, p.ldb = a.ld, p.K = len, t.rows = s.dk, t.cols = s.dv;
        t.at = s.n_scores() + (int64_t(c) * s.bh() + bh) * s.dk * s.dv, t.stride = s.dv;
        ls_tile<T, LT_STATES>(sm, t, a.p0, a.qkv_ms != nullptr, a.z, a.out);
    }
}

template <typename T>
__global__ void __launch_bounds__(LA_THREADS)
    k_ls_output(const LaShape s, const __grid_constant__ LaOutArgs<T> a, int down, int across)
{
    __shared__ alignas(16) T sm[4][32][LS_W<T>];
    const int per = down * across, nc = s.chunks();
    const int64_t r = blockIdx.x / per, bc = r / s.H, h = r - bc * s.H, b = bc / nc, bh = b * s.H + h;
    const int which = int(blockIdx.x - r * per), c = int(bc - b * nc), len = s.len(c);
    LsTile<T> t;
    LtPair<T> &p = t.p[0], &q = t.p[1];
    t.i0 = 32 * (which / across), t.j0 = 32 * (which % across);
    if (t.i0 >= len) return;
    const int64_t t0 = b * s.T + int64_t(c) * s.C, ov = t0 * a.ld + 2 * int64_t(s.H) * s.dk + h * s.dv;
    const int64_t op = bh * s.tri() + s.tri_at(c), oq = (bh * s.T + int64_t(c) * s.C) * s.dk;
    const int64_t os = (c ? s.n_scores() + int64_t(c - 1) * s.n_state() : 0) + bh * s.dk * s.dv;
    const T *const st = c ? a.ps : a.s0, *const st_ms = c ? a.ps_ms : a.s0_ms;
    p.a = a.ps + op, p.a_ms = a.ps_ms + op, p.b = a.qkv + ov, p.b_ms = a.qkv_ms + ov, p.lda = 0, p.ldb = a.ld, p.K = len;
    q.a = a.qd + oq, q.a_ms = a.qd_ms + oq, q.b = st + os, q.b_ms = st_ms + os, q.lda = s.dk, q.ldb = s.dv, q.K = s.dk;
    t.pairs = st ? 2 : 1, t.rows = len, t.cols = s.dv;
    t.at = (t0 * s.H + h) * s.dv, t.stride = int64_t(s.H) * s.dv;
    ls_tile<T, LT_OUTPUT>(sm, t, a.p0, a.qkv_ms != nullptr, a.z, a.out);
}

// ------------------------------------------------------------------ one token
//
// A block takes CX x V columns of one head's state, its 256 / CX thread rows
// stride over dk: S, its mask share and the dealer's word are read once and
// the new state written once (4 words moved and 5 multiply-adds per entry, so
// bound by memory); q . S comes out of the same pass, summed over the thread
// rows in shared memory.  Two rows ahead and four blocks an SM: 1024 heads x 128 x
// 128 in 50 us (5.3 TB/s), 512 x 64 x 128 over Z_2^64 in 31 us (4.3 TB/s: as many
// blocks with half the bytes each, so what a block does once, its first loads and the
// sum over its rows, weighs twice; barriers take 2 of 16 cycles an instruction there,
// 1.3 of 22 here); four rows and three blocks took 54 and 39, one wave of blocks that
// loop over heads 73 and 47.
template <typename T, int V>
__global__ void __launch_bounds__(LA_THREADS, 4)
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
    // a thread's next U rows, in flight while the present ones are worked on (the
    // first ones while q, k and v arrive)
    constexpr int U = 2;
    PV S[U], m[U], z[U];
    const int64_t at = bh * per + col;
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * ry;
            if (!on || i >= s.dk) continue;
            const int64_t o = at + int64_t(i) * s.dv;
            S[u] = *reinterpret_cast<const PV *>(a.s + o), z[u] = *reinterpret_cast<const PV *>(a.z + o);
            if (a.qkv_ms) m[u] = *reinterpret_cast<const PV *>(a.s_ms + o);
        }
    };
    fetch(y0);
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
    const T lam = a.lam * __ldg(a.pow + s.pow_at(uint32_t(h)) + 1);
    __syncthreads();
    for (int i0 = y0; i0 < s.dk; i0 += U * ry) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * ry;
            if (!on || i >= s.dk) continue;
            const T q = qs[i], key = ks[i], mq = rq[i], mk = rk[i];
            PV n;
#pragma unroll
            for (int k = 0; k < V; k++) {
                n.e[k] = z[u].e[k] + lam * S[u].e[k] + key * vr[k] - mk * v[k];
                acc[k] += q * (a.p0 * S[u].e[k] - (a.qkv_ms ? m[u].e[k] : T(0))) - mq * S[u].e[k];
            }
            *reinterpret_cast<PV *>(a.out + at + int64_t(i) * s.dv) = n;
        }
        fetch(i0 + U * ry);
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
        T right = a.p0 * a.qkv[ov], acc = a.lam * a.pow[s.pow_at(uint32_t(h)) + 1] * a.yw[e];
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
static int la_tile_ready(K kern, uint32_t smem, int (&configured)[64], uint32_t **err)
{
    int dev = 0;
    DDG_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        DDG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
        if (dev >= 0 && dev < 64) configured[dev] = 1;
    }
    return ring_gemm_err_word(err);
}

inline unsigned la_tile_grid(int64_t tiles) { return unsigned(tiles < 2 * 148 ? tiles : 2 * 148); }

// The CUDA cores while their 32 x 32 tiles (a short last chunk has fewer) take
// nine quarters of a round on the SMs for the chunk stage at 32 bits, one and a half for the
// output stage, one for either at 64.  For 4 / 16 / 32 heads x 128 tokens x 64, in us
// on CUDA cores against tensor cores: chunk stage 7.0 / 11.1 / 17.0 against 14.6 /
// 15.0 / 15.2, over Z_2^64 15.3 / 23.9 / 40.4 against 22.8 / 22.4 / 27.3; output stage
// 10.0 / 10.2 / 17.8 against 17.3 / 17.4 / 17.5 (24 heads: 16.5 and 17.3), over Z_2^64
// 22.9 / 23.1 / 41.6 against 23.2 / 23.2 / 23.4, and for 16 heads x 32 tokens there
// 13.0 against 13.9; 16 heads x 138 tokens x 47 (304 tiles) chunk stage 11.2 and 19.7.
// Tiles are counted without their K, so short prompts leave the CUDA cores early: the
// chunk stage of 32 heads x 8 tokens over Z_2^64 takes 15.5 where 11.6 is possible.
static bool ls_fits(const LaShape &s, int64_t tiles_full, int64_t tiles_last, int64_t most)
{
    return s.bh() * ((s.chunks() - 1) * tiles_full + tiles_last) <= most;
}

template <typename T>
int la_chunk(const LaShape &s, const LaChunkArgs<T> &a, cudaStream_t st)
{
    if (!s.n_ps()) return DDG_OK;
    const int rows = (s.len(0) + 31) / 32, tri = rows * (rows + 1) / 2;
    const int square = ((s.dk + 31) / 32) * ((s.dv + 31) / 32);
    const int last = (s.len(s.chunks() - 1) + 31) / 32;
    if (ls_fits(s, tri + square, last * (last + 1) / 2 + square, sizeof(T) == 4 ? 148 * 9 / 4 : 148)) {
        k_ls_chunk<T><<<unsigned(s.bh() * s.chunks() * (tri + square)), LA_THREADS, 0, st>>>(s, a, tri, square);
        return launched();
    }
    using S = LtShape<T>;
    static thread_local int configured[64];
    const int np = (s.len(0) + S::NT - 1) / S::NT, ns = (s.dv + S::NT - 1) / S::NT;
    uint32_t *err = nullptr;
    DDG_TRY(la_tile_ready(k_la_chunk<T>, S::SMEM, configured, &err));
    // two CTAs per SM, shared out by the two lists' K-steps (a tile's epilogue takes about as long as three)
    const int64_t chunks = s.bh() * s.chunks(), scores = chunks * np, states = chunks * ns;
    const int64_t grid = scores + states < 2 * 148 ? scores + states : 2 * 148;
    const double cs = double(scores) * (2 * steps32(s.dk) + 3), ct = double(states) * (2 * steps32(s.len(0)) + 3);
    int64_t mine = int64_t(double(grid) * cs / (cs + ct) + 0.5);
    mine = mine < 1 ? 1 : mine > grid - 1 ? grid - 1 : mine;
    k_la_chunk<T><<<unsigned(grid), LT_THREADS, S::SMEM, st>>>(s, a, np, ns, int(mine), err);
    return launched();
}

template <typename T, int V>
static int launch_carry(const LaShape &s, const T *pow, const T *ps, const T *s0, T *out, cudaStream_t st)
{
    const int64_t per = int64_t(s.dk) * s.dv, state_slices = la_blocks(per, V);
    const int64_t score_slices = (s.tri() + V + LC_SLICE * V - 1) / (LC_SLICE * V);
    DDG_CHECK(s.bh() * (state_slices + score_slices) <= 0x7fffffff, DDG_ERR_ARG,
              "linear attention: %lld score entries are too many for one call", (long long)s.n_scores());
    // the states first: theirs are the long dependent sums
    k_la_carry<T, V><<<unsigned(s.bh() * (state_slices + score_slices)), LA_THREADS, 0, st>>>(
        s, pow, ps, s0, out, int(state_slices), int(score_slices), s.bh() * state_slices);
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
    const int down = (s.len(0) + 31) / 32, across = (s.dv + 31) / 32;
    if (ls_fits(s, down * across, (s.len(s.chunks() - 1) + 31) / 32 * across, sizeof(T) == 4 ? 148 * 3 / 2 : 148)) {
        k_ls_output<T><<<unsigned(s.bh() * s.chunks() * down * across), LA_THREADS, 0, st>>>(s, a, down, across);
        return launched();
    }
    using S = LtShape<T>;
    static thread_local int configured[64];
    const int tiles = (s.dv + S::NT - 1) / S::NT;
    const int64_t count = s.bh() * s.chunks() * tiles;
    uint32_t *err = nullptr;
    DDG_TRY(la_tile_ready(k_la_output<T>, S::SMEM, configured, &err));
    k_la_output<T><<<la_tile_grid(count), LT_THREADS, S::SMEM, st>>>(s, a, count, tiles, err);
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
