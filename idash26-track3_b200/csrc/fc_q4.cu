// Fully connected layers with 4-bit public weights and group steps:
//
//   out[m][n] = sign * sum_k x[m][k] W[k][n] + bias[n] + Add[m][n]   modulo 2^bw
//   W[k][n]   = step[k / group][n] * (code(n, k) - 8)
//
// Two kernels, both exact modulo 2^bw, so the result does not depend on how K
// is split over lanes, warps or CTAs.
//
// k_q4_gemv, for one row or two of a smaller product: 8-bit limb products on the CUDA cores.  x
// sits in shared memory as byte planes, four k of one limb to a word, and
// dp4a multiplies a word by four codes: per unit of 32 codes (one 16-byte
// load, one step)
//   sum_k x_k W_k = step * ( sum_l 2^(8l) dp4a(code, limb l of x) - 8 sum_k x_k ).
//
// k_q4_tc, for everything else: the weights are 16-bit numbers, W + 2^15 = w0 + 2^8 w1
// with unsigned bytes, and x = sum_l 2^(8l) x_l, so
//   x . W = sum_s 2^(8s) sum_k (w0 x_s + w1 x_{s-1})  -  2^15 sum_k x_k .
// The weights are the M side of the MMA (128 outputs) as they are, two bytes a
// weight; the N side has a row (x_s, x_{s-1}) per k for every limb s of MT rows
// of x (limb-major, P * MT columns).  So a weight costs one multiply-add for
// two of them and no byte shuffles, one MMA of 32 bytes covers 16 k of every
// limb, and the whole product takes 2 P byte products where full-width ring
// weights take P(P+1)/2.  One warp loads codes and x with TMA, one issues the
// MMAs, the others expand codes and split x.  The sums of a split K meet in the
// cluster's shared memory.
//
// Measured on one B200 (graph replays, launch included, weights from memory).
// CUDA cores: 1 x 376 x 1024 4.0 us, 1 x 4096 x 4096 9.3 us and 1 x 4096 x 8192
// 13.0 us (1.3 TB/s of codes), 7.7 and 10.7 with the weights in L2; over Z_2^64
// 1 x 4096 x 4096 12.7.  Bound by latency: a scheduler issues in 0.34 to 0.38 of
// its cycles, 21 % of the warps are there, and a warp waits 2.8 of its 9 cycles an
// instruction for memory, 0.7 to 1.1 at barriers, 1 for shared memory; each is
// one chain of the split of x and its segments, with one segment in flight.
// Tensor cores: 256 x 1024 x 512 7.1 us; 16 x 4096 x 8192 18.0 us (16.8 MB of
// codes, 0.9 TB/s; 14.5 in L2), bound by the hand-off of a stage from copy to
// expansion to MMA in one CTA an SM (issue 0.40, tensor pipe 13 %, 4.1 of 11
// cycles an instruction waiting for memory or tensor memory); 2048 x 4096 x 4096
// 229 us (0.30 P ring flop/s, 1.2 P byte products/s: tensor pipe 62 % busy, bound
// by shared memory), over Z_2^64 468 us.
#include <type_traits>

#include "tma.cuh"
#include "token.cuh"

namespace ddg {

namespace {

// ------------------------------------------------------------------ one or two rows

template <typename T>
constexpr int GV_R = gv_outputs(int(sizeof(T)));

template <typename T, int MR>
__global__ void __launch_bounds__(Q4_THREADS, 2)
    k_q4_gemv(const __grid_constant__ Q4Args<T> a, const __grid_constant__ GvGeom g, int64_t row_bytes, int vec)
{
    constexpr int P = int(sizeof(T)), R = GV_R<T>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint4 *const xs = reinterpret_cast<uint4 *>(smem_raw);                   // [MR][2P][U]
    T *const xsum8 = reinterpret_cast<T *>(xs + size_t(MR) * 2 * P * g.U);  // [MR][U]: 8 * sum of the unit's x
    T *const red = xsum8 + MR * g.U;                                        // [warp][lane group][R][MR]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int li = lane & (g.L - 1), grp = lane / g.L, ngrp = 32 / g.L;
    const int ks = warp % g.KS, ws = warp / g.KS;
    const bool active = ws < GV_WARPS / g.KS;
    const int slot = ws * ngrp + grp;

    struct Codes {
        uint4 c[R];
        uint32_t s[R];
    };
    auto fetch = [&](int blk, int seg, Codes &f) {
        const int u = seg * g.L + li;
        const int64_t n0 = (int64_t(blk) * g.slots + slot) * R;
#pragma unroll
        for (int r = 0; r < R; r++) {
            f.c[r] = make_uint4(0, 0, 0, 0), f.s[r] = 0;
            if (active && blk < g.blocks && seg < g.nseg && u < g.U && n0 + r < a.w.N) {
                f.c[r] = __ldg(reinterpret_cast<const uint4 *>(a.w.q + (n0 + r) * row_bytes) + u);
                f.s[r] = __ldg(a.w.step + int64_t(u * 32 / a.w.group) * a.w.N + n0 + r) & Q4_STEP_MAX;
            }
        }
    };

    // the first codes are in flight while x is split, then those of the next segment (two ahead took no less time)
    Codes cur, next;
    int fblk = blockIdx.x, fseg = ks;  // the next segment to fetch
    auto fetch_next = [&](Codes &f) {
        fetch(fblk, fseg, f);
        fseg += g.KS;
        if (fseg >= g.nseg) fseg = ks, fblk += gridDim.x;
    };
    fetch_next(cur);
    const int quarters = MR * g.U * 4;
    for (int i0 = warp * 32; i0 < quarters; i0 += Q4_THREADS) {  // warp-uniform: the shuffles below are whole
        const bool in = i0 + lane < quarters;
        const int i = in ? i0 + lane : 0;
        const int m = i / (g.U * 4), u = (i >> 2) % g.U, j = i & 3;
        T e[8], sum = 0;
        const int k0 = u * 32 + j * 8;
        const T *const xp = a.x + int64_t(m) * a.ldx + k0;
        if (in && vec && k0 + 8 <= a.w.K) {
#pragma unroll
            for (int t = 0; t < P / 2; t++)
                *reinterpret_cast<uint4 *>(e + t * (16 / P)) = __ldg(reinterpret_cast<const uint4 *>(xp) + t);
        } else {
#pragma unroll
            for (int t = 0; t < 8; t++) e[t] = in && k0 + t < a.w.K ? __ldg(xp + t) : T(0);
        }
#pragma unroll
        for (int t = 0; t < 8; t++) sum += e[t];
        if (in) {
#pragma unroll
            for (int par = 0; par < 2; par++) {
                uint32_t p[4];
                byte_planes(uint32_t(e[par]), uint32_t(e[par + 2]), uint32_t(e[par + 4]), uint32_t(e[par + 6]), p);
                const int q = (j * 2 + par) * (P / 4);
                xs[(size_t(m) * 2 * P + q) * g.U + u] = make_uint4(p[0], p[1], p[2], p[3]);
                if constexpr (P == 8) {
                    byte_planes(uint32_t(uint64_t(e[par]) >> 32), uint32_t(uint64_t(e[par + 2]) >> 32),
                                uint32_t(uint64_t(e[par + 4]) >> 32), uint32_t(uint64_t(e[par + 6]) >> 32), p);
                    xs[(size_t(m) * 2 * P + q + 1) * g.U + u] = make_uint4(p[0], p[1], p[2], p[3]);
                }
            }
        }
        // the four quarters of a unit sit in four neighbouring lanes
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (in && j == 0) xsum8[m * g.U + u] = sum * T(8);
    }
    __syncthreads();

    for (int blk = blockIdx.x; blk < g.blocks; blk += gridDim.x) {
        T acc[R][MR];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int m = 0; m < MR; m++) acc[r][m] = 0;
        for (int seg = ks; seg < g.nseg; seg += g.KS) {
            fetch_next(next);
            const int u = seg * g.L + li;
            if (active && u < g.U) {
#pragma unroll
                for (int m = 0; m < MR; m++) {
                    uint32_t part[R][P];
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int l = 0; l < P; l++) part[r][l] = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int par = 0; par < 2; par++) {
                            uint32_t xw[P];
#pragma unroll
                            for (int w = 0; w < P / 4; w++) {
                                const uint4 v = xs[(size_t(m) * 2 * P + (j * 2 + par) * (P / 4) + w) * g.U + u];
                                xw[4 * w] = v.x, xw[4 * w + 1] = v.y, xw[4 * w + 2] = v.z, xw[4 * w + 3] = v.w;
                            }
#pragma unroll
                            for (int r = 0; r < R; r++) {
                                const uint32_t c4 = j == 0 ? cur.c[r].x : j == 1 ? cur.c[r].y : j == 2 ? cur.c[r].z : cur.c[r].w;
                                const uint32_t code = (c4 >> (4 * par)) & 0x0f0f0f0fu;
#pragma unroll
                                for (int l = 0; l < P; l++) part[r][l] = __dp4a(code, xw[l], part[r][l]);
                            }
                        }
                    const T off = xsum8[m * g.U + u];
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        T v = T(0) - off;
#pragma unroll
                        for (int l = 0; l < P; l++) v += T(part[r][l]) << (8 * l);
                        acc[r][m] += v * T(cur.s[r]);
                    }
                }
            }
            cur = next;
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int m = 0; m < MR; m++) {
                for (int o = 1; o < g.L; o <<= 1) acc[r][m] += __shfl_xor_sync(0xffffffffu, acc[r][m], o);
                if (li == 0) red[((warp * ngrp + grp) * R + r) * MR + m] = acc[r][m];
            }
        __syncthreads();
        for (int i = tid; i < g.slots * R * MR; i += Q4_THREADS) {
            const int m = i % MR, row = i / MR, sl = row / R, r = row % R;
            const int64_t n = int64_t(blk) * g.slots * R + row;
            if (n >= a.w.N) continue;
            T v = 0;
            for (int k = 0; k < g.KS; k++)
                v += red[(((sl / ngrp * g.KS + k) * ngrp + sl % ngrp) * R + r) * MR + m];
            v *= a.sign;
            if (a.bias) v += __ldg(a.bias + n);
            const int64_t e = int64_t(m) * a.w.N + n;
            if (a.Add) v += a.Add[e];
            a.out[e] = v;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ more rows: tensor cores

// operands lie in 16-byte chunks of 8 k, chunk-major: rows 16 bytes apart,
// chunks of A 2048 and of B 16 NB + 16 bytes apart (the pad spreads the chunks
// of one row, written by neighbouring lanes, over the banks)
constexpr uint32_t QT_A_CHUNK = TC_BM * 16;

// MT rows of x per CTA and NA 128-output weight tiles, which share the split of x
template <typename T, int MT, int NA>
struct QtShape {
    static constexpr int P = int(sizeof(T));
    static constexpr int NB = P * MT;                              // MMA columns
    // k per stage: narrower MMAs are issue-bound (a commit takes as long as five
    // of them), so they get twice the K per commit
    static constexpr int KC = NB <= 128 ? 128 : 64;
    static constexpr int BOXES = KC / 64;                          // 32-byte boxes of codes per row and stage
    // sixteen warps to expand; a unit of codes for each thread of the first UNITS
    static constexpr int THREADS = 512, UNITS = NA * BOXES * 256;
    static constexpr int NST = NB <= 64 ? 3 : 2;                   // stages of planes
    static constexpr int CH = KC / 8, XROW = KC / 8;               // chunks per stage; x items of 8 k per row
    // one weight tile goes straight to tensor memory (KC / 2 columns a stage), which
    // spares the shared memory half of its traffic; beside two tiles' 512
    // accumulator columns there is no room for it
    static constexpr bool A_TMEM = NA == 1;
    static constexpr int A_COLS = A_TMEM ? KC / 2 : 0, COLS = tmem_cols(NA * NB + NST * A_COLS);
    static constexpr uint32_t B_CHUNK = NB * 16 + 16;
    static constexpr uint32_t A_TILE = CH * QT_A_CHUNK, A_STAGE = A_TMEM ? 0 : NA * A_TILE, STAGE = A_STAGE + CH * B_CHUNK;
    static constexpr int ITEMS = MT * XROW, XPT = (ITEMS + THREADS - 1) / THREADS;
    // A stage's codes (BOXES of 32 bytes a row) and x as they lie in
    // memory, loaded RD stages ahead: the memory needs about 40 KB of codes in
    // flight per SM for its latency.  (Asynchronous 16-byte copies by the
    // expanding threads took 600-1000 cycles a stage to issue.)
    static constexpr uint32_t RAW_BOX = NA * TC_BM * 32, RAW_X = BOXES * RAW_BOX, RAW = RAW_X + MT * KC * P;
    static constexpr int RD_FIT = int((212 * 1024 - NST * STAGE) / RAW);
    static constexpr int RD = RD_FIT < 2 ? 2 : RD_FIT > 8 ? 8 : RD_FIT;
    // [barriers, TMEM address | sums of x | pad to 1024 | stages | raw stages | slack]
    static constexpr uint32_t HEAD = 256 + MT * P;
    static constexpr uint32_t XPITCH = (ITEMS < THREADS ? ITEMS : THREADS) * 16;  // between 16-byte pieces of the x items
    static constexpr uint32_t SMEM = HEAD + 1024 + NST * STAGE + RD * RAW + 2048;
    static_assert(NB % 16 == 0 && NB <= 256 && STAGE % 128 == 0 && RAW % 128 == 0 && RAW_X % 128 == 0, "tile");
    static_assert(UNITS <= THREADS && THREADS % XROW == 0 && (ITEMS % THREADS == 0 || XPT == 1), "x items");
};

// (.aligned: the lanes of a warp arrive together, whatever branches they come from)
__device__ __forceinline__ void cluster_sync()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ T ld_cluster(const T *p, uint32_t rank)
{
    uint32_t addr;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_addr(p)), "r"(rank));
    if constexpr (sizeof(T) == 4) {
        uint32_t v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
        return v;
    } else {
        uint64_t v;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
        return v;
    }
}

// 8 codes times a step, plus 2^15, as 16-bit weights in the order k = 0 4 1 5 2 6 3 7
__device__ __forceinline__ uint4 q4_expand(uint32_t c, uint32_t s, uint32_t bias)
{
    // codes k and k + 4 in the two halves of a word: one multiply-add makes both weights (no carry
    // between the halves: 0 <= s * code + 2^15 - 8 s < 2^16 for s <= 4095)
    return make_uint4((c & 0x000f000fu) * s + bias, ((c >> 4) & 0x000f000fu) * s + bias,
                      ((c >> 8) & 0x000f000fu) * s + bias, ((c >> 12) & 0x000f000fu) * s + bias);
}

// bytes (s, s - 1) of a, then of b
__device__ __forceinline__ uint32_t byte_pair(uint32_t a, uint32_t b, int s)
{
    return s == 0 ? __byte_perm(a, b, 0x0400) & 0x00ff00ffu
                  : __byte_perm(a, b, uint32_t(s | (s - 1) << 4 | (s + 4) << 8 | (s + 3) << 12));
}

template <typename T, int MT, int NA>
__global__ void __launch_bounds__(QtShape<T, MT, NA>::THREADS + 64, 1)
    k_q4_tc(const __grid_constant__ Q4Args<T> a, const __grid_constant__ CUtensorMap codes_map,
            const __grid_constant__ CUtensorMap x_map, int per, int vec, uint32_t group_magic, uint32_t *err)
{
    using S = QtShape<T, MT, NA>;
    constexpr int P = S::P, THREADS = S::THREADS, KC = S::KC, WARPS = THREADS / 32, NST = S::NST;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint64_t *const empty = reinterpret_cast<uint64_t *>(smem_raw), *const full = empty + NST;
    uint64_t *const raw_full = full + NST, *const raw_empty = raw_full + 8;  // (3 + 3 + 8 + 8) x 8 bytes
    uint32_t &s_tmem = *reinterpret_cast<uint32_t *>(smem_raw + 192);
    T *const xsum = reinterpret_cast<T *>(smem_raw + 256);  // [MT]
    uint8_t *const smem = smem_raw + S::HEAD + ((1024u - ((smem_addr(smem_raw) + S::HEAD) & 1023u)) & 1023u);

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const bool mma_warp = warp == WARPS, tma_warp = warp == WARPS + 1, expands = warp < WARPS;
    const int half = expands && NA == 2 ? warp >> 3 : 0;  // this thread's weight tile
    const int n0 = (blockIdx.x * NA + half) * TC_BM, m0 = blockIdx.y * MT;
    const int nkc = (a.w.K + KC - 1) / KC, c0 = blockIdx.z * per;
    const int nk = nkc - c0 < per ? (nkc - c0 > 0 ? nkc - c0 : 0) : per;

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                     "r"(S::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < NST; i++) mbar_init(empty + i, 1), mbar_init(full + i, WARPS);
        for (int i = 0; i < S::RD; i++) mbar_init(raw_full + i, 1), mbar_init(raw_empty + i, WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < MT) xsum[tid] = 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    // this thread's unit of codes (row, 32 k) and items of x (row, 8 k each) of every stage
    // (in tensor memory a warp reaches the rows of its quarter only)
    const int arow = S::A_TMEM ? 32 * (warp & 3) + lane : 16 * (warp & 7) + (lane & 15);
    const int aun = S::A_TMEM ? warp >> 2 : lane >> 4;
    const int xk = tid % S::XROW * 8, xm = tid / S::XROW;
    const bool has_x = expands && tid < S::ITEMS, has_codes = expands && tid < S::UNITS;
    const int units = (a.w.K + 31) / 32;
    T sum[S::XPT];
#pragma unroll
    for (int i = 0; i < S::XPT; i++) sum[i] = 0;
    uint8_t *const raw = smem + NST * S::STAGE;
    const uint32_t raw_x = smem_addr(raw) + S::RAW_X + 16 * tid;
    // step of this thread's unit of stage c: unit u's is u / (group / 32), by the exact reciprocal (u < 2^13)
    const bool step_row = has_codes && n0 + arow < a.w.N;
    const uint16_t *const step_col = a.w.step + n0 + arow;
    auto step_of = [&](int c) -> uint32_t {
        const int u = KC / 32 * c + aun;
        const uint32_t g = group_magic ? __umulhi(uint32_t(u), group_magic) : uint32_t(u);
        return step_row && u < units ? __ldg(step_col + int64_t(g) * a.w.N) : 0;
    };
    // x of stage c into raw stage r where its rows are not on 16-byte boundaries; what lies outside the matrix
    // arrives as zeros
    auto issue = [&](int c, int r) {
        const uint32_t ro = uint32_t(r) * S::RAW;
        if (has_x && !vec) {
#pragma unroll
            for (int j = 0; j < S::XPT; j++) {
                const int m = xm + j * (THREADS / S::XROW), k = c * KC + xk;
                const T *const xp = a.x + int64_t(m0 + m) * a.ldx + k;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const bool in = m0 + m < a.M && k + i < a.w.K;
                    cp_async<P>(raw_x + ro + j * THREADS * 8 * P + i / (16 / P) * S::XPITCH + i % (16 / P) * P,
                                in ? xp + i : a.x, in ? P : 0);
                }
            }
        }
        cp_async_commit();
    };
    // expands raw stage r into the planes of stage st
    auto store_stage = [&](int r, int st, uint32_t step) {
        uint8_t *const base = smem + st * S::STAGE;
        const uint8_t *const rp = raw + uint32_t(r) * S::RAW;
        if (has_codes) {
            const uint4 code = *reinterpret_cast<const uint4 *>(rp + (aun >> 1) * S::RAW_BOX + (half * TC_BM + arow) * 32 +
                                                                (aun & 1) * 16);
            step &= Q4_STEP_MAX;
            const uint32_t bias = (0x8000u - 8u * step) * 0x10001u;
            const uint4 w[4] = {q4_expand(code.x, step, bias), q4_expand(code.y, step, bias), q4_expand(code.z, step, bias),
                                q4_expand(code.w, step, bias)};
            if constexpr (S::A_TMEM) {
                const uint32_t v[16] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w,
                                        w[2].x, w[2].y, w[2].z, w[2].w, w[3].x, w[3].y, w[3].z, w[3].w};
                tc_fence_after();  // the MMAs that read this stage are done
                tmem_st16(tmem + (uint32_t(32 * (warp & 3)) << 16) + NA * S::NB + st * S::A_COLS + aun * 16, v);
            } else {
                uint8_t *const pa = base + half * S::A_TILE + aun * 4 * QT_A_CHUNK + arow * 16;
#pragma unroll
                for (int i = 0; i < 4; i++) *reinterpret_cast<uint4 *>(pa + i * QT_A_CHUNK) = w[i];
            }
        }
        if (has_x) {
#pragma unroll
            for (int j = 0; j < S::XPT; j++) {
                T xe[8];
#pragma unroll
                for (int i = 0; i < P / 2; i++)
                    *reinterpret_cast<uint4 *>(xe + i * (16 / P)) = *reinterpret_cast<const uint4 *>(
                        rp + S::RAW_X +
                        (vec ? uint32_t((xm + j * (THREADS / S::XROW)) * KC + xk) * P + i * 16
                             : j * THREADS * 8 * P + i * S::XPITCH + tid * 16));
#pragma unroll
                for (int i = 0; i < 8; i++) sum[j] += xe[i];
                uint8_t *const pb = base + S::A_STAGE + (xk >> 3) * S::B_CHUNK + (xm + j * (THREADS / S::XROW)) * 16;
#pragma unroll
                for (int l = 0; l < P; l++) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t lo0 = uint32_t(xe[i]), lo1 = uint32_t(xe[i + 4]);
                        if constexpr (P == 4) {
                            w[i] = byte_pair(lo0, lo1, l);
                        } else {
                            const uint32_t hi0 = uint32_t(uint64_t(xe[i]) >> 32), hi1 = uint32_t(uint64_t(xe[i + 4]) >> 32);
                            if (l < 4)
                                w[i] = byte_pair(lo0, lo1, l);
                            else if (l < 7)  // bytes 3..6 of x
                                w[i] = byte_pair(__funnelshift_l(lo0, hi0, 8), __funnelshift_l(lo1, hi1, 8), l - 3);
                            else
                                w[i] = byte_pair(hi0, hi1, 3);
                        }
                    }
                    *reinterpret_cast<uint4 *>(pb + l * MT * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    };

    // this thread's outputs, and the first ones' Add and bias on their way while the products are formed
    constexpr int PITCH = NA * TC_BM, ROWS = THREADS / PITCH;                    // outputs per row of x, rows per pass
    constexpr int U = MT / ROWS < 1 ? 1 : MT / ROWS < 8 ? MT / ROWS : 8;         // passes per batch
    const int parts = int(gridDim.z), pitch_m = ROWS * parts;
    const int ol = tid % PITCH, on = blockIdx.x * PITCH + ol, om = int(blockIdx.z) * ROWS + tid / PITCH;
    T add[U], bias = 0;
    auto load_add = [&](int mb) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int m = mb + i * pitch_m;
            add[i] = a.Add && on < a.w.N && m < MT && m0 + m < a.M ? a.Add[int64_t(m0 + m) * a.w.N + on] : T(0);
        }
    };
    if (expands) {
        load_add(om);
        if (a.bias && on < a.w.N) bias = __ldg(a.bias + on);
    }

    constexpr uint32_t IDESC = i8_idesc(S::NB, false);
    bool ok = true;
    if (mma_warp) {
        const bool leader = elect_one();
        for (int c = 0; c < nk && ok; c++) {
            const int st = c % NST;
            ok = mbar_wait(&full[st], uint32_t((c / NST) & 1));
            tc_fence_after();
            if (ok && leader) {
                // descriptors step by constants in their address field (16-byte units)
                const uint32_t sa = smem_addr(smem + st * S::STAGE), sb = sa + S::A_STAGE;
                const uint64_t db = smem_desc(sb, S::B_CHUNK, 128), da = smem_desc(sa, QT_A_CHUNK, 128);
                const uint32_t ta = tmem + S::NB + st * S::A_COLS;
#pragma unroll
                for (int h = 0; h < KC / 16; h++) {
#pragma unroll
                    for (int t = 0; t < NA; t++) {
                        const uint64_t dbh = db + uint64_t(h * 2 * S::B_CHUNK >> 4);
                        if constexpr (S::A_TMEM)
                            mma_i8_ts(tmem, ta + h * 8, dbh, IDESC, (c > 0 || h > 0) ? 1u : 0u);
                        else
                            mma_i8(tmem + t * S::NB, da + uint64_t((t * S::A_TILE + h * 2 * QT_A_CHUNK) >> 4), dbh, IDESC,
                                   (c > 0 || h > 0) ? 1u : 0u);
                    }
                }
                mma_commit(&empty[st]);
            }
            __syncwarp();
        }
    } else if (tma_warp) {
        const bool leader = elect_one();
        if (leader) {
            tma_prefetch(&codes_map);
            if (vec) tma_prefetch(&x_map);
        }
        for (int c = 0, r = 0; c < nk && ok; c++, r = r + 1 == S::RD ? 0 : r + 1) {
            // (not the full barriers: between two uses of a raw stage they can pass two phases, and a parity
            // tells only neighbouring ones apart)
            if (c >= S::RD) ok = mbar_wait(&raw_empty[r], uint32_t((c / S::RD - 1) & 1));
            if (ok && leader) {
                const uint32_t ra = smem_addr(raw) + uint32_t(r) * S::RAW;
                mbar_expect(&raw_full[r], S::BOXES * S::RAW_BOX + (vec ? MT * KC * P : 0));
#pragma unroll
                for (int i = 0; i < S::BOXES; i++)
                    tma_load_2d(ra + i * S::RAW_BOX, &codes_map, (c0 + c) * (KC / 2) + 32 * i, n0, &raw_full[r]);
                if (vec) tma_load_2d(ra + S::RAW_X, &x_map, (c0 + c) * KC, m0, &raw_full[r]);
            }
            __syncwarp();
        }
        // nobody leaves with copies in flight
        if (ok && nk > 0) ok = mbar_wait(&raw_full[(nk - 1) % S::RD], uint32_t(((nk - 1) / S::RD) & 1));
    } else {
        if (!vec)
            for (int c = 0; c < S::RD; c++) {
                if (c < nk)
                    issue(c0 + c, c);
                else
                    cp_async_commit();
            }
        uint32_t step = nk > 0 ? step_of(c0) : 0;
        for (int c = 0, r = 0; c < nk; c++, r = r + 1 == S::RD ? 0 : r + 1) {
            const int st = c % NST;
            if (!vec) cp_async_wait<S::RD - 1>();  // this thread's copies of stage c have landed
            ok = mbar_wait(&raw_full[r], uint32_t((c / S::RD) & 1));
            if (ok && c >= NST) ok = mbar_wait(&empty[st], uint32_t((c / NST - 1) & 1));
            if (!__all_sync(0xffffffffu, ok)) break;
            store_stage(r, st, step);
            if (c + 1 < nk) step = step_of(c0 + c + 1);
            if (!vec) {
                if (c + S::RD < nk)
                    issue(c0 + c + S::RD, r);
                else
                    cp_async_commit();
            }
            proxy_fence();
            if constexpr (S::A_TMEM) {
                __syncwarp();  // the wait is .aligned, and the lanes' loads of steps and x are their own
                tmem_st_wait();
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[st]), mbar_arrive(&raw_empty[r]);
        }
        cp_async_wait<0>();
    }
    // the last stage's commit covers every MMA before it
    if (ok && nk > 0) ok = mbar_wait(&empty[(nk - 1) % NST], uint32_t(((nk - 1) / NST) & 1));
    if (has_x) {
        using U = std::conditional_t<P == 4, unsigned int, unsigned long long>;
#pragma unroll
        for (int j = 0; j < S::XPT; j++) atomicAdd(reinterpret_cast<U *>(xsum + xm + j * (THREADS / S::XROW)), U(sum[j]));
    }
    const int all_ok = __syncthreads_and(ok ? 1 : 0);
    tc_fence_after();

    // this CTA's sums of (row m, output n) to shared memory (the stages are done), all of them added up
    // over the cluster and written in batches whose loads overlap
    T *const part = reinterpret_cast<T *>(smem);  // [MT][PITCH]
    if (all_ok && expands) {
        constexpr int CW = MT < 8 ? MT : 8, GROUPS = WARPS / (4 * NA);  // rows of x per pass; warps per TMEM quarter
        const int q = warp & 3, h = (warp >> 2) % GROUPS, nl = half * TC_BM + 32 * q + lane;
        const uint32_t lanes = tmem + half * S::NB + (uint32_t(32 * q) << 16);
        {
#pragma unroll 1
            for (int m = h * CW; m < MT; m += GROUPS * CW) {
                uint32_t v[P][8];
                if constexpr (MT >= 8) {
#pragma unroll
                    for (int s = 0; s < P; s++) tmem_ld8(lanes + s * MT + m, v[s]);
                } else {
                    // MT = 4 or 2: eight columns hold 8 / MT limbs
                    uint32_t t[S::NB / 8][8];
#pragma unroll
                    for (int i = 0; i < S::NB / 8; i++) tmem_ld8(lanes + 8 * i, t[i]);
                    tmem_ld_wait();
#pragma unroll
                    for (int s = 0; s < P; s++)
#pragma unroll
                        for (int e = 0; e < CW; e++) v[s][e] = t[(s * MT + e) / 8][(s * MT + e) % 8];
                }
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < CW; e++) {
                    T r = T(0) - (xsum[m + e] << 15);
#pragma unroll
                    for (int s = 0; s < P; s++) r += T(v[s][e]) << (8 * s);
                    part[(m + e) * PITCH + nl] = nk > 0 ? r : T(0);  // a split's last CTA may have no stage
                }
            }
        }
    }
    if (!all_ok && tid == 0) atomicOr(err, 4u);
    tc_fence_before();
    const bool split = gridDim.z > 1;
    if (split)
        cluster_sync();
    else
        __syncthreads();
    if (expands && all_ok && on < a.w.N) {
        for (int mb = om; mb < MT; mb += U * pitch_m) {
            T v[U];
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int m = mb + i * pitch_m;
                v[i] = !split && m < MT ? part[m * PITCH + ol] : T(0);
            }
            if (split)
                for (int z = 0; z < parts; z++)
#pragma unroll
                    for (int i = 0; i < U; i++) {
                        const int m = mb + i * pitch_m;
                        if (m < MT) v[i] += ld_cluster(part + m * PITCH + ol, z);
                    }
#pragma unroll
            for (int i = 0; i < U; i++) v[i] = a.sign * v[i] + bias + add[i];
            load_add(mb + U * pitch_m);
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int m = mb + i * pitch_m;
                if (m < MT && m0 + m < a.M) a.out[int64_t(m0 + m) * a.w.N + on] = v[i];
            }
        }
    }
    if (split) cluster_sync();  // nobody leaves while its sums are read
    __syncwarp();               // lanes without an output of theirs are here first
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
    }
}

// an empty sum: out = bias + Add
template <typename T>
__global__ void __launch_bounds__(Q4_THREADS) k_q4_empty(const __grid_constant__ Q4Args<T> a)
{
    const int64_t n = int64_t(a.M) * a.w.N;
    for (int64_t e = int64_t(blockIdx.x) * Q4_THREADS + threadIdx.x; e < n; e += int64_t(gridDim.x) * Q4_THREADS)
        a.out[e] = (a.bias ? a.bias[e % a.w.N] : T(0)) + (a.Add ? a.Add[e] : T(0));
}

// one group of one output per thread: the smallest step whose codes -7..7
// reach the group's largest weight (at most 4095, beyond which codes saturate),
// codes rounded to nearest
__global__ void __launch_bounds__(256)
    k_q4_quantize(int64_t K, int64_t N, int64_t group, const int64_t *w, uint8_t *q, uint16_t *step, int64_t row_bytes)
{
    // K and group go up to the largest int, and their sum beyond it
    const int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t ng = (K + group - 1) / group;
    if (e >= ng * N) return;
    const int64_t n = e % N, k0 = e / N * group, k1 = K - k0 < group ? K : k0 + group;
    auto mag = [](int64_t v) { return v < 0 ? uint64_t(0) - uint64_t(v) : uint64_t(v); };
    uint64_t top = 0;
    for (int64_t k = k0; k < k1; k++) {
        const uint64_t a = mag(w[k * N + n]);
        top = a > top ? a : top;
    }
    const uint64_t fit = top / 7 + (top % 7 ? 1 : 0);
    const uint64_t s = fit < 1 ? 1 : fit > uint64_t(Q4_STEP_MAX) ? uint64_t(Q4_STEP_MAX) : fit;
    step[e] = uint16_t(s);
    const int64_t kend = k1 == K ? 2 * row_bytes : k1;  // the row's padding holds zero weights
    for (int64_t k = k0; k < kend; k += 2) {
        uint32_t byte = 0;
        for (int i = 0; i < 2; i++) {
            uint32_t code = 8;
            if (k + i < K) {
                const int64_t v = w[(k + i) * N + n];
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

template <typename K>
static int q4_smem_limit(K kern, uint64_t bytes, int (&configured)[64])
{
    int dev = 0;
    DDG_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || configured[dev] < int(bytes)) {
        DDG_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
        if (dev >= 0 && dev < 64) configured[dev] = int(bytes);
    }
    return DDG_OK;
}

// 16-byte loads of x: its rows start on 16-byte boundaries
template <typename T>
static int q4_vec(const Q4Args<T> &a)
{
    return (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && a.ldx * int64_t(sizeof(T)) % 16 == 0;
}

template <typename T, int MR>
static int launch_gemv(const Q4Args<T> &a, cudaStream_t st)
{
    static thread_local int configured[64];
    auto kern = k_q4_gemv<T, MR>;
    const GvGeom g = gv_geom(a.w.K, a.w.N, GV_R<T>);
    DDG_TRY(q4_smem_limit(kern, GV_SMEM_MAX, configured));
    // two CTAs an SM, each splitting x once for all its outputs
    const int grid = g.blocks < 2 * 148 ? g.blocks : 2 * 148;
    kern<<<grid, Q4_THREADS, gv_smem(g, MR, int(sizeof(T))), st>>>(a, g, int64_t(q4_row_bytes(a.w.K)), q4_vec(a));
    note_launch();
    DDG_CUDA(cudaGetLastError());
    return DDG_OK;
}

template <typename T, int MT, int NA>
static int launch_tc_q4(const Q4Args<T> &a, int split, cudaStream_t st)
{
    using S = QtShape<T, MT, NA>;
    static thread_local int configured[64];
    auto kern = k_q4_tc<T, MT, NA>;
    DDG_TRY(q4_smem_limit(kern, S::SMEM, configured));
    uint32_t *err = nullptr;
    DDG_TRY(ring_gemm_err_word(&err));
    const int nkc = (a.w.K + S::KC - 1) / S::KC;
    const int64_t gn = (int64_t(a.w.N) + NA * TC_BM - 1) / (NA * TC_BM), gm = (int64_t(a.M) + MT - 1) / MT;
    const int per = (nkc + split - 1) / split;
    const int vec = q4_vec(a);
    const uint32_t gd = uint32_t(a.w.group / 32);
    const uint32_t magic = gd == 1 ? 0 : uint32_t((uint64_t(1) << 32) / gd + 1);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(gn), unsigned(gm), unsigned(split));
    cfg.blockDim = dim3(S::THREADS + 64);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = unsigned(split);
    cfg.attrs = at, cfg.numAttrs = 1;
    const uint64_t row_bytes = q4_row_bytes(a.w.K);
    CUtensorMap codes_map, x_map = {};
    DDG_TRY(tma_map_2d(&codes_map, a.w.q, 1, row_bytes, a.w.N, row_bytes, 32, NA * TC_BM));
    if (vec) DDG_TRY(tma_map_2d(&x_map, a.x, sizeof(T), a.w.K, a.M, a.ldx * sizeof(T), S::KC, MT));
    DDG_CUDA(cudaLaunchKernelEx(&cfg, kern, a, codes_map, x_map, per, vec, magic, err));
    note_launch();
    return DDG_OK;
}

template <typename T>
int fc_q4(const Q4Args<T> &args, cudaStream_t st)
{
    Q4Args<T> a = args;
    if (int64_t(a.M) * a.w.N == 0) return DDG_OK;
    // a single row's stride is not used: any value goes, also one that no tensor map takes
    constexpr int V = 16 / int(sizeof(T));
    if (a.M == 1) a.ldx = (a.w.K + V - 1) / V * V;
    const Q4Plan plan = q4_plan(int(sizeof(T)), a.M, a.w.K, a.w.N);
    if (plan.kernel == Q4_EMPTY) {
        k_q4_empty<T><<<148, Q4_THREADS, 0, st>>>(a);
        note_launch();
        DDG_CUDA(cudaGetLastError());
        return DDG_OK;
    }
    if (plan.kernel == Q4_GEMV) return a.M == 1 ? launch_gemv<T, 1>(a, st) : launch_gemv<T, 2>(a, st);
    DDG_CHECK(plan.kernel >= 0, DDG_ERR_ARG, "fc_q4: %d rows of K = %d are too many for one call", a.M, a.w.K);
    constexpr int F = sizeof(T) / 4;
    static_assert(QtShape<T, 4 / F, 1>::KC == Q4_TILE[0].kc && QtShape<T, 8 / F, 1>::KC == Q4_TILE[1].kc &&
                      QtShape<T, 16 / F, 1>::KC == Q4_TILE[2].kc && QtShape<T, 32 / F, 1>::KC == Q4_TILE[3].kc &&
                      QtShape<T, 64 / F, 1>::KC == Q4_TILE[4].kc && QtShape<T, 64 / F, 2>::KC == Q4_TILE[5].kc,
                  "stages of the plan and of the kernels");
    static int (*const launch[Q4_TILES])(const Q4Args<T> &, int, cudaStream_t) = {
        launch_tc_q4<T, 4 / F, 1>,  launch_tc_q4<T, 8 / F, 1>,  launch_tc_q4<T, 16 / F, 1>,
        launch_tc_q4<T, 32 / F, 1>, launch_tc_q4<T, 64 / F, 1>, launch_tc_q4<T, 64 / F, 2>};
    return launch[plan.kernel](a, plan.split, st);
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
