// Fully connected layers with 4-bit public weights and group steps:
//
//   out[m][n] = sign * sum_k x[m][k] W[k][n] + bias[n] + Add[m][n]   modulo 2^bw
//   W[k][n]   = step[k / group][n] * (code(n, k) - 8)
//
// Two kernels, both exact modulo 2^bw, so the result does not depend on how K
// is split over lanes, warps or CTAs.
//
// k_q4_gemv, for one or two rows: 8-bit limb products on the CUDA cores.  x
// sits in shared memory as byte planes, four k of one limb to a word, and
// dp4a multiplies a word by four codes: per unit of 32 codes (one 16-byte
// load, one step)
//   sum_k x_k W_k = step * ( sum_l 2^(8l) dp4a(code, limb l of x) - 8 sum_k x_k ).
//
// k_q4_tc, for more rows: the weights are 16-bit numbers, W + 2^15 = w0 + 2^8 w1
// with unsigned bytes, and x = sum_l 2^(8l) x_l, so
//   x . W = sum_s 2^(8s) (x_s . w0 + x_{s-1} . w1) - 2^15 sum_k x_k .
// The weights are the M side of the MMA (128 outputs), and the limbs of MT
// rows of x its N side (limb-major, P * MT columns): one MMA with w0 covers
// every limb, one with w1 into the columns of the next limb every shifted one.
// 2 wide MMAs per 32 k, and 2 P byte products where full-width ring weights
// take P(P+1)/2.  Codes are expanded by all threads while the MMAs of earlier
// stages run; the sums of a split K meet in the cluster's shared memory.
#include <type_traits>

#include "token.cuh"
#include "umma.cuh"

namespace ddg {

namespace {

constexpr int Q4_THREADS = 256;

// ------------------------------------------------------------------ one or two rows

constexpr int GV_WARPS = Q4_THREADS / 32;
constexpr int GV_R = 4;                       // outputs per lane group and pass
constexpr uint64_t GV_SMEM_MAX = 96 * 1024;

// units of 32 k; a group of L lanes takes one unit each, KS warps of the CTA split the units
struct GvGeom {
    int U, L, nseg, KS, slots, blocks;
};

inline GvGeom gv_geom(int K, int N)
{
    GvGeom g;
    g.U = (K + 31) / 32;
    g.L = 1;
    while (g.L < 32 && g.L < g.U) g.L *= 2;
    g.nseg = (g.U + g.L - 1) / g.L;
    g.KS = g.nseg < 1 ? 1 : g.nseg < GV_WARPS ? g.nseg : GV_WARPS;
    g.slots = GV_WARPS / g.KS * (32 / g.L);
    g.blocks = (N + g.slots * GV_R - 1) / (g.slots * GV_R);
    return g;
}

template <typename T>
uint64_t gv_smem(const GvGeom &g, int rows)
{
    return uint64_t(rows) * g.U * (32 * sizeof(T) + sizeof(T)) + uint64_t(GV_WARPS) * 32 * GV_R * rows * sizeof(T);
}

template <typename T, int MR>
__global__ void __launch_bounds__(Q4_THREADS)
    k_q4_gemv(const __grid_constant__ Q4Args<T> a, const __grid_constant__ GvGeom g, int64_t row_bytes)
{
    constexpr int P = int(sizeof(T)), R = GV_R;
    extern __shared__ __align__(16) uint8_t smem_raw[];
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

    // the first codes are in flight while x is split
    Codes cur;
    fetch(blockIdx.x, ks, cur);
    const int quarters = MR * g.U * 4;
    for (int i0 = warp * 32; i0 < quarters; i0 += Q4_THREADS) {  // warp-uniform: the shuffles below are whole
        const bool in = i0 + lane < quarters;
        const int i = in ? i0 + lane : 0;
        const int m = i / (g.U * 4), u = (i >> 2) % g.U, j = i & 3;
        T e[8], sum = 0;
#pragma unroll
        for (int t = 0; t < 8; t++) {
            const int k = u * 32 + j * 8 + t;
            e[t] = in && k < a.w.K ? __ldg(a.x + int64_t(m) * a.ldx + k) : T(0);
            sum += e[t];
        }
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
            Codes next;
            if (seg + g.KS < g.nseg)
                fetch(blk, seg + g.KS, next);
            else
                fetch(blk + gridDim.x, ks, next);
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

constexpr int QT_KC = 64;     // k per stage (two MMA K-steps)
constexpr int QT_STAGES = 3;
constexpr int QT_MAX_CHUNKS = 32768 / QT_KC;
constexpr uint32_t QT_PLANE = TC_BM * 32;  // bytes of one weight plane per K-step

template <typename T, int MT>
struct QtShape {
    static constexpr int P = int(sizeof(T));
    static constexpr int NB = P * MT;                              // columns of the w0 MMA
    static constexpr int NH = ((P - 1) * MT + 15) / 16 * 16;       // columns of the w1 MMA (from column MT)
    static constexpr int COLS = tmem_cols(NB > MT + NH ? NB : MT + NH);
    static constexpr uint32_t B_STEP = NB * 32;                    // bytes of the x limbs per K-step
    static constexpr uint32_t A_STAGE = 2 * 2 * QT_PLANE, STAGE = A_STAGE + 2 * B_STEP;
    static constexpr int EK = 64 / P;                              // k per x item (64 bytes)
    static constexpr int ITEMS = MT * (QT_KC / EK);
    // [barriers, TMEM address | sums of x | pad to 1024 | stages | slack]
    static constexpr uint32_t HEAD = 64 + MT * P;
    static constexpr uint32_t SMEM = HEAD + 1024 + QT_STAGES * STAGE + 4096;
    static_assert(NB % 16 == 0 && NB <= 256 && ITEMS <= Q4_THREADS, "tile");
};

__device__ __forceinline__ void cluster_sync()
{
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

// 8 codes times a step, plus 2^15: byte planes (low, high) of k = 0..3 and 4..7
__device__ __forceinline__ void q4_expand(uint32_t c, uint32_t s, uint32_t bias, uint32_t &lo0, uint32_t &lo1,
                                          uint32_t &hi0, uint32_t &hi1)
{
    // codes k and k + 4 in the two halves of a word: one multiply-add makes both 16-bit weights (no
    // carry between the halves: 0 <= s * code + 2^15 - 8 s < 2^16 for s <= 4095)
    uint32_t p[4];
    byte_planes((c & 0x000f000fu) * s + bias, ((c >> 4) & 0x000f000fu) * s + bias, ((c >> 8) & 0x000f000fu) * s + bias,
                ((c >> 12) & 0x000f000fu) * s + bias, p);
    lo0 = p[0], hi0 = p[1], lo1 = p[2], hi1 = p[3];
}

template <typename T, int MT>
__global__ void __launch_bounds__(Q4_THREADS, 2)
    k_q4_tc(const __grid_constant__ Q4Args<T> a, int64_t row_bytes, int per, int vec, uint32_t *err)
{
    using S = QtShape<T, MT>;
    constexpr int P = S::P;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint64_t *const bars = reinterpret_cast<uint64_t *>(smem_raw);
    uint32_t &s_tmem = *reinterpret_cast<uint32_t *>(smem_raw + 32);
    T *const xsum = reinterpret_cast<T *>(smem_raw + 64);  // [MT]
    uint8_t *const smem = smem_raw + S::HEAD + ((1024u - ((smem_addr(smem_raw) + S::HEAD) & 1023u)) & 1023u);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n0 = blockIdx.x * TC_BM, m0 = blockIdx.y * MT;
    const int nkc = (a.w.K + QT_KC - 1) / QT_KC, c0 = blockIdx.z * per;
    const int nk = nkc - c0 < per ? (nkc - c0 > 0 ? nkc - c0 : 0) : per;

    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                     "r"(S::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < QT_STAGES; i++) mbar_init(bars + i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid < MT) xsum[tid] = 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    // this thread's unit of codes (row, 32 k) and item of x (row, EK k) of every stage
    const int arow = 16 * warp + (lane & 15), aun = lane >> 4;
    const int xm = tid % MT, xk = tid / MT;
    const bool has_x = tid < S::ITEMS, xrow = has_x && m0 + xm < a.M;
    const uint4 *const crow = reinterpret_cast<const uint4 *>(a.w.q + int64_t(n0 + arow) * row_bytes);
    const int units = (a.w.K + 31) / 32;
    const bool arow_ok = n0 + arow < a.w.N;
    const T *const xptr = a.x + int64_t(m0 + xm) * a.ldx;
    T sum = 0;
    uint4 code;
    uint32_t step;
    T xe[S::EK];

    auto load_stage = [&](int c) {
        const int u = 2 * c + aun;
        code = make_uint4(0, 0, 0, 0), step = 0;
        if (arow_ok && u < units) {
            code = __ldg(crow + u);
            step = __ldg(a.w.step + int64_t(u * 32 / a.w.group) * a.w.N + n0 + arow) & Q4_STEP_MAX;
        }
        const int k = c * QT_KC + xk * S::EK;
        if (xrow && vec && k + S::EK <= a.w.K) {
            const uint4 *v = reinterpret_cast<const uint4 *>(xptr + k);
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<uint4 *>(xe + i * (16 / P)) = __ldg(v + i);
        } else {
#pragma unroll
            for (int i = 0; i < S::EK; i++) xe[i] = xrow && k + i < a.w.K ? __ldg(xptr + k + i) : T(0);
        }
    };
    auto store_stage = [&](int st) {
        uint8_t *const base = smem + st * S::STAGE;
        const uint32_t bias = (0x8000u - 8u * step) * 0x10001u;
        const uint32_t cw[4] = {code.x, code.y, code.z, code.w};
        uint8_t *const pa = base + aun * 2 * QT_PLANE + (arow >> 3) * 256 + (arow & 7) * 16;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            uint4 lo, hi;
            q4_expand(cw[2 * hf], step, bias, lo.x, lo.y, hi.x, hi.y);
            q4_expand(cw[2 * hf + 1], step, bias, lo.z, lo.w, hi.z, hi.w);
            *reinterpret_cast<uint4 *>(pa + hf * 128) = lo;
            *reinterpret_cast<uint4 *>(pa + QT_PLANE + hf * 128) = hi;
        }
        if (has_x) {
#pragma unroll
            for (int i = 0; i < S::EK; i++) sum += xe[i];
            const int k = xk * S::EK;  // within the stage
            uint8_t *const pb = base + S::A_STAGE + (k >> 5) * S::B_STEP + ((k >> 4) & 1) * 128 + (k & 15);
            uint32_t w[P][S::EK / 4];
#pragma unroll
            for (int i = 0; i < S::EK / 4; i++) {
                uint32_t p[4];
                byte_planes(uint32_t(xe[4 * i]), uint32_t(xe[4 * i + 1]), uint32_t(xe[4 * i + 2]),
                            uint32_t(xe[4 * i + 3]), p);
#pragma unroll
                for (int l = 0; l < 4; l++) w[l][i] = p[l];
                if constexpr (P == 8) {
                    byte_planes(uint32_t(uint64_t(xe[4 * i]) >> 32), uint32_t(uint64_t(xe[4 * i + 1]) >> 32),
                                uint32_t(uint64_t(xe[4 * i + 2]) >> 32), uint32_t(uint64_t(xe[4 * i + 3]) >> 32), p);
#pragma unroll
                    for (int l = 0; l < 4; l++) w[4 + l][i] = p[l];
                }
            }
#pragma unroll
            for (int l = 0; l < P; l++) {
                const int row = l * MT + xm;
                uint8_t *const d = pb + (row >> 3) * 256 + (row & 7) * 16;
                if constexpr (P == 4)
                    *reinterpret_cast<uint4 *>(d) = make_uint4(w[l][0], w[l][1], w[l][2], w[l][3]);
                else
                    *reinterpret_cast<uint2 *>(d) = make_uint2(w[l][0], w[l][1]);
            }
        }
    };

    constexpr uint32_t ID0 = i8_idesc(S::NB, false), ID1 = i8_idesc(S::NH, false);
    bool ok = true;
    if (nk > 0) load_stage(c0);
    for (int c = 0; c < nk; c++) {
        const int st = c % QT_STAGES;
        bool mine = true;
        if (c >= QT_STAGES) mine = mbar_wait(&bars[st], uint32_t((c / QT_STAGES - 1) & 1));
        if (mine) store_stage(st);
        if (c + 1 < nk) load_stage(c0 + c + 1);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // CTA-uniform: every thread leaves the loop together if any wait gave up
        if (!__syncthreads_and(mine ? 1 : 0)) {
            ok = false;
            break;
        }
        if (tid == 0) {
            tc_fence_after();
            const uint32_t sa = smem_addr(smem + st * S::STAGE), sb = sa + S::A_STAGE;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint64_t db = smem_desc(sb + h * S::B_STEP, 128, 256);
                mma_i8(tmem, smem_desc(sa + h * 2 * QT_PLANE, 128, 256), db, ID0, (c > 0 || h > 0) ? 1u : 0u);
                // columns past limb P-1 collect products of 2^(8P) and above, which nobody reads
                mma_i8(tmem + MT, smem_desc(sa + (h * 2 + 1) * QT_PLANE, 128, 256), db, ID1, 1u);
            }
            mma_commit(&bars[st]);
        }
    }
    if (ok && nk > 0) ok = mbar_wait(&bars[(nk - 1) % QT_STAGES], uint32_t(((nk - 1) / QT_STAGES) & 1));
    if (has_x) atomicAdd(reinterpret_cast<std::conditional_t<P == 4, unsigned int, unsigned long long> *>(xsum + xm), sum);
    const int all_ok = __syncthreads_and(ok ? 1 : 0);
    tc_fence_after();

    // out += or hand over: this CTA's sum of (row m, output n0 + 32 q + lane)
    const bool split = gridDim.z > 1;
    T *const part = reinterpret_cast<T *>(smem);  // [MT][128], the stages are done
    const int q = warp & 3, h = warp >> 2, nl = 32 * q + lane;
    auto give = [&](int m, T v) {
        if (nk > 0)
            v -= xsum[m] << 15;
        else
            v = 0;
        if (split) {
            part[m * TC_BM + nl] = v;
        } else if (n0 + nl < a.w.N && m0 + m < a.M) {
            const int64_t e = int64_t(m0 + m) * a.w.N + n0 + nl;
            v *= a.sign;
            if (a.bias) v += __ldg(a.bias + n0 + nl);
            if (a.Add) v += a.Add[e];
            a.out[e] = v;
        }
    };
    if (all_ok) {
        const uint32_t lanes = tmem + (uint32_t(32 * q) << 16);
        if constexpr (MT >= 16) {
#pragma unroll 1
            for (int m = h * (MT / 2); m < (h + 1) * (MT / 2); m += 8) {
                T r[8];
#pragma unroll
                for (int e = 0; e < 8; e++) r[e] = 0;
#pragma unroll
                for (int s = 0; s < P; s++) {
                    uint32_t v[8];
                    tmem_ld8(lanes + s * MT + m, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; e++) r[e] += T(v[e]) << (8 * s);
                }
#pragma unroll
                for (int e = 0; e < 8; e++) give(m + e, r[e]);
            }
        } else if (h == 0) {
            uint32_t v[S::NB];
#pragma unroll
            for (int i = 0; i < S::NB; i += 8) {
                uint32_t t[8];
                tmem_ld8(lanes + i, t);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 8; e++) v[i + e] = t[e];
            }
#pragma unroll
            for (int m = 0; m < MT; m++) {
                T r = 0;
#pragma unroll
                for (int s = 0; s < P; s++) r += T(v[s * MT + m]) << (8 * s);
                give(m, r);
            }
        }
    } else if (tid == 0) {
        atomicOr(err, 4u);
    }
    tc_fence_before();
    if (split) {
        cluster_sync();
        const int S_ = gridDim.z, rank = blockIdx.z;
        const int rows = a.M - m0 < MT ? a.M - m0 : MT;
        for (int i = rank * Q4_THREADS + tid; i < rows * TC_BM; i += S_ * Q4_THREADS) {
            const int m = i / TC_BM, n = n0 + i % TC_BM;
            if (n >= a.w.N) continue;
            T v = 0;
            for (int z = 0; z < S_; z++) v += ld_cluster(part + i, z);
            const int64_t e = int64_t(m0 + m) * a.w.N + n;
            v *= a.sign;
            if (a.bias) v += __ldg(a.bias + n);
            if (a.Add) v += a.Add[e];
            a.out[e] = v;
        }
        cluster_sync();  // nobody leaves while its sums are read
    } else {
        __syncthreads();
    }
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
    }
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

template <typename T, int MR>
static int launch_gemv(const Q4Args<T> &a, cudaStream_t st)
{
    static thread_local int configured[64];
    auto kern = k_q4_gemv<T, MR>;
    const GvGeom g = gv_geom(a.w.K, a.w.N);
    DDG_TRY(q4_smem_limit(kern, GV_SMEM_MAX, configured));
    // up to three CTAs an SM, each splitting x once for all its outputs
    const int grid = g.blocks < 3 * 148 ? g.blocks : 3 * 148;
    kern<<<grid, Q4_THREADS, gv_smem<T>(g, MR), st>>>(a, g, int64_t(q4_row_bytes(a.w.K)));
    note_launch();
    DDG_CUDA(cudaGetLastError());
    return DDG_OK;
}

template <typename T, int MT>
static int launch_tc_q4(const Q4Args<T> &a, cudaStream_t st)
{
    using S = QtShape<T, MT>;
    static thread_local int configured[64];
    auto kern = k_q4_tc<T, MT>;
    DDG_TRY(q4_smem_limit(kern, S::SMEM, configured));
    uint32_t *err = nullptr;
    DDG_TRY(ring_gemm_err_word(&err));
    const int nkc = (a.w.K + QT_KC - 1) / QT_KC;
    const int64_t gn = (int64_t(a.w.N) + TC_BM - 1) / TC_BM, gm = (int64_t(a.M) + MT - 1) / MT;
    DDG_CHECK(gm <= 65535, DDG_ERR_ARG, "fc_q4: %d rows are too many for one call", a.M);
    // K split over a cluster until two CTAs an SM are busy, two stages each at the least
    int split = 1;
    while (split < 8 && gn * gm * split * 2 <= 2 * 148 && nkc >= 4 * split) split *= 2;
    // a column's sum stays below 2^32: 2 * 255^2 * K per CTA, K <= 2^15
    while (split < 8 && nkc > QT_MAX_CHUNKS * split) split *= 2;
    DDG_CHECK(nkc <= QT_MAX_CHUNKS * split, DDG_ERR_ARG, "fc_q4: K = %d is too long (at most %d for %d rows)", a.w.K,
              QT_MAX_CHUNKS * 8 * QT_KC, a.M);
    const int per = nkc ? (nkc + split - 1) / split : 1;
    const int vec = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && a.ldx * int64_t(sizeof(T)) % 16 == 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(gn), unsigned(gm), unsigned(split));
    cfg.blockDim = dim3(Q4_THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = unsigned(split);
    cfg.attrs = at, cfg.numAttrs = 1;
    DDG_CUDA(cudaLaunchKernelEx(&cfg, kern, a, int64_t(q4_row_bytes(a.w.K)), per, vec, err));
    note_launch();
    return DDG_OK;
}

template <typename T>
int fc_q4(const Q4Args<T> &a, cudaStream_t st)
{
    if (int64_t(a.M) * a.w.N == 0) return DDG_OK;
    const GvGeom g = gv_geom(a.w.K, a.w.N);
    if (a.M <= 2 && gv_smem<T>(g, a.M) <= GV_SMEM_MAX)
        return a.M == 1 ? launch_gemv<T, 1>(a, st) : launch_gemv<T, 2>(a, st);
    // the fewest rows per tile that hold them all, up to 256 MMA columns
    if constexpr (sizeof(T) == 4) {
        if (a.M <= 4) return launch_tc_q4<T, 4>(a, st);
        if (a.M <= 8) return launch_tc_q4<T, 8>(a, st);
        if (a.M <= 16) return launch_tc_q4<T, 16>(a, st);
        if (a.M <= 32) return launch_tc_q4<T, 32>(a, st);
        return launch_tc_q4<T, 64>(a, st);
    } else {
        if (a.M <= 2) return launch_tc_q4<T, 2>(a, st);
        if (a.M <= 4) return launch_tc_q4<T, 4>(a, st);
        if (a.M <= 8) return launch_tc_q4<T, 8>(a, st);
        if (a.M <= 16) return launch_tc_q4<T, 16>(a, st);
        return launch_tc_q4<T, 32>(a, st);
    }
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
