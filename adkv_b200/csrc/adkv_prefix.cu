// Part of libadkv_b200.so (sm_100a).  See include/adkv_b200.h for the contract of every entry point.
//
// Decode step of many sequences that begin with the same tokens: the packed prefix exists once, is replayed once a step for all of
// them, and each sequence adds the tokens that it has cached itself and the new one.
//
// With x the replayed keys and y the replayed values of one KV head, the prefix part of all R = B * Hq / Hkv query rows is
//   S = Q x^T,  P = exp2(S * scaling * log2(e) - m),  O = P y,  l = sum P
// two products of matrices around a recurrence that serves every row, so the recurrence stays on the SIMT side, a channel a thread, and
// the products go to tcgen05: 128 query rows by 64 tokens at a time, Q and the replayed tiles in shared memory, S, P and O in tensor
// memory.  A CTA takes 128 rows of one head and a run of checkpoint intervals (state checkpoints make runs independent), leaves maximum,
// denominator and sums of each row in scratch memory, and the merge of adkv_split.cu joins them with the sequences' own parts.
//
// Values are rounded to fp16 for the products, as a cache of fp16 keys and values would hold them, but as differences from the zero
// point at the start of the run: that point's share of a logit is the same for the whole run and is added in fp32 to the maximum, its
// share of the result to the sums, so a channel far from zero keeps the bits of its deviations.  They are held in units of 16, a power
// of two, so that differences up to a million are in range.  Weights are rounded to fp16, sums of both products are fp32.
#include "adkv_host.h"

#include "adkv_softmax.cuh"
#include "adkv_tensor.cuh"

namespace adkv {

constexpr int kPreTok = 64, kPreRows = 128;   // tokens of a tile, query rows of a CTA
constexpr int kPreWarps = 14;                 // 0-3: K, 4-7: V (a channel a thread), 8-11: softmax (a row a thread), 12, 13: products
constexpr int kPreThreads = 32 * kPreWarps;
constexpr float kPreUnit = 16.f;              // values are held in units of this
constexpr float kPreSlack = 8.f;              // a row's sums are rescaled when its maximum has grown by 2^this: weights stay below 2^8

struct PrefixArgs {
    const __half *q;                 // [B, Hq, kD]
    const uint8_t *cache[2];         // K, V: [Hkv, n_super_cap, kD] words
    const float *ckpt[2];            // [Hkv, n_ckpt_cap, 2, kD]; entry i = state before token (i + 1) * interval
    ParamPtrs p[2];
    float *scratch;                  // [B * Hkv, n_parts, G, kPartStride]
    int Hq, Hkv, rows, row_tiles, n_super_cap, n_ckpt_cap, tokens, interval;
    int run, n_runs, n_parts;        // tokens of a run (a multiple of interval), runs, parts of a stream in scratch
    float scaling, smin, smax;
};

struct PrefixShared {
    alignas(128) __half q[kD / 8][kPreRows][8];          // [channel / 8][row][channel % 8]
    alignas(128) __half x[2][2][kPreTok / 8][kD][8];     // K, V; buffer; [token / 8][channel][token % 8]
    float z0[kD];                                        // zero points of K before the run
    uint32_t tmem;
    int dead;                                            // a bounded wait gave up
    // of tile i, buffer i % 2: K and V values are there; S is there (and K has been read); weights are there; O is added up (V, P read)
    uint64_t full[2][2], sdone[2], pfull[2], odone[2];
};

// K-major shared-memory matrix without swizzle: element (m, k) lies at (m / 8) * m_stride + (k / 8) * k_stride + (m % 8) * 16 + (k % 8) * 2.
__device__ __forceinline__ uint64_t k_major_desc(const void *p, uint32_t k_stride, uint32_t m_stride) { return mn_major_desc(p, k_stride, m_stride); }
// fp16 x fp16 -> fp32, A K-major; B K-major or N-major
__host__ __device__ constexpr uint32_t pre_mma_desc(int M, int N, bool b_mn)
{
    return 1u << 4 | uint32_t(b_mn) << 16 | uint32_t(N >> 3) << 17 | uint32_t(M >> 4) << 24;
}

// What one thread keeps of its channel, in units of kPreUnit; the zero point counts from the start of the run.
struct PrefixChan {
    float zp, s, alpha, beta, tc, lo, hi;   // lo, hi: scales that eight updates cannot bring to a bound
    __device__ __forceinline__ bool safe() const { return __all_sync(kFull, s >= lo && s <= hi); }
};
// Eight tokens, fields 0..7 of w, contracted as in k_chunk2.
template <int BITS, bool GUARDED>
__device__ __forceinline__ void prefix_window(uint32_t w, const FieldConsts<BITS> &fc, PrefixChan &c, float smin, float smax, float eps, float (&x)[8])
{
    static_for<8>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        const float q = fc.template code<j % 4>(j < 4 ? w : w >> (4 * BITS));
        const float rh = __fmul_rn(q, GUARDED ? fmaxf(c.s, eps) : c.s);
        x[j] = __fadd_rn(rh, c.zp);
        c.zp = fmaf(c.alpha, rh, c.zp);
        c.s *= fmaf(c.beta, fabsf(q), c.tc);
        if (GUARDED) c.s = fminf(fmaxf(c.s, smin), smax);
    });
}
struct PrefixWindow {
    float x[8], zp, s;
};
template <int BITS>
__device__ __noinline__ PrefixWindow prefix_window_guarded(uint32_t w, PrefixChan c, float smin, float smax, float eps)
{
    FieldConsts<BITS> fc;
    fc.init();
    PrefixWindow r;
    prefix_window<BITS, true>(w, fc, c, smin, smax, eps, r.x);
    r.zp = c.zp;
    r.s = c.s;
    return r;
}

__device__ __forceinline__ float exp2_fast(float v)   // underflows to zero; the arguments are at most kPreSlack
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void warp_arrive(uint64_t *bar, int lane)
{
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

template <int BITS>
__global__ void __launch_bounds__(kPreThreads, 2) prefix_kernel(const __grid_constant__ PrefixArgs a)
{
    extern __shared__ __align__(128) uint8_t smem_raw[];
    PrefixShared &sh = *reinterpret_cast<PrefixShared *>(smem_raw);
    constexpr int TPW = Codec<BITS>::TPW, ROWS = kPreTok / TPW;                 // word rows of a tile
    constexpr uint32_t kColS = 0, kColO = 2 * kPreTok, kColumns = 256;          // S (and P in its place) twice, O
    const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rt = blockIdx.x % a.row_tiles, h = blockIdx.x / a.row_tiles % a.Hkv, run = blockIdx.x / a.row_tiles / a.Hkv;
    const int G = a.Hq / a.Hkv;
    const int t0 = run * a.run, ntok = min(a.run, a.tokens - t0), n_tiles = (ntok + kPreTok - 1) / kPreTok;
    const int n_rows = (ntok + TPW - 1) / TPW;                                  // word rows of the run
    const int rows = min(kPreRows, a.rows - rt * kPreRows);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.full[0][i], 4);
            mbar_init(&sh.full[1][i], 4);
            mbar_init(&sh.sdone[i], 1);
            mbar_init(&sh.pfull[i], 4);
            mbar_init(&sh.odone[i], 1);
        }
        sh.dead = 0;
        mbar_init_fence();
    }
    if (warp == 12) tmem_alloc(&sh.tmem, kColumns);
    // query rows, negated where the scaling is negative (rows behind the last one as zeros)
    const uint32_t sign = a.scaling < 0.f ? 0x80008000u : 0u;
    for (int i = threadIdx.x; i < kPreRows * (kD / 8); i += kPreThreads) {
        const int r = i / (kD / 8), k = i % (kD / 8), n = rt * kPreRows + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            const uint2 *src = reinterpret_cast<const uint2 *>(a.q + (size_t(n / G) * a.Hq + size_t(h) * G + n % G) * kD + 8 * k);
            const uint2 lo = src[0], hi = src[1];
            v = make_uint4(lo.x ^ sign, lo.y ^ sign, hi.x ^ sign, hi.y ^ sign);
        }
        *reinterpret_cast<uint4 *>(&sh.q[k][r][0]) = v;
    }
    const int which = warp >> 2 & 1;   // of the scanning warps: 0 K, 1 V
    const int c = threadIdx.x & (kD - 1);
    PrefixChan ch;
    float start = 0.f;                 // zero point before the run: K, and V for the threads that store the result
    if (warp < 8) {
        const ParamPtrs &p = a.p[which];
        const size_t po = size_t(h) * kD + c;
        const float alpha = __half2float(p.alpha[po]), beta = __half2float(p.beta[po]), target = __half2float(p.target[po]);
        float s;
        if (t0 > 0) {
            const float *init = a.ckpt[which] + (size_t(h) * a.n_ckpt_cap + t0 / a.interval - 1) * 2 * kD;
            start = init[c];
            s = init[kD + c];
        } else {
            start = __half2float(p.zp_init[po]);
            s = __half2float(p.scale_init[po]);
        }
        if (which == 0) sh.z0[c] = start;
        SafeRange safe{0.f, INFINITY};
        const float be[1] = {beta}, tg[1] = {target};
        safe.template init<BITS, 1>(be, tg, a.smin, a.smax);
        ch = PrefixChan{0.f, s * (1.f / kPreUnit), alpha, beta, fmaf(-beta, target, 1.0f), safe.lo * (1.f / kPreUnit), safe.hi * (1.f / kPreUnit)};
    }
    fence_async_shared();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    bool ok = true;

    if (warp < 8) {
        // ------------------------------------------------------------------------------ K and V values
        FieldConsts<BITS> fc;
        fc.init();
        const uint32_t *words = reinterpret_cast<const uint32_t *>(a.cache[which]) + (size_t(h) * a.n_super_cap + t0 / TPW) * kD + c;
        const float smin = a.smin * (1.f / kPreUnit), smax = a.smax * (1.f / kPreUnit), eps = kEps * (1.f / kPreUnit);
        uint64_t *freed = which ? sh.odone : sh.sdone;
        uint32_t next[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) next[r] = r < n_rows ? words[size_t(r) * kD] : 0u;
        bool safe = ch.safe();
#pragma unroll 1
        for (int i = 0; i < n_tiles; ++i) {
            const int buf = i & 1;
            uint32_t w[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) w[r] = next[r];
#pragma unroll
            for (int r = 0; r < ROWS; ++r) next[r] = (i + 1) * ROWS + r < n_rows ? words[size_t((i + 1) * ROWS + r) * kD] : 0u;
            if (i >= 2 && !(ok = mbar_wait(&freed[buf], (i / 2 & 1) ^ 1, kStatKWait))) break;
            uint8_t *dst = reinterpret_cast<uint8_t *>(&sh.x[which][buf][0][c][0]);
            const int left = ntok - i * kPreTok;
#pragma unroll
            for (int n = 0; n < kPreTok / 8; ++n) {
                const uint32_t word = BITS == 4 ? w[n % ROWS] : w[n / 2 % ROWS] >> (16 * (n & 1));
                float x[8];
                if (safe) {
                    prefix_window<BITS, false>(word, fc, ch, smin, smax, eps, x);
                } else {
                    const PrefixWindow r = prefix_window_guarded<BITS>(word, ch, smin, smax, eps);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = r.x[j];
                    ch.zp = r.zp;
                    ch.s = r.s;
                }
                safe = ch.safe();
                if (left < 8 * n + 8) {   // behind the last token: whatever the words hold there does not count
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = 8 * n + j < left ? x[j] : 0.f;
                }
                *reinterpret_cast<uint4 *>(dst + n * kD * 16) = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
            }
            fence_async_shared();
            warp_arrive(&sh.full[which][buf], lane);
        }
        if (!ok && lane == 0) sh.dead = 1;
        __syncthreads();
    } else if (warp < 12) {
        // ------------------------------------------------------------------------------ weights, a row a thread
        const int e = warp & 3, r = 32 * e + lane;
        const bool busy = 32 * e < rows;
        const uint32_t lanes = tmem + (uint32_t(32 * e) << 16);
        const float scale2 = a.scaling * 1.4426950408889634f, f = fabsf(scale2) * kPreUnit;
        float m = -INFINITY, l = 0.f;
#pragma unroll 1
        for (int i = 0; i < n_tiles; ++i) {
            const int buf = i & 1;
            if (!(ok = mbar_wait(&sh.sdone[buf], i / 2 & 1, kStatLFullWait))) break;
            if (busy) {
                tc_fence_after();
                const uint32_t at = lanes + kColS + kPreTok * buf;
                const int left = ntok - i * kPreTok;
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < kPreTok; n += 16) {
                    uint32_t v[16];
                    tmem_ld(v, at + n);
                    tmem_wait_ld(v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) top = fmaxf(top, n + j < left ? __uint_as_float(v[j]) : -INFINITY);
                }
                top *= f;
                const bool grown = top > m + kPreSlack;   // the first tile: m is -inf
                if (__any_sync(kFull, grown)) {
                    const float corr = grown ? exp2_fast(m - top) : 1.f;
                    if (i > 0) {
                        // all sums so far are in: O can be changed
                        if (!(ok = mbar_wait(&sh.odone[buf ^ 1], ((i - 1) / 2 & 1), kStatVWait))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int n = 0; n < kD; n += 16) {
                            uint32_t v[16];
                            tmem_ld(v, lanes + kColO + n);
                            tmem_wait_ld(v);
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * corr);
#pragma unroll
                            for (int j = 0; j < 16; j += 4) tmem_st4(lanes + kColO + n + j, v[j], v[j + 1], v[j + 2], v[j + 3]);
                        }
                    }
                    l *= corr;
                    if (grown) m = top;
                }
#pragma unroll
                for (int n = 0; n < kPreTok; n += 16) {
                    uint32_t v[16];
                    tmem_ld(v, at + n);
                    tmem_wait_ld(v);
                    float p[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        p[j] = exp2_fast(fmaf(__uint_as_float(v[j]), f, -m));
                        if (n + j >= left) p[j] = 0.f;
                        l += p[j];
                    }
#pragma unroll
                    for (int j = 0; j < 16; j += 8)
                        tmem_st4(at + (n + j) / 2, pack2(p[j], p[j + 1]), pack2(p[j + 2], p[j + 3]), pack2(p[j + 4], p[j + 5]), pack2(p[j + 6], p[j + 7]));
                }
                tmem_wait_st();
                tc_fence_before();
            }
            warp_arrive(&sh.pfull[buf], lane);
        }
        if (ok) ok = mbar_wait(&sh.odone[(n_tiles - 1) & 1], (n_tiles - 1) / 2 & 1, kStatVWait);
        if (!ok && lane == 0) sh.dead = 1;
        __syncthreads();
        const bool dead = sh.dead != 0;
        if (busy) {
            tc_fence_after();
            const int n_row = rt * kPreRows + r, b = n_row / G, g = n_row % G;
            float *part = a.scratch + ((size_t(b * a.Hkv + h) * a.n_parts + run) * G + g) * kPartStride;
            float base = 0.f;   // what the zero points before the run add to every logit of the row
#pragma unroll 4
            for (int k = 0; k < kD / 8; ++k) {
                float qv[4];
                load_half4(qv, &sh.q[k][r][0]);
#pragma unroll
                for (int j = 0; j < 4; ++j) base = fmaf(qv[j], sh.z0[8 * k + j], base);
                load_half4(qv, &sh.q[k][r][4]);
#pragma unroll
                for (int j = 0; j < 4; ++j) base = fmaf(qv[j], sh.z0[8 * k + 4 + j], base);
            }
            if (r < rows) {
                part[0] = dead ? -INFINITY : fmaf(base, fabsf(scale2), m);
                part[1] = dead ? __int_as_float(0x7fc00000) : l;
            }
            const float *init = a.ckpt[1] + (size_t(h) * a.n_ckpt_cap + (t0 > 0 ? t0 / a.interval - 1 : 0)) * 2 * kD;
#pragma unroll 1
            for (int n = 0; n < kD; n += 16) {
                uint32_t v[16];
                tmem_ld(v, lanes + kColO + n);
                tmem_wait_ld(v);
                if (r < rows) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        float z[4];
                        if (t0 > 0) {
                            const float4 z4 = *reinterpret_cast<const float4 *>(init + n + j);
                            z[0] = z4.x; z[1] = z4.y; z[2] = z4.z; z[3] = z4.w;
                        } else {
                            load_half4(z, a.p[1].zp_init + size_t(h) * kD + n + j);
                        }
                        float o[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[k] = dead ? 0.f : fmaf(l, z[k], kPreUnit * __uint_as_float(v[j + k]));
                        *reinterpret_cast<float4 *>(part + 4 + n + j) = make_float4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
        }
    } else if (warp == 12) {
        // ------------------------------------------------------------------------------ S = Q x^T
        constexpr uint32_t desc = pre_mma_desc(kPreRows, kPreTok, true);
        int i = 0;
#pragma unroll 1
        for (; i < n_tiles; ++i) {
            const int buf = i & 1;
            if (!(ok = mbar_wait(&sh.full[0][buf], i / 2 & 1, kStatKWait))) break;
            if (i >= 2 && !(ok = mbar_wait(&sh.odone[buf], (i / 2 & 1) ^ 1, kStatVWait))) break;   // the weights in S's place are used
            tc_fence_after();
            if (elect_one()) {
                const uint64_t qd = k_major_desc(&sh.q[0][0][0], kPreRows * 16, 128), xd = mn_major_desc(&sh.x[0][buf][0][0][0], 128, kD * 16);
#pragma unroll
                for (int n = 0; n < kD / 16; ++n)
                    mma_smem(tmem + kColS + kPreTok * buf, qd + 2 * (kPreRows * 16 / 16) * n, xd + 16 * n, desc, n > 0);
                mma_commit(&sh.sdone[buf]);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) sh.dead = 1;
        __syncthreads();
        if (sh.dead)   // products in flight
            for (int k = max(i - 2, 0); k < i; ++k) mbar_wait(&sh.sdone[k & 1], k / 2 & 1, kStatDrain);
    } else {
        // ------------------------------------------------------------------------------ O += P y
        constexpr uint32_t desc = pre_mma_desc(kPreRows, kD, false);
        int i = 0;
#pragma unroll 1
        for (; i < n_tiles; ++i) {
            const int buf = i & 1;
            if (!(ok = mbar_wait(&sh.full[1][buf], i / 2 & 1, kStatVWait))) break;
            if (!(ok = mbar_wait(&sh.pfull[buf], i / 2 & 1, kStatVWait))) break;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t yd = k_major_desc(&sh.x[1][buf][0][0][0], kD * 16, 128);
#pragma unroll
                for (int n = 0; n < kPreTok / 16; ++n)
                    mma_tmem(tmem + kColO, tmem + kColS + kPreTok * buf + 8 * n, yd + 2 * (kD * 16 / 16) * n, desc, i > 0 || n > 0);
                mma_commit(&sh.odone[buf]);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) sh.dead = 1;
        __syncthreads();
        if (sh.dead)
            for (int k = max(i - 2, 0); k < i; ++k) mbar_wait(&sh.odone[k & 1], k / 2 & 1, kStatDrain);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_free(tmem, kColumns);
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the merge waits for this kernel, and with it for the one before
}

// =========================================================================================
// The tokens that a sequence has cached itself, from the state behind the prefix, and the new one: one CTA per stream, as the
// checkpointed step has one per segment.
template <int BITS, int G>
__global__ void __launch_bounds__(64) prefix_own_kernel(KArgs ka, VArgs va, const float *__restrict__ k_state, const float *__restrict__ v_state,
                                                        const int *__restrict__ seq_lens, float scaling, float *__restrict__ scratch, int n_parts)
{
    constexpr int TOK = 64, ST = 2;
    __shared__ alignas(128) uint8_t kbuf[ST * Tile<BITS, TOK>::BYTES];
    __shared__ alignas(128) uint8_t vbuf[ST * Tile<BITS, TOK>::BYTES];
    __shared__ alignas(16) float red[G * 8 * kRedRow];
    __shared__ alignas(16) float2 wts[G * TOK];
    __shared__ FusedShared<G, 1, TOK> fs;
    __shared__ uint64_t kbar[ST], vbar[ST];

    const int bh = blockIdx.x, b = bh / ka.Hkv, h = bh % ka.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float *part = scratch + (size_t(bh) * n_parts + n_parts - 1) * G * kPartStride;
    if (seq_lens) {
        const int T = seq_lens[b];
        if (T < 0 || T / Codec<BITS>::TPW >= ka.n_super_cap) {   // does not fit: nothing is appended, the outputs of the sequence are NaN
            if (threadIdx.x == 0) atomicExch(&g_status, kStatCapacity);
            for (int i = threadIdx.x; i < G * kPartStride; i += 64)
                part[i] = i % kPartStride == 0 ? -INFINITY : i % kPartStride == 1 ? __int_as_float(0x7fc00000) : 0.f;
            return;
        }
        ka.T = T;
        va.T = T;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) { mbar_init(&kbar[i], 1); mbar_init(&vbar[i], 1); }
        fs.init_barriers(1);
        mbar_init_fence();
    }
    __syncthreads();
    const float *init = (warp == 0 ? k_state : v_state) + size_t(h) * 2 * kD;
    const Seg seg{0, ka.T, true, init, nullptr, 0};
    if (warp == 0) {
        RingSink<G, 1, TOK> sink{&fs, 0, 0};
        k_warp<BITS, G, kArithFma, RingSink<G, 1, TOK>, ST, false, BITS == 4 && G == 1, 8, TOK>(ka, seg, b, h, lane, kbuf, kbar, red, sink);
    } else {
        using Src = PartialSrc<G, false, TOK>;
        Src src;
        src.sh = &fs;
        src.wts = wts;
        src.mask = nullptr;
        src.scale2 = scaling * 1.4426950408889634f;
        src.n_tiles = (ka.T + TOK - 1) / TOK;
        src.t_begin = 0;
        src.part = part;
        src.init();
        v_warp<BITS, G, kArithFma, Src, ST, false, BITS == 4 && G == 1, TOK>(va, seg, b, h, lane, vbuf, vbar, wts, src);
    }
}

// Intervals of a run: few enough runs to be set up cheaply, enough to fill the chip evenly.  Two CTAs share an SM.
static int run_intervals(int tokens, int interval, int Hkv, int row_tiles)
{
    if (interval <= 0 || tokens <= interval) return 1;
    const int n = (tokens + interval - 1) / interval;
    int best = 1;
    double least = 1e30;
    for (int k = 1; k <= n; ++k) {
        const int runs = (n + k - 1) / k;
        if (runs > 128) continue;
        const long long ctas = (long long)runs * Hkv * row_tiles, rounds = (ctas + 2 * kSMs - 1) / (2 * kSMs);
        const double cost = double(rounds) * (double(k) * interval + 96);
        if (cost < least) {
            least = cost;
            best = k;
        }
    }
    return best;
}
static int prefix_runs(int tokens, int interval, int Hkv, int row_tiles, int *run)
{
    if (tokens == 0) { *run = 0; return 0; }
    *run = interval > 0 ? run_intervals(tokens, interval, Hkv, row_tiles) * interval : tokens;
    return (tokens + *run - 1) / *run;
}

}  // namespace adkv

using namespace adkv;

ADKV_HIDDEN int adkv_launch_merge(const float *scratch, __half *out, int B, int Hq, int Hkv, int n_seg, cudaStream_t s);

ADKV_DEFINE_TU_STATUS(adkv_tu_status_prefix)

template <int BITS>
static int launch_prefix(const PrefixArgs &a, cudaStream_t s)
{
    constexpr int bytes = int(sizeof(PrefixShared));
    static_assert(2 * (bytes + 1024) <= 228 * 1024, "two CTAs share an SM");
    const auto kernel = prefix_kernel<BITS>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return launch_status();
    kernel<<<a.n_runs * a.Hkv * a.row_tiles, kPreThreads, bytes, s>>>(a);
    return launch_status();
}

extern "C" {

long long adkv_decode_attn_prefix_scratch_bytes(int B, int Hq, int Hkv, int prefix_tokens, int interval)
{
    if (B < 0 || Hq <= 0 || Hkv <= 0 || prefix_tokens < 0 || interval < 0 || Hq % Hkv != 0) return ADKV_E_SHAPE;
    int run;
    const int runs = prefix_runs(prefix_tokens, interval, Hkv, int(((long long)B * (Hq / Hkv) + kPreRows - 1) / kPreRows), &run);
    return (long long)B * Hq * (runs + 1) * kPartStride * (long long)sizeof(float);
}

int adkv_decode_attn_prefix(const void *q, const adkv_prefix *prefix, void *k_cache, void *v_cache, const void *k_new, const void *v_new,
                            const adkv_params *kp, const adkv_params *vp, void *k_tail, void *v_tail, const void *seq_lens, int T, void *out,
                            void *scratch, long long scratch_bytes, int B, int Hq, int Hkv, int D, int n_super_cap, int bits, float scaling,
                            float scale_min, float scale_max, unsigned flags, void *stream)
{
    if (!q || !prefix || !k_cache || !v_cache || !k_new || !v_new || !out || !params_ok(kp) || !params_ok(vp) || !k_tail || !v_tail || !scratch ||
        !prefix->k_tail || !prefix->v_tail || (prefix->tokens > 0 && (!prefix->k_cache || !prefix->v_cache)))
        return ADKV_E_NULL;
    if (D != kD) return ADKV_E_HEAD_DIM;
    if (seq_lens) T = 0;
    if (int rc = check_common(B, Hq, Hkv, T, D, n_super_cap, bits, T + 1)) return rc;
    const int G = Hq / Hkv;
    if (G != 1 && G != 2 && G != 4 && G != 8) return ADKV_E_SHAPE;
    if (flags & ~unsigned(ADKV_FLAG_TAIL_KEEP | ADKV_FLAG_FAST_REPLAY)) return ADKV_E_FLAGS;
    const int P = prefix->tokens, iv = prefix->interval;
    if (P < 0 || prefix->n_super_cap < 0 || iv < 0 || iv % kTileTok || prefix->n_ckpt_cap < 0) return ADKV_E_SHAPE;
    if (((long long)P + 32 / bits - 1) / (32 / bits) > prefix->n_super_cap) return ADKV_E_CAPACITY;
    if (iv > 0 && P > iv) {
        if (!prefix->k_ckpt || !prefix->v_ckpt) return ADKV_E_NULL;
        if ((P - 1) / iv > prefix->n_ckpt_cap) return ADKV_E_CAPACITY;
    }
    if (!aligned8(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned8(k_new) || !aligned8(v_new) || !aligned8(out) || !params_aligned(kp) ||
        !params_aligned(vp) || !aligned16(k_tail) || !aligned16(v_tail) || !aligned16(scratch) || !aligned16(prefix->k_cache) ||
        !aligned16(prefix->v_cache) || !aligned16(prefix->k_tail) || !aligned16(prefix->v_tail) || !aligned16(prefix->k_ckpt) ||
        !aligned16(prefix->v_ckpt) || (reinterpret_cast<uintptr_t>(seq_lens) & 3u))
        return ADKV_E_ALIGN;
    const long long rows = (long long)B * G;
    if (rows > (1 << 24)) return ADKV_E_SHAPE;
    if (scratch_bytes < adkv_decode_attn_prefix_scratch_bytes(B, Hq, Hkv, P, iv)) return ADKV_E_SCRATCH;
    if (B == 0) return 0;

    PrefixArgs pa{};
    pa.q = static_cast<const __half *>(q);
    pa.cache[0] = static_cast<const uint8_t *>(prefix->k_cache);
    pa.cache[1] = static_cast<const uint8_t *>(prefix->v_cache);
    pa.ckpt[0] = static_cast<const float *>(prefix->k_ckpt);
    pa.ckpt[1] = static_cast<const float *>(prefix->v_ckpt);
    pa.p[0] = to_ptrs(kp);
    pa.p[1] = to_ptrs(vp);
    pa.scratch = static_cast<float *>(scratch);
    pa.Hq = Hq;
    pa.Hkv = Hkv;
    pa.rows = int(rows);
    pa.row_tiles = (pa.rows + kPreRows - 1) / kPreRows;
    pa.n_super_cap = prefix->n_super_cap;
    pa.n_ckpt_cap = prefix->n_ckpt_cap;
    pa.tokens = P;
    pa.interval = iv;
    pa.n_runs = prefix_runs(P, iv, Hkv, pa.row_tiles, &pa.run);
    pa.n_parts = pa.n_runs + 1;
    pa.scaling = scaling;
    pa.smin = scale_min;
    pa.smax = scale_max;
    const bool keep = flags & ADKV_FLAG_TAIL_KEEP;
    const KArgs ka{pa.q, static_cast<uint8_t *>(k_cache), static_cast<const __half *>(k_new), pa.p[0], Hq, Hkv, T, n_super_cap, scale_min, scale_max, D,
                   static_cast<float *>(k_tail), keep};
    const VArgs va{static_cast<uint8_t *>(v_cache), static_cast<const __half *>(v_new), static_cast<__half *>(out), pa.p[1], Hq, Hkv, T, n_super_cap,
                   scale_min, scale_max, D, static_cast<float *>(v_tail), keep};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (pa.n_runs)
        if (int rc = bits == 4 ? launch_prefix<4>(pa, s) : launch_prefix<2>(pa, s)) return rc;
    ADKV_DISPATCH_H(bits, G, (prefix_own_kernel<BITS, G><<<B * Hkv, 64, 0, s>>>(ka, va, static_cast<const float *>(prefix->k_tail),
                                                                               static_cast<const float *>(prefix->v_tail),
                                                                               static_cast<const int *>(seq_lens), scaling, pa.scratch, pa.n_parts)))
    if (int rc = launch_status()) return rc;
    return adkv_launch_merge(pa.scratch, static_cast<__half *>(out), B, Hq, Hkv, pa.n_parts, s);
}

}  // extern "C"
