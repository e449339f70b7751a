// Part of libadkv_b200.so (sm_100a).  See include/adkv_b200.h for the contract of every entry point.
//
// Decode step of many sequences that begin with the same tokens: the packed prefix exists once, is replayed once a step for all of
// them, and each sequence adds the tokens that it has cached itself and the new one.
//
// With x the replayed keys and y the replayed values of one KV head, the prefix part of all R = B * Hq / Hkv query rows is
//   S = Q x^T,  P = exp2(S * scaling * log2(e) - m),  O = P y,  l = sum P
// two products of matrices around a recurrence that serves every row, so the recurrence stays on the SIMT side, a channel a thread, and
// the products go to tcgen05: 128 query rows by 32 tokens at a time, the replayed tiles in shared memory, Q, S, P and O in tensor
// memory.  A CTA takes 128 rows of one head and a run of checkpoint intervals (state checkpoints make runs independent), leaves maximum,
// denominator and sums of each row in scratch memory, and a join adds the runs up with the sequences' own parts.
//
// Values are fp16 numbers for the products, as differences from the zero point at the start of the run: that point's share of a logit is
// the same for the whole run and is added in fp32 to the maximum, its share of the result to the sums, so a channel far from zero keeps the
// bits of its deviations.  They are held in units of 16, a power of two, so that differences up to a million (16 x 65504) are in range.  One fp16 number
// is 2^-11 of a value: with channels that reach 50, as the outliers of this library's benchmark do, logits would be off by some 1e-3 and
// results by up to 2.7 times what its results may be off (2e-3 and 2e-3 of the value); with weights of 11 bits it would be up to 1.2 times.
// So K, V and the weights are pairs, rounded number and remainder (22 bits), for three more products, and sums are fp32: what is left are
// the fp16 queries and results that every step of the library has.  The pairs of the weights cost 1 % (64 sequences 69.4 -> 70.4 us).
// fp16 numbers have no step below 2^-24: a value is off by up to 2^-21 (half of that, in units of 16) however small it is.  The denominator adds up
// the weights as they were, so what small ones lose does not cancel; the largest therefore starts at 2^7 and grows to 2^15, which leaves a
// loss of 2^-32 of the largest at most per token.
//
// 8192 tokens of 32 heads, 4-bit: 57 us for 4 sequences, 65 us for 64, 79 us for 128; 16000 of 8 heads, 2-bit, 45 us for 32 x 4.  The bytes
// would take 5 us.  The scans bound it: 256 recurrences of some 20 instructions a token and head, 10.2 cycles a value and scheduler in a
// bare loop, here a third more for waits among the warps, and a sixth of the time is filling and emptying (first words 2 us, results 3 us).
// Tiles of 64 tokens, worked on in halves: within 3 % of that, but 15.2 instead of 14.0 us where the prefix has 300 tokens.
#include "adkv_host.h"

#include <algorithm>

#include "adkv_softmax.cuh"
#include "adkv_tensor.cuh"

namespace adkv {

constexpr int kPreTok = 32, kPreRows = 128;   // tokens of a tile, query rows of a CTA
constexpr int kPreWords = 4, kPreKV = 3, kPreP = 2;   // tiles of words, of K and of V values, and of S and weights that are on their way at once
constexpr int kPreWarps = 14;                 // 0-3: K, 4-7: V (a channel a thread), 8-11: softmax (a row a thread), 12, 13: products
constexpr int kPreThreads = 32 * kPreWarps;
constexpr float kPreUnit = 16.f;              // values are held in units of this
constexpr float kPreTop = 7.f, kPreSlack = 8.f;   // the weight of a row's maximum is 2^kPreTop; sums are rescaled when it has grown by 2^kPreSlack

struct PrefixArgs {
    const __half *q;                 // [B, Hq, kD]
    const uint8_t *cache[2];         // K, V: [Hkv, n_super_cap, kD] words
    const float *ckpt[2];            // [Hkv, n_ckpt_cap, 2, kD]; entry i = state before token (i + 1) * interval
    ParamPtrs p[2];
    float *scratch;                  // [B * Hkv, n_parts, G, kPartStride]
    int Hq, Hkv, rows, n_super_cap, n_ckpt_cap, tokens;
    float scaling, smin, smax;
    bool mute_k;                     // self-test (ADKV_FLAG_SELFTEST_MUTE_K): the K warps do nothing, so the waits behind them run out
};

// How the prefix is laid over CTAs.  The intervals of all units (128 rows of one head) form one line, of which every CTA takes an equal
// piece: whole intervals, so that it can enter anywhere.  A piece that crosses from one unit to the next is two runs.
struct PrefixPlan {
    int n_int, interval, row_tiles, ctas, n_parts;   // intervals of a unit, their tokens; n_parts: room for the parts of a stream
    int each;                                        // CTAs of a unit where no piece crosses from one to the next, else 0
    long long n;                                     // intervals of all units
    __host__ __device__ long long first(int cta) const { return n * cta / ctas; }
    __host__ __device__ int cta_of(long long at) const { return int(((at + 1) * ctas - 1) / n); }
    // first CTA of a unit, and how many have a piece of it
    __host__ __device__ int first_cta(int unit) const { return each ? unit * each : cta_of((long long)unit * n_int); }
    __host__ __device__ int parts(int unit) const { return each ? each : cta_of((long long)unit * n_int + n_int - 1) - first_cta(unit) + 1; }
};

template <int BITS>
struct PrefixShared {
    // values of a tile: [token / 8][channel][token % 8], the rounded ones in the first half and the remainders in the other
    alignas(128) __half k[kPreKV][2 * kPreTok / 8][kD][8];
    alignas(128) __half v[kPreKV][2 * kPreTok / 8][kD][8];
    alignas(128) uint32_t words[2][kPreWords][kPreTok * BITS / 32][kD];   // packed tiles of K and V
    alignas(16) float base[kPreRows];                    // what the zero points of K before the run add to every logit of a row
    // The results of the run lie in k and v, a row every kPartStride floats (no two of eight in the same banks), and the zero points of V
    // before the run in the last row of words, where only their own thread has read.
    __device__ float *row(int r) { return reinterpret_cast<float *>(&k[0][0][0][0]) + r * kPartStride; }
    __device__ float *z0_v() { return reinterpret_cast<float *>(&words[1][kPreWords - 1][kPreTok * BITS / 32 - 1][0]); }
    uint32_t tmem;
    int dead;                                            // a bounded wait gave up
    // of a tile: words are there; K values are there, have been read; V values are there; S is there; weights are there; O is added up (and
    // V and the weights have been read)
    uint64_t loaded[2][kPreWords], kfull[kPreKV], kread[kPreKV], vfull[kPreKV], sdone[kPreP], pfull[kPreP], odone[kPreKV];
};

// K-major shared-memory matrix without swizzle: element (m, k) lies at (m / 8) * m_stride + (k / 8) * k_stride + (m % 8) * 16 + (k % 8) * 2.
__device__ __forceinline__ uint64_t k_major_desc(const void *p, uint32_t k_stride, uint32_t m_stride) { return mn_major_desc(p, k_stride, m_stride); }
// fp16 x fp16 -> fp32, A K-major; B K-major or N-major
__host__ __device__ constexpr uint32_t pre_mma_desc(int M, int N, bool b_mn, bool neg_a = false)
{
    return 1u << 4 | uint32_t(neg_a) << 13 | uint32_t(b_mn) << 16 | uint32_t(N >> 3) << 17 | uint32_t(M >> 4) << 24;
}

// What one thread keeps of its channel, in units of kPreUnit; the zero point counts from the start of the run.
struct PrefixChan {
    float zp, s, alpha, beta, tc;
};
// Eight tokens, fields 0..7 of w, contracted as in k_chunk2; the values go to dst, the remainders behind.  GUARDED: with the eps guard, the clamps and the
// end of the run (left tokens).  Otherwise least and most take in the scale before every fourth token, which tells afterwards whether
// the guards would have done anything.
template <int BITS, bool GUARDED>
__device__ __forceinline__ void prefix_window(uint32_t w, const FieldConsts<BITS> &fc, PrefixChan &c, float smin, float smax, int left, float &least,
                                              float &most, uint8_t *dst)
{
    float x[8];
    if constexpr (GUARDED) {
        static_for<8>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            const float q = fc.template code<j % 4>(j < 4 ? w : w >> (4 * BITS));
            const float rh = __fmul_rn(q, fmaxf(c.s, kEps / kPreUnit));
            x[j] = j < left ? __fadd_rn(rh, c.zp) : 0.f;   // behind the last token: whatever the words hold there does not count
            c.zp = fmaf(c.alpha, rh, c.zp);
            c.s = fminf(fmaxf(c.s * fmaf(c.beta, fabsf(q), c.tc), smin), smax);
        });
    } else {
        // Codes and scale factors of two tokens at a time: they need no state.  With the other products in pairs, too, register moves and
        // reads eat up what that saves: 12.1 cycles a value and scheduler one by one, 10.2 like this, 10.9 and 11.3 with more pairs (bare loop).
        const f32x2 beta2 = pk2(c.beta, c.beta), tc2 = pk2(c.tc, c.tc);
        float s0 = 0.f;
        static_for<4>([&](auto jc) {
            constexpr int j = 2 * decltype(jc)::value, k = j % 4;
            if (j == 0) s0 = c.s;
            if (j == 4) {
                least = fminf(fminf(least, s0), c.s);
                most = fmaxf(fmaxf(most, s0), c.s);
            }
            const uint32_t group = j < 4 ? w : w >> (4 * BITS);
            uint32_t f0, f1;   // FieldConsts::code of fields k and k + 1, before the constant is taken off
            asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(f0) : "r"(group), "n"(Codec<BITS>::FIELD << (BITS * k)), "r"(fc.e[k]));
            asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(f1) : "r"(group), "n"(Codec<BITS>::FIELD << (BITS * (k + 1))), "r"(fc.e[k + 1]));
            const f32x2 q2 = add2(pk2(__uint_as_float(f0), __uint_as_float(f1)), pk2(__uint_as_float(fc.negc[k]), __uint_as_float(fc.negc[k + 1])));
            float q[2], f[2];
            upk2(q2, q[0], q[1]);
            upk2(fma2(beta2, abs2(q2), tc2), f[0], f[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float rh = __fmul_rn(q[i], c.s);
                x[j + i] = __fadd_rn(rh, c.zp);
                c.zp = fmaf(c.alpha, rh, c.zp);
                c.s *= f[i];
            }
        });
    }
    const uint4 hi = make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7]));
    *reinterpret_cast<uint4 *>(dst) = hi;
    *reinterpret_cast<uint4 *>(dst + (kPreTok / 8) * kD * 16) = make_uint4(pack_remainder(hi.x, x[0], x[1]), pack_remainder(hi.y, x[2], x[3]),
                                                                           pack_remainder(hi.z, x[4], x[5]), pack_remainder(hi.w, x[6], x[7]));
}

__device__ __forceinline__ float exp2_fast(float v)   // underflows to zero; the arguments are at most kPreTop + kPreSlack
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ void warp_arrive(uint64_t *bar, int lane, int count = 1)
{
    __syncwarp();
    if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
// A row of results goes to scratch as one copy of its own thread, once that thread's writes can be seen by the copy engine.
__device__ __forceinline__ void bulk_store(void *dst, const void *src, uint32_t bytes)
{
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(__cvta_generic_to_global(dst)), "r"(smem_u32(src)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// a warp's 32 lanes x 32 columns; finished at tmem_wait_ld
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t at)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
                 "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                   "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
                   "=r"(r[31])
                 : "r"(at));
}

template <int BITS>
__global__ void __launch_bounds__(kPreThreads, 2) prefix_kernel(const __grid_constant__ PrefixArgs a, const __grid_constant__ PrefixPlan plan)
{
    extern __shared__ __align__(128) uint8_t smem_raw[];
    PrefixShared<BITS> &sh = *reinterpret_cast<PrefixShared<BITS> *>(smem_raw);
    constexpr int TPW = Codec<BITS>::TPW, WORDS = kPreTok / TPW;                // word rows of a tile
    constexpr uint32_t kColQ = 0, kColS = kD / 2, kColO = kColS + kPreP * kPreTok, kColumns = 256;   // Q; S, with the weights in its place; O
    static_assert(kColO + kD <= kColumns, "columns of tensor memory");
    const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hkv;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the sequences' own tokens may be scanned beside this kernel

    if (threadIdx.x == 0) {
        for (int i = 0; i < kPreWords; ++i) {
            mbar_init(&sh.loaded[0][i], 1);
            mbar_init(&sh.loaded[1][i], 1);
        }
        for (int i = 0; i < kPreKV; ++i) {
            mbar_init(&sh.kfull[i], 4);
            mbar_init(&sh.kread[i], 1);
            mbar_init(&sh.vfull[i], 4);
            mbar_init(&sh.odone[i], 1);
        }
        for (int i = 0; i < kPreP; ++i) {
            mbar_init(&sh.sdone[i], 1);
            mbar_init(&sh.pfull[i], 4);
        }
        sh.dead = 0;
        mbar_init_fence();
    }
    if (warp == 12) tmem_alloc(&sh.tmem, kColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int which = warp >> 2 & 1;   // of the scanning warps: 0 K, 1 V
    const int c = threadIdx.x & (kD - 1);
    const float scale2 = a.scaling * 1.4426950408889634f;
    const int log_g = __ffs(G) - 1;    // 1, 2, 4 or 8 heads
    bool ok = true;
    int done = 0;                      // tiles of the runs so far

    const long long last = plan.first(blockIdx.x + 1);
#pragma unroll 1
    for (long long at = plan.first(blockIdx.x); at < last;) {
        // ------------------------------------------------------------------------------ a run: intervals i0 .. i1 of a unit
        const int unit = int(at / plan.n_int), i0 = int(at % plan.n_int), i1 = int(min((long long)plan.n_int, i0 + last - at));
        at += i1 - i0;
        const int rt = unit % plan.row_tiles, h = unit / plan.row_tiles;
        const int t0 = i0 * plan.interval, ntok = int(min((long long)a.tokens, (long long)i1 * plan.interval)) - t0, n_tiles = (ntok + kPreTok - 1) / kPreTok;
        const int rows = min(kPreRows, a.rows - rt * kPreRows);
        // packed tile i of K or V, by one lane of a warp
        const auto load_tile = [&](int tensor, int i) {
            const int slot = (done + i) % kPreWords, n = min(WORDS, (ntok + TPW - 1) / TPW - i * WORDS);
            uint64_t *bar = &sh.loaded[tensor][slot];
            mbar_expect_tx(bar, n * kD * 4);
            bulk_load(&sh.words[tensor][slot][0][0], a.cache[tensor] + (size_t(h) * a.n_super_cap + t0 / TPW + size_t(i) * WORDS) * kD * 4, n * kD * 4, bar);
        };

        if (warp < 8) {
            // -------------------------------------------------------------------------- K and V values
            FieldConsts<BITS> fc;
            fc.init();
            const ParamPtrs &p = a.p[which];
            const size_t po = size_t(h) * kD + c;
            const float alpha = __half2float(p.alpha[po]), beta = __half2float(p.beta[po]), target = __half2float(p.target[po]);
            float s, start;
            if (i0 > 0) {
                const float *init = a.ckpt[which] + (size_t(h) * a.n_ckpt_cap + i0 - 1) * 2 * kD;
                start = init[c];
                s = init[kD + c];
            } else {
                start = __half2float(p.zp_init[po]);
                s = __half2float(p.scale_init[po]);
            }
            // Scales from which four updates cannot leave the bounds: inside, guards and clamps are the identity.  (SafeRange is the
            // same for eight; of 4-bit caches with the usual parameters 2 % of the windows begin outside that, next to none outside this.)
            const float g0 = 1.f - beta * target, g1 = g0 + beta * float(Codec<BITS>::BIAS), gmn = fminf(fminf(g0, g1), 1.f), gmx = fmaxf(fmaxf(g0, g1), 1.f);
            const float lo = gmn > 0.f ? fmaxf(a.smin, kEps) * (1.f / kPreUnit) / (gmn * gmn * gmn * gmn * (1.f - 2e-5f)) : INFINITY;
            const float hi = a.smax * (1.f / kPreUnit) / (gmx * gmx * gmx * gmx * (1.f + 2e-5f));
            PrefixChan ch{0.f, s * (1.f / kPreUnit), alpha, beta, fmaf(-beta, target, 1.0f)};
            bool tame = true;   // no scale of the warp was outside its interval when last looked at
#pragma unroll 1
            for (int i = which == 0 && a.mute_k ? n_tiles : 0; i < n_tiles; ++i) {
                const int tile = done + i, slot = tile % kPreWords, buf = tile % kPreKV;
                // the words have come, and the products that read this buffer before are done
                uint64_t *freed = tile < kPreKV ? nullptr : which ? &sh.odone[buf] : &sh.kread[buf];
                if (!(ok = mbar_wait_both(&sh.loaded[which][slot], tile / kPreWords & 1, freed, (tile / kPreKV & 1) ^ 1, kStatKWait))) break;
                uint8_t *dst = reinterpret_cast<uint8_t *>(which ? &sh.v[buf][0][c][0] : &sh.k[buf][0][c][0]);
                const uint32_t *row = &sh.words[which][slot][0][c];
                const int left = ntok - i * kPreTok;
                uint32_t w[WORDS];
#pragma unroll
                for (int k = 0; k < WORDS; ++k) w[k] = row[k * kD];
                // Without guards first, which is right if every fourth scale was inside its interval: one vote a tile.  Where it was not the
                // tile is done again with guards, and so are the next ones at once until it is.
                const float zp = ch.zp, s = ch.s;
                bool inside = tame && left >= kPreTok;
                if (inside) {
                    float least = INFINITY, most = -INFINITY;
                    static_for<kPreTok / 8>([&](auto nc) {
                        constexpr int n = decltype(nc)::value;
                        prefix_window<BITS, false>(BITS == 4 ? w[n % WORDS] : w[n / 2 % WORDS] >> (16 * (n & 1)), fc, ch, 0.f, 0.f, 0, least, most, dst + n * kD * 16);
                    });
                    inside = __all_sync(kFull, least >= lo && most <= hi);
                }
                if (!inside) {
                    ch.zp = zp;
                    ch.s = s;
                    float least = INFINITY, most = -INFINITY;
#pragma unroll 1
                    for (int n = 0; n < kPreTok / 8; ++n) {   // rolled: the words move up
                        least = fminf(least, ch.s);
                        most = fmaxf(most, ch.s);
                        prefix_window<BITS, true>(w[0], fc, ch, a.smin * (1.f / kPreUnit), a.smax * (1.f / kPreUnit), left - 8 * n, least, most, dst + n * kD * 16);
                        if (BITS == 2 && !(n & 1)) {
                            w[0] >>= 16;
                        } else {
#pragma unroll
                            for (int k = 0; k + 1 < WORDS; ++k) w[k] = w[k + 1];
                        }
                    }
                    tame = __all_sync(kFull, least >= lo && most <= hi);
                }
                fence_async_shared();
                warp_arrive(which ? &sh.vfull[buf] : &sh.kfull[buf], lane);
            }
            if (which == 1) sh.z0_v()[c] = start;
            if (!ok && lane == 0) sh.dead = 1;
            __syncthreads();
        } else if (warp < 12) {
            // -------------------------------------------------------------------------- weights, a row a thread
            const int e = warp & 3, r = 32 * e + lane;
            const bool busy = 32 * e < rows;
            const uint32_t lanes = tmem + (uint32_t(32 * e) << 16);
            const float f = fmaxf(fabsf(scale2) * kPreUnit, 1e-30f);   // not 0: columns behind the last token are -inf times this
            const int idle = e == 0 ? 4 - (rows + 31) / 32 : 0;        // warps without rows do not take part; the first arrives for them
            float m = -INFINITY, l = 0.f;
            if (busy) {   // the thread's query row, negated where the scaling is negative (rows behind the last one as zeros)
                const uint32_t sign = a.scaling < 0.f ? 0x80008000u : 0u;
                const int n_row = rt * kPreRows + r;
                const uint2 *src = reinterpret_cast<const uint2 *>(a.q + (size_t(n_row >> log_g) * a.Hq + (size_t(h) << log_g) + (n_row & (G - 1))) * kD);
                const __half *z_init = a.p[0].zp_init + size_t(h) * kD;
                const float *z_ckpt = a.ckpt[0] + (size_t(h) * a.n_ckpt_cap + i0 - 1) * 2 * kD;
                float sum[4] = {};
#pragma unroll 1
                for (int n = 0; n < kD / 4; n += 8) {
                    uint2 v[8];
                    float4 z[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = r < rows ? src[n + j] : make_uint2(sign, sign);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (i0 > 0) {
                            z[j] = reinterpret_cast<const float4 *>(z_ckpt)[n + j];
                        } else {
                            const uint2 zh = reinterpret_cast<const uint2 *>(z_init)[n + j];
                            const float2 z0 = __half22float2(*reinterpret_cast<const __half2 *>(&zh.x)), z1 = __half22float2(*reinterpret_cast<const __half2 *>(&zh.y));
                            z[j] = make_float4(z0.x, z0.y, z1.x, z1.y);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        v[j].x ^= sign;
                        v[j].y ^= sign;
                        const float2 q0 = __half22float2(*reinterpret_cast<const __half2 *>(&v[j].x)), q1 = __half22float2(*reinterpret_cast<const __half2 *>(&v[j].y));
                        sum[0] = fmaf(q0.x, z[j].x, sum[0]);
                        sum[1] = fmaf(q0.y, z[j].y, sum[1]);
                        sum[2] = fmaf(q1.x, z[j].z, sum[2]);
                        sum[3] = fmaf(q1.y, z[j].w, sum[3]);
                    }
#pragma unroll
                    for (int j = 0; j < 8; j += 2) tmem_st4(lanes + kColQ + 2 * (n + j), v[j].x, v[j].y, v[j + 1].x, v[j + 1].y);
                }
                sh.base[r] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                tc_fence_before();
            }
            asm volatile("bar.sync 1, 160;" ::: "memory");   // with the warp that issues the products
#pragma unroll 1
            for (int i = 0; i < n_tiles && busy; ++i) {
                const int tile = done + i, buf = tile % kPreP;
                if (!(ok = mbar_wait(&sh.sdone[buf], tile / kPreP & 1, kStatLFullWait))) break;
                tc_fence_after();
                const uint32_t cols = lanes + kColS + kPreTok * buf;
                const int left = ntok - i * kPreTok;
                uint32_t v[kPreTok];
                tmem_ld32(v, cols);
                tmem_wait_ld(v);
                if (left < kPreTok) {
#pragma unroll
                    for (int j = 0; j < kPreTok; ++j) v[j] = j < left ? v[j] : 0xff800000u;
                }
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < kPreTok; j += 2) top = fmaxf(fmaxf(top, __uint_as_float(v[j])), __uint_as_float(v[j + 1]));
                top *= f;
                const bool grown = top > m + (kPreTop + kPreSlack);   // the first tile: m is -inf
                if (__any_sync(kFull, grown)) {
                    const float corr = grown ? exp2_fast(m - (top - kPreTop)) : 1.f;
                    if (i > 0) {
                        // all sums so far are in: O can be changed
                        if (!(ok = mbar_wait(&sh.odone[(tile - 1) % kPreKV], (tile - 1) / kPreKV & 1, kStatVWait))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int n = 0; n < kD; n += 16) {
                            uint32_t o[16];
                            tmem_ld(o, lanes + kColO + n);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
#pragma unroll
                            for (int j = 0; j < 16; j += 4) tmem_st4(lanes + kColO + n + j, o[j], o[j + 1], o[j + 2], o[j + 3]);
                        }
                    }
                    l *= corr;
                    if (grown) m = top - kPreTop;
                }
                float sum[4] = {};
#pragma unroll
                for (int j = 0; j < kPreTok; j += 8) {
                    uint32_t p[4], rest[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float p0 = exp2_fast(fmaf(__uint_as_float(v[j + 2 * k]), f, -m)), p1 = exp2_fast(fmaf(__uint_as_float(v[j + 2 * k + 1]), f, -m));
                        p[k] = pack_half2(p0, p1);
                        rest[k] = pack_remainder(p[k], p0, p1);
                        sum[k] += p0 + p1;
                    }
                    tmem_st4(cols + j / 2, p[0], p[1], p[2], p[3]);
                    tmem_st4(cols + kPreTok / 2 + j / 2, rest[0], rest[1], rest[2], rest[3]);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                tc_fence_before();
                warp_arrive(&sh.pfull[buf], lane, 1 + idle);
            }
            const int end = done + n_tiles - 1;
            if (ok && busy) ok = mbar_wait(&sh.odone[end % kPreKV], end / kPreKV & 1, kStatVWait);
            if (!ok && lane == 0) sh.dead = 1;
            __syncthreads();
            const bool dead = sh.dead != 0;
            if (busy) {
                tc_fence_after();
                const int n_row = rt * kPreRows + r;
                const int slot = blockIdx.x - plan.first_cta(unit);
                float *part = a.scratch + ((size_t(n_row >> log_g) * a.Hkv + h) * plan.n_parts + slot) * (kPartStride << log_g) + (n_row & (G - 1)) * kPartStride;
                float *row = sh.row(r);
                *reinterpret_cast<float4 *>(row) = dead ? make_float4(-INFINITY, __int_as_float(0x7fc00000), 0.f, 0.f)
                                                        : make_float4(fmaf(sh.base[r], fabsf(scale2), m), l, 0.f, 0.f);
#pragma unroll 1
                for (int n = 0; n < kD; n += 32) {
                    uint32_t v[32];
                    tmem_ld32(v, lanes + kColO + n);
                    tmem_wait_ld(v);
#pragma unroll
                    for (int k = 0; k < 32; k += 16) {
                        float4 z[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[j] = *reinterpret_cast<const float4 *>(sh.z0_v() + n + k + 4 * j);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t *o = &v[k + 4 * j];
                            const float4 x = make_float4(fmaf(l, z[j].x, kPreUnit * __uint_as_float(o[0])), fmaf(l, z[j].y, kPreUnit * __uint_as_float(o[1])),
                                                         fmaf(l, z[j].z, kPreUnit * __uint_as_float(o[2])), fmaf(l, z[j].w, kPreUnit * __uint_as_float(o[3])));
                            *reinterpret_cast<float4 *>(row + 4 + n + k + 4 * j) = dead ? make_float4(0.f, 0.f, 0.f, 0.f) : x;
                        }
                    }
                }
                fence_async_shared();
                if (r < rows) {
                    bulk_store(part, row, kPartStride * 4);
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                }
            }
        } else if (warp == 12) {
            // -------------------------------------------------------------------------- S = Q x^T
            constexpr uint32_t hi_desc = pre_mma_desc(kPreRows, kPreTok, true), lo_desc = pre_mma_desc(kPreRows, kPreTok, true, true);
            int i = 0, issued = min(kPreWords, n_tiles);
            if (elect_one())
                for (int k = 0; k < issued; ++k) load_tile(0, k);
            __syncwarp();
            asm volatile("bar.sync 1, 160;" ::: "memory");   // Q is in place
#pragma unroll 1
            for (; i < n_tiles; ++i) {
                const int tile = done + i, slot = tile % kPreKV, buf = tile % kPreP;
                uint64_t *freed = tile >= kPreP ? &sh.odone[(tile - kPreP) % kPreKV] : nullptr;
                if (!(ok = mbar_wait_both(&sh.kfull[slot], tile / kPreKV & 1, freed, max(tile - kPreP, 0) / kPreKV & 1, kStatKWait)))
                    break;   // K is there, the weights in S's place are used
                tc_fence_after();
                if (elect_one()) {
                    if (issued < n_tiles) load_tile(0, issued);   // the words of this tile are read
                    const uint32_t d = tmem + kColS + kPreTok * buf;
                    const uint64_t xd = mn_major_desc(&sh.k[slot][0][0][0], 128, kD * 16);
#pragma unroll
                    for (int n = 0; n < kD / 16; ++n) mma_tmem(d, tmem + kColQ + 8 * n, xd + 16 * n, hi_desc, n > 0);
#pragma unroll
                    for (int n = 0; n < kD / 16; ++n) mma_tmem(d, tmem + kColQ + 8 * n, xd + (kPreTok / 8) * kD + 16 * n, lo_desc, true);
                    mma_commit(&sh.kread[slot]);
                    mma_commit(&sh.sdone[buf]);
                }
                ++issued;
                __syncwarp();
            }
            if (!ok && lane == 0) sh.dead = 1;
            __syncthreads();
            if (sh.dead) {   // products and copies in flight
                for (int k = done + max(i - kPreP, 0); k < done + i; ++k) mbar_wait(&sh.sdone[k % kPreP], k / kPreP & 1, kStatDrain);
                issued = min(issued, n_tiles);
                for (int k = done + max(issued - kPreWords, 0); k < done + issued; ++k) mbar_wait(&sh.loaded[0][k % kPreWords], k / kPreWords & 1, kStatDrain);
            }
        } else {
            // -------------------------------------------------------------------------- O += P y
            constexpr uint32_t hi_desc = pre_mma_desc(kPreRows, kD, false), lo_desc = pre_mma_desc(kPreRows, kD, false, true);
            int i = 0, issued = min(kPreWords, n_tiles);
            if (elect_one())
                for (int k = 0; k < issued; ++k) load_tile(1, k);
            __syncwarp();
#pragma unroll 1
            for (; i < n_tiles; ++i) {
                const int tile = done + i, buf = tile % kPreKV, place = tile % kPreP;
                if (!(ok = mbar_wait(&sh.vfull[buf], tile / kPreKV & 1, kStatVWait))) break;
                if (elect_one() && issued < n_tiles) load_tile(1, issued);
                ++issued;
                __syncwarp();
                if (!(ok = mbar_wait(&sh.pfull[place], tile / kPreP & 1, kStatVWait))) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t pa = tmem + kColS + kPreTok * place;
                    const uint64_t yd = k_major_desc(&sh.v[buf][0][0][0], kD * 16, 128);
#pragma unroll
                    for (int n = 0; n < kPreTok / 16; ++n) {
                        mma_tmem(tmem + kColO, pa + 8 * n, yd + 2 * kD * n, hi_desc, i > 0 || n > 0);
                        mma_tmem(tmem + kColO, pa + 8 * n, yd + (kPreTok / 8) * kD + 2 * kD * n, lo_desc, true);
                        mma_tmem(tmem + kColO, pa + kPreTok / 2 + 8 * n, yd + 2 * kD * n, lo_desc, true);
                    }
                    mma_commit(&sh.odone[buf]);
                }
                __syncwarp();
            }
            if (!ok && lane == 0) sh.dead = 1;
            __syncthreads();
            if (sh.dead) {
                for (int k = done + max(i - kPreKV, 0); k < done + i; ++k) mbar_wait(&sh.odone[k % kPreKV], k / kPreKV & 1, kStatDrain);
                issued = min(issued, n_tiles);
                for (int k = done + max(issued - kPreWords, 0); k < done + issued; ++k) mbar_wait(&sh.loaded[1][k % kPreWords], k / kPreWords & 1, kStatDrain);
            }
        }
        done += n_tiles;
        tc_fence_before();
        fence_async_shared();
        __syncthreads();
        tc_fence_after();
        if (sh.dead) break;   // the runs that are left: their parts are marked below
    }
    if (sh.dead && warp >= 8 && warp < 12) {
        // every part of this CTA makes the results of its rows NaN (the runs that it did not come to have nothing else to say so)
        for (long long at = plan.first(blockIdx.x); at < last; at += plan.n_int - at % plan.n_int) {
            const int unit = int(at / plan.n_int), row = unit % plan.row_tiles * kPreRows + (threadIdx.x & 127), h = unit / plan.row_tiles;
            if (row >= a.rows) continue;
            float *part = a.scratch + ((size_t(row / G * a.Hkv + h) * plan.n_parts + blockIdx.x - plan.first_cta(unit)) * G + row % G) * kPartStride;
            part[0] = -INFINITY;
            part[1] = __int_as_float(0x7fc00000);
        }
    }
    if (warp == 12) tmem_free(tmem, kColumns);
}

// =========================================================================================
// The tokens that a sequence has cached itself, from the state behind the prefix, and the new one: one CTA per stream, as in the fused
// step of adkv_fused.cu.  Its part comes behind those of the prefix's runs.
// Where a row has few parts the kernel adds them up itself, with a part's 128 sums 16 bytes a lane: a launch less, 3 us on the host, which
// bounds small calls, and on the device 14.0 -> 12.9 us for 3 parts, 55.7 -> 51.4 for 4 of eight heads, 47.5 us either way for 8; 17.9 ->
// 18.9 for 8 of four heads, 37.5 -> 40.7 us for 18 of two, so the more are left to the four warps a row of the join.
constexpr int kFoldParts = 8, kFoldLoads = 8;   // kFoldLoads: rows of parts that are under way at once
template <int G, int TOK>
struct OwnSrc : SoftmaxSrc<G, 1, false, TOK> {
    float *part;   // [G][kPartStride]
    int fold;      // parts of the prefix's runs, in front of this one, that are added up here; -1: the join does it
    __device__ __forceinline__ void store(const VArgs &a, int b, int h, int c0, const float (&acc)[G][4]) const
    {
        if (fold >= 0) {
            float m[G], l[G];
            float4 o[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                m[g] = this->m[g];
                l[g] = this->denominator(g);
                o[g] = make_float4(acc[g][0], acc[g][1], acc[g][2], acc[g][3]);
            }
            const float *base = part - size_t(fold) * G * kPartStride;
            asm volatile("griddepcontrol.wait;" ::: "memory");   // the prefix kernel's results
#pragma unroll 1
            for (int j0 = 0; j0 < fold; j0 += kFoldLoads / G) {
                float2 part_ml[kFoldLoads];   // of all heads at once: the rounds of loads are what takes time
                float4 x[kFoldLoads];
#pragma unroll
                for (int u = 0; u < kFoldLoads; ++u) {
                    const float *p = base + (min(j0 + u / G, fold - 1) * G + u % G) * kPartStride;
                    part_ml[u] = *reinterpret_cast<const float2 *>(p);
                    x[u] = *reinterpret_cast<const float4 *>(p + 4 + c0);
                }
#pragma unroll
                for (int u = 0; u < kFoldLoads; ++u) {
                    const int g = u % G;
                    if (j0 + u / G < fold) {
                        const float top = fmaxf(m[g], part_ml[u].x), corr = m[g] == -INFINITY ? 0.f : exp2f(m[g] - top),
                                    w = part_ml[u].x == -INFINITY ? 0.f : exp2f(part_ml[u].x - top);
                        m[g] = top;
                        l[g] = fmaf(part_ml[u].y, w, l[g] * corr);   // a NaN: the part could not be finished
                        o[g].x = fmaf(x[u].x, w, o[g].x * corr);
                        o[g].y = fmaf(x[u].y, w, o[g].y * corr);
                        o[g].z = fmaf(x[u].z, w, o[g].z * corr);
                        o[g].w = fmaf(x[u].w, w, o[g].w * corr);
                    }
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                __half *out = a.out + (size_t(b) * a.Hq + h * G + g) * kD + c0;
                *reinterpret_cast<uint2 *>(out) = make_uint2(pack_half2(o[g].x / l[g], o[g].y / l[g]), pack_half2(o[g].z / l[g], o[g].w / l[g]));
            }
            return;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float l = this->denominator(g);
            if (c0 == 0) *reinterpret_cast<float2 *>(part + g * kPartStride) = make_float2(this->m[g], l);
            *reinterpret_cast<float4 *>(part + g * kPartStride + 4 + c0) = make_float4(acc[g][0], acc[g][1], acc[g][2], acc[g][3]);
        }
    }
    // a bounded wait gave up, or the length did not fit: the result is NaN
    __device__ __forceinline__ void give_up(const VArgs &a, int b, int h, int c0) const
    {
#pragma unroll 1
        for (int g = 0; g < G; ++g) {
            if (fold >= 0) {
                *reinterpret_cast<uint2 *>(a.out + (size_t(b) * a.Hq + h * G + g) * kD + c0) = make_uint2(0x7fff7fffu, 0x7fff7fffu);
                continue;
            }
            if (c0 == 0) *reinterpret_cast<float2 *>(part + g * kPartStride) = make_float2(-INFINITY, __int_as_float(0x7fc00000));
            *reinterpret_cast<float4 *>(part + g * kPartStride + 4 + c0) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
};

// Parts of the prefix's runs that the rows of a sequence have (G divides the rows of a unit: all of its heads lie in one).
__device__ __forceinline__ int prefix_parts(const PrefixPlan &plan, int b, int h, int G)
{
    if (!plan.ctas) return 0;
    return plan.parts(h * plan.row_tiles + b * G / kPreRows);
}

template <int BITS, int G, int TOK>
__global__ void __launch_bounds__(64, G == 8 ? 6 : 10) prefix_own_kernel(KArgs ka, VArgs va, const float *__restrict__ k_state, const float *__restrict__ v_state,
                                                        const int *__restrict__ seq_lens, float scaling, float *__restrict__ scratch,
                                                        const __grid_constant__ PrefixPlan plan, int fold)
{
    constexpr int ST = TOK == 64 ? 2 : 3;   // tiles in flight
    __shared__ alignas(128) uint8_t kbuf[ST * Tile<BITS, TOK>::BYTES];
    __shared__ alignas(128) uint8_t vbuf[ST * Tile<BITS, TOK>::BYTES];
    __shared__ alignas(16) float red[G * 8 * kRedRow];
    __shared__ alignas(16) float2 wts[G * TOK];
    __shared__ FusedShared<G, 1, TOK> fs;
    __shared__ uint64_t kbar[ST], vbar[ST];

    const int bh = blockIdx.x, b = bh / ka.Hkv, h = bh % ka.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    bool fits = true;
    if (seq_lens) {
        ka.T = va.T = seq_lens[b];
        fits = ka.T >= 0 && ka.T / Codec<BITS>::TPW < ka.n_super_cap;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; ++i) { mbar_init(&kbar[i], 1); mbar_init(&vbar[i], 1); }
        fs.init_barriers(1);
        mbar_init_fence();
        if (!fits) atomicExch(&g_status, kStatCapacity);
    }
    __syncthreads();
    const float *init = (warp == 0 ? k_state : v_state) + size_t(h) * 2 * kD;
    const Seg seg{0, ka.T, true, init, nullptr, 0};
    if (warp == 0 && fits) {
        RingSink<G, 1, TOK> sink{&fs, 0, 0};
        k_warp<BITS, G, kArithFma, RingSink<G, 1, TOK>, ST, false, BITS == 4 && G == 1, 8, TOK>(ka, seg, b, h, lane, kbuf, kbar, red, sink);
    } else if (warp == 1) {
        using Src = OwnSrc<G, TOK>;
        Src src;
        src.sh = &fs;
        src.wts = wts;
        src.mask = nullptr;
        src.scale2 = scaling * 1.4426950408889634f;
        src.n_tiles = (ka.T + TOK - 1) / TOK;
        src.t_begin = 0;
        const int n = prefix_parts(plan, b, h, G);
        src.part = scratch + (size_t(bh) * plan.n_parts + n) * G * kPartStride;
        src.fold = fold ? n : -1;
        src.init();
        if (fits) v_warp<BITS, G, kArithFma, Src, ST, false, BITS == 4 && G == 1, TOK>(va, seg, b, h, lane, vbuf, vbar, wts, src);
        else src.give_up(va, b, h, 4 * lane);
    }
    // What waits for this kernel waits for the prefix kernel, too.  One CTA sees to that: the others make room.
    if (blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// out[b, hq] = sum_j x_j 2^(m_j - M) / sum_j l_j 2^(m_j - M) over the parts of a row.  Four warps share a row's parts, a part's 128 sums are
// 16 bytes a lane; all loads of a row are in flight at once, which is what bounds it.
constexpr int kJoinWarps = 4, kJoinLoads = 4;
__global__ void __launch_bounds__(32 * kJoinWarps) prefix_join_kernel(const float *__restrict__ scratch, __half *__restrict__ out, int Hq, int Hkv,
                                                                      const __grid_constant__ PrefixPlan plan)
{
    __shared__ float4 sums[kJoinWarps][32];
    __shared__ float2 ml[kJoinWarps];
    const int b = blockIdx.x / Hq, hq = blockIdx.x % Hq, G = Hq / Hkv, h = hq / G, g = hq % G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = prefix_parts(plan, b, h, G) + 1;
    const float *base = scratch + (size_t(b * Hkv + h) * plan.n_parts * G + g) * kPartStride;
    const size_t stride = size_t(G) * kPartStride;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int j0 = warp; j0 < n; j0 += kJoinWarps * kJoinLoads) {
        float2 part_ml[kJoinLoads];
        float4 x[kJoinLoads];
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u) {
            const float *part = base + size_t(min(j0 + u * kJoinWarps, n - 1)) * stride;
            part_ml[u] = *reinterpret_cast<const float2 *>(part);
            x[u] = *reinterpret_cast<const float4 *>(part + 4 + 4 * lane);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u) top = fmaxf(top, part_ml[u].x);
        const float corr = m == -INFINITY ? 0.f : exp2f(m - top);
        l *= corr;
        o.x *= corr; o.y *= corr; o.z *= corr; o.w *= corr;
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u)
            if (j0 + u * kJoinWarps < n) {
                const float w = part_ml[u].x == -INFINITY ? 0.f : exp2f(part_ml[u].x - top);
                l = fmaf(part_ml[u].y, w, l);   // a NaN: the part could not be finished
                o.x = fmaf(x[u].x, w, o.x);
                o.y = fmaf(x[u].y, w, o.y);
                o.z = fmaf(x[u].z, w, o.z);
                o.w = fmaf(x[u].w, w, o.w);
            }
        m = top;
    }
    sums[warp][lane] = o;
    if (lane == 0) ml[warp] = make_float2(m, l);
    __syncthreads();
    const int c = threadIdx.x;
    float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) M = fmaxf(M, ml[w].x);
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        const float f = ml[w].x == -INFINITY ? 0.f : exp2f(ml[w].x - M);
        L = fmaf(ml[w].y, f, L);
        A = fmaf(reinterpret_cast<const float *>(&sums[w][0])[c], f, A);
    }
    out[size_t(blockIdx.x) * kD + c] = __float2half_rn(A / L);
}

// Two CTAs share an SM, 296 places.  A run costs, besides its tokens, what filling and emptying the pipeline and storing the result take, about
// as long as 300 tokens: so either every unit gets the same number of CTAs, or the line is cut evenly and most CTAs come to have two runs.
// CTAs of own tokens find room on an SM once it has only one of the prefix's.  So a unit gets no more CTAs than its longest run asks for (64
// intervals: eight of eight, not nine of seven or eight): 64 x 32 heads behind 8192 tokens, 128 of their own 86.4 -> 82.8 us, 16 behind 2047,
// 200 47.8 -> 37.0, 32 x 16 of two heads behind 8192, 10 52.7 -> 47.1; without own tokens 128 x 32 heads 74.9 -> 78.6.  Up to 256 streams, which the
// free places can take in, 32 are left free always: 32 x 8 of four heads behind 4700 tokens, 128 of their own 44.5 -> 33.2 us, 30 35.2 -> 30.0, none
// 27.7 -> 29.0; 4 x 32 heads behind 3400 38.9 -> 34.1, 30.7 -> 33.8, 29.6 -> 33.9; with 512 streams, 16 x 32 behind 2300, 38.7 -> 41.2 instead.
static PrefixPlan prefix_plan(int tokens, int interval, int B, int G, int Hkv)
{
    PrefixPlan p{};
    p.row_tiles = int(((long long)B * G + kPreRows - 1) / kPreRows);
    p.n_parts = 1;   // the sequence's own
    if (tokens == 0 || B == 0) return p;
    p.interval = interval > 0 ? interval : tokens;
    p.n_int = int(((long long)tokens + p.interval - 1) / p.interval);
    p.n = (long long)p.n_int * Hkv * p.row_tiles;
    const int units = Hkv * p.row_tiles, places = 2 * kSMs - ((long long)B * Hkv <= 256 ? 32 : 0);
    int each = std::min(places / units, p.n_int);
    if (each) {
        const int longest = (p.n_int + each - 1) / each;
        each = (p.n_int + longest - 1) / longest;
    }
    const long long even = (p.n + places - 1) / places, whole = each ? (p.n_int + each - 1) / each : even;
    p.each = whole * p.interval <= even * p.interval + 300 ? each : 0;
    p.ctas = p.each ? units * each : int(std::min((long long)places, p.n));
    p.n_parts += p.each ? p.each : int((long long)(p.n_int - 1) * p.ctas / p.n) + 2;
    return p;
}

}  // namespace adkv

using namespace adkv;

ADKV_DEFINE_TU_STATUS(adkv_tu_status_prefix)

template <int BITS>
static int launch_prefix(const PrefixArgs &a, const PrefixPlan &plan, cudaStream_t s)
{
    constexpr int bytes = int(sizeof(PrefixShared<BITS>));
    static_assert(2 * (bytes + 1024) <= 228 * 1024, "two CTAs share an SM");
    const auto kernel = prefix_kernel<BITS>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return launch_status();
    kernel<<<plan.ctas, kPreThreads, bytes, s>>>(a, plan);
    return launch_status();
}

// As a programmatic dependent of the launch before it, or, where that is refused, behind it: by then something has run that must not be
// left without its end.
template <class... Params, class... Args>
static int launch_beside(void (*kernel)(Params...), int grid, int block, cudaStream_t s, const Args &...args)
{
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        cudaGetLastError();
        kernel<<<grid, block, 0, s>>>(args...);
    }
    return launch_status();
}

template <int BITS, int G>
static int launch_own(const KArgs &ka, const VArgs &va, const float *k_state, const float *v_state, const int *seq_lens, float scaling,
                      float *scratch, const PrefixPlan &plan, int B, int most, int fold, cudaStream_t s)
{
    // Tiles of 32 tokens where a sequence is short, and with eight query heads, 4-bit, where 64 leave room for fewer CTAs (see short_tiles in
    // adkv_fused.cu).  Whole step behind 64 tokens, 64 -> 32 tokens a tile: 64 x 32 heads, 100 tokens 32.2 -> 31.2 us, 600 81.9 -> 81.9 us; 32 x 8 of four
    // heads, 2-bit, 100 20.5 -> 19.9 us, 600 56.4 -> 60.9 us; 128 x 8 of eight heads 100 49.0 -> 42.4 us, 600 118.9 -> 114.2 us, 1500 243 -> 252 us.
    const auto kernel = most <= (BITS == 4 && G == 8 ? 1000 : 128) ? prefix_own_kernel<BITS, G, 32> : prefix_own_kernel<BITS, G, 64>;
    if (plan.ctas) return launch_beside(kernel, B * ka.Hkv, 64, s, ka, va, k_state, v_state, seq_lens, scaling, scratch, plan, fold);
    kernel<<<B * ka.Hkv, 64, 0, s>>>(ka, va, k_state, v_state, seq_lens, scaling, scratch, plan, fold);
    return launch_status();
}

extern "C" {

long long adkv_decode_attn_prefix_scratch_bytes(int B, int Hq, int Hkv, int prefix_tokens, int interval)
{
    if (B < 0 || Hq <= 0 || Hkv <= 0 || prefix_tokens < 0 || interval < 0 || Hq % Hkv != 0 || (long long)B * Hq > 0x7fffffffll) return ADKV_E_SHAPE;
    const PrefixPlan plan = prefix_plan(prefix_tokens, interval, B, Hq / Hkv, Hkv);
    return (long long)B * Hq * plan.n_parts * kPartStride * (long long)sizeof(float);
}

int adkv_decode_attn_prefix(const void *q, const adkv_prefix *prefix, void *k_cache, void *v_cache, const void *k_new, const void *v_new,
                            const adkv_params *kp, const adkv_params *vp, void *k_tail, void *v_tail, const void *seq_lens, int T, void *out,
                            void *scratch, long long scratch_bytes, int B, int Hq, int Hkv, int D, int n_super_cap, int bits, float scaling,
                            float scale_min, float scale_max, unsigned flags, void *stream)
{
    if (!q || !prefix || !k_cache || !v_cache || !k_new || !v_new || !out || !params_ok(kp) || !params_ok(vp) || !k_tail || !v_tail ||
        !prefix->k_tail || !prefix->v_tail || (prefix->tokens > 0 && (!prefix->k_cache || !prefix->v_cache)))
        return ADKV_E_NULL;
    if (D != kD) return ADKV_E_HEAD_DIM;
    if (seq_lens) T = 0;
    if (int rc = check_common(B, Hq, Hkv, T, D, n_super_cap, bits, T + 1)) return rc;
    const int G = Hq / Hkv;
    if (G != 1 && G != 2 && G != 4 && G != 8) return ADKV_E_SHAPE;
    if (flags & ~unsigned(ADKV_FLAG_TAIL_KEEP | ADKV_FLAG_FAST_REPLAY | ADKV_FLAG_SELFTEST_MUTE_K)) return ADKV_E_FLAGS;
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
    if (rows > (1 << 24) || (long long)B * Hq > 0x7fffffffll) return ADKV_E_SHAPE;
    const long long need = adkv_decode_attn_prefix_scratch_bytes(B, Hq, Hkv, P, iv);
    if (need > 0 && !scratch) return ADKV_E_NULL;
    if (scratch_bytes < need) return ADKV_E_SCRATCH;
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
    pa.n_super_cap = prefix->n_super_cap;
    pa.n_ckpt_cap = prefix->n_ckpt_cap;
    pa.tokens = P;
    pa.scaling = scaling;
    pa.smin = scale_min;
    pa.smax = scale_max;
    pa.mute_k = flags & ADKV_FLAG_SELFTEST_MUTE_K;
    const bool keep = flags & ADKV_FLAG_TAIL_KEEP;
    const KArgs ka{pa.q, static_cast<uint8_t *>(k_cache), static_cast<const __half *>(k_new), pa.p[0], Hq, Hkv, T, n_super_cap, scale_min, scale_max, D,
                   static_cast<float *>(k_tail), keep};
    const VArgs va{static_cast<uint8_t *>(v_cache), static_cast<const __half *>(v_new), static_cast<__half *>(out), pa.p[1], Hq, Hkv, T, n_super_cap,
                   scale_min, scale_max, D, static_cast<float *>(v_tail), keep};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const PrefixPlan plan = prefix_plan(P, iv, B, G, Hkv);
    if (plan.ctas)
        if (int rc = bits == 4 ? launch_prefix<4>(pa, plan, s) : launch_prefix<2>(pa, plan, s)) return rc;
    const int most = seq_lens ? int(std::min((long long)n_super_cap * (32 / bits), 1ll << 30)) : T;   // own tokens of a sequence, at most
    const int fold = plan.n_parts - 1 <= kFoldParts;
    int rc = 0;
    ADKV_DISPATCH_H(bits, G, (rc = launch_own<BITS, G>(ka, va, static_cast<const float *>(prefix->k_tail), static_cast<const float *>(prefix->v_tail),
                                                         static_cast<const int *>(seq_lens), scaling, pa.scratch, plan, B, most, fold, s)))
    if (rc || fold) return rc;
    return launch_beside(prefix_join_kernel, B * Hq, 32 * kJoinWarps, s, pa.scratch, static_cast<__half *>(out), Hq, Hkv, plan);
}

}  // extern "C"
