// Part of libadkv_b200.so (sm_100a).  See include/adkv_b200.h for the contract of every entry point.
//
// What a decode or prefill step does around the attention kernels: the rotation (and normalisation per head) of queries and keys
// between the projection and the cache, and the penalties, biases and masks on the logits with the choice of the next token.
#include "adkv_host.h"

#include <cuda_bf16.h>

#include <algorithm>

namespace adkv {

constexpr int kStatPosition = 8;   // a position held on the device lies outside the rotation tables

// Four consecutive elements of a row as they lie in memory, and as floats.
template <class T>
struct Four;
template <>
struct Four<__half> {
    using Raw = uint2;
    __device__ static void get(float (&v)[4], const uint2 &a)
    {
        const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&a.x)), hi = __half22float2(*reinterpret_cast<const __half2 *>(&a.y));
        v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
    }
    __device__ static uint2 put(const float (&v)[4])
    {
        const __half2 lo = __floats2half2_rn(v[0], v[1]), hi = __floats2half2_rn(v[2], v[3]);
        return make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    }
};
template <>
struct Four<__nv_bfloat16> {
    using Raw = uint2;
    __device__ static void get(float (&v)[4], const uint2 &a)
    {
        v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
        v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
    }
    __device__ static uint2 put(const float (&v)[4])
    {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
        return make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    }
};
template <>
struct Four<float> {
    using Raw = float4;
    __device__ static void get(float (&v)[4], const float4 &a) { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; }
    __device__ static float4 put(const float (&v)[4]) { return make_float4(v[0], v[1], v[2], v[3]); }
};

// =========================================================================================
// Rotation of queries and keys, with the root-mean-square norm of each head before it:
//   y = x / sqrt(mean(x^2) + eps) * w          (w given)
//   (a, b) -> (a cos - b sin, b cos + a sin)   for the rot / 2 pairs of channels: (i, i + rot / 2), or (2i, 2i + 1) interleaved
// in fp32, one rounding at the end; products and sums of the rotation are rounded one by one, as the torch expression in e2e_llama
// does.  Values pass through, so that all of [B, T, (Hq + 2 Hkv) D] leaves in the [B, H, T, D] layout that the caches take.
//
// Every element is read and written once, the tables are 1 % of it: 8191 tokens of 48 heads of 128 take 39.7 us, 0.79 of the rate of a copy,
// 16 x 777 tokens of 48 heads of 256 102.6 us, 0.91 (replayed from a graph; called one after another 41 to 45 and 109 to 115).  128 single
// tokens take 3.0 us, a launch and a round trip.  fp32 in, 8191 x 48 x 128: 51 us to fp16, 0.90, 74 us to fp32, 0.83.  A lane holds eight or
// sixteen channels of a head, in pairs of groups of four, so that both halves of a pair are its own and nothing but the sum of squares
// crosses lanes; a thread takes the same channels of up to kRopeRows heads of one token, so cosines and sines are loaded once for them.
// A CTA goes on from token to token, and the next two are on their way to shared memory while it works on one: with a token a CTA, half
// of the time nothing is.  Every thread reads what it has copied itself, so nothing has to be waited for but its own copies, and CTAs are
// as small as they may be for the registers to hold many tokens: 256 threads and eight channels a lane 44.0 and 120 us, and with sixteen 43.6
// and 115, 128 threads 45.9 and 102; of 64 threads with one head each 44.2 and 119, with three 45.8 and 120, 32 threads 40.5 and 103, four
// tokens on their way 45.7 and 117.
struct RopeArgs {
    const void *qkv;
    long long stride_b, stride_t;      // elements
    void *q, *k, *v;
    const void *q_weight, *k_weight;   // [D] in the input's type, or nullptr
    const float *cos, *sin;            // [table_rows, >= rot / 2]
    const int *positions;              // [B] (per_token false: of the first token) or [B, T], or nullptr
    long long table_stride;
    int table_rows, rot, per_token, start, tokens, T, Hq, Hkv, interleaved;
    int rows;                          // heads of a thread, at most kRopeRows
    float eps;
};
constexpr int kRopeThreads = 64, kRopeRows = 2;
constexpr int kRopeCtas = 12;            // of an SM
template <int D>
__host__ __device__ constexpr int rope_units() { return D >= 128 ? 2 : 1; }   // groups of eight channels of a lane

template <int D, class In>
__host__ __device__ constexpr int rope_slot_bytes() { return kRopeRows * rope_units<D>() * 2 * kRopeThreads * int(sizeof(typename Four<In>::Raw)); }   // of a stage
template <int D, class In>
__host__ __device__ constexpr int rope_stages() { return rope_slot_bytes<D, In>() > 4096 ? 2 : 3; }   // so that all CTAs find room
__device__ __forceinline__ void copy_async(uint2 *dst, const void *src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(__cvta_generic_to_global(src)) : "memory"); }
__device__ __forceinline__ void copy_async(float4 *dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(__cvta_generic_to_global(src)) : "memory"); }

template <int D, class In, class Out>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas) norm_rope_kernel(const __grid_constant__ RopeArgs a)
{
    constexpr int UNITS = rope_units<D>(), LANES = D / 8 / UNITS;   // LANES: of a head
    constexpr int HEADS = kRopeThreads / LANES;                      // heads that the CTA takes side by side
    using Raw = typename Four<In>::Raw;
    const int lane = threadIdx.x % LANES, H = a.Hq + 2 * a.Hkv, half = a.rot / 2;
    const int h0 = blockIdx.y * HEADS * a.rows + threadIdx.x / LANES;

    // first channels of the lane's two groups of four: pairs (first, second), or channels that are left as they are
    int at0[UNITS], at1[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int pair = 4 * (lane + LANES * u);
        const bool split = pair < half && !a.interleaved;
        at0[u] = split ? pair : 2 * pair;
        at1[u] = split ? pair + half : 2 * pair + 4;
    }
    constexpr int ST = rope_stages<D, In>();
    extern __shared__ __align__(16) uint8_t rope_smem[];
    // stage, row, group of the lane's channels, half: the thread's own slot
    const auto slot = [&](int st, int r, int u, int k) {
        return reinterpret_cast<Raw *>(rope_smem) + (((st * kRopeRows + r) * UNITS + u) * 2 + k) * kRopeThreads + threadIdx.x;
    };
    // a token as its sequence and its place there, and the step from one of the CTA's tokens to the next
    struct Place {
        int b, t;
    };
    const int step_b = int(gridDim.x) / a.T, step_t = int(gridDim.x) % a.T;
    const auto advance = [&](Place &p) {
        p.b += step_b;
        p.t += step_t;
        if (p.t >= a.T) { p.t -= a.T; ++p.b; }
    };
    const int B = a.tokens / a.T;
    const auto load = [&](const Place &p, int st) {
        if (p.b < B) {
            const In *src = static_cast<const In *>(a.qkv) + p.b * a.stride_b + p.t * a.stride_t + h0 * D;
#pragma unroll
            for (int r = 0; r < kRopeRows; ++r) {
                if (r >= a.rows || h0 + HEADS * r >= H) break;
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    copy_async(slot(st, r, u, 0), src + HEADS * r * D + at0[u]);
                    copy_async(slot(st, r, u, 1), src + HEADS * r * D + at1[u]);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const bool q_norm = a.q_weight, k_norm = a.k_weight, whole = a.table_stride % 4 == 0 && a.rot % 8 == 0 &&
               ((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) & 15) == 0;   // cosines and sines four at a time
    Raw weight[2][UNITS][2] = {};   // of queries and keys
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        if (q_norm) {
            weight[0][u][0] = *reinterpret_cast<const Raw *>(static_cast<const In *>(a.q_weight) + at0[u]);
            weight[0][u][1] = *reinterpret_cast<const Raw *>(static_cast<const In *>(a.q_weight) + at1[u]);
        }
        if (k_norm) {
            weight[1][u][0] = *reinterpret_cast<const Raw *>(static_cast<const In *>(a.k_weight) + at0[u]);
            weight[1][u][1] = *reinterpret_cast<const Raw *>(static_cast<const In *>(a.k_weight) + at1[u]);
        }
    }
    const auto finish = [&](const Place &p, int st) {
        int pos = a.start + p.t;
        if (a.positions) pos = a.per_token ? a.positions[p.b * a.T + p.t] : int(uint32_t(a.positions[p.b]) + uint32_t(p.t));   // behind the largest int: negative
        float c[UNITS][4], s[UNITS][4];
        bool turns[UNITS];   // channels behind the rotated ones are copied (0 times an infinite neighbour is not 0); without a position all are NaN
        const bool inside = pos >= 0 && pos < a.table_rows;
        if (!inside && threadIdx.x == 0 && blockIdx.y == 0) atomicExch(&g_status, kStatPosition);
        const float *cos = a.cos + (long long)pos * a.table_stride, *sin = a.sin + (long long)pos * a.table_stride;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int pair = 4 * (lane + LANES * u);
            turns[u] = pair < half || !inside;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[u][i] = inside ? 1.f : __int_as_float(0x7fc00000);
                s[u][i] = 0.f;
            }
            if (inside && pair < half) {
                if (whole) {
                    Four<float>::get(c[u], *reinterpret_cast<const float4 *>(cos + pair));
                    Four<float>::get(s[u], *reinterpret_cast<const float4 *>(sin + pair));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        c[u][i] = cos[pair + i];
                        s[u][i] = sin[pair + i];
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kRopeRows; ++r) {
            if (r >= a.rows) break;
            const int h = h0 + HEADS * r;
            const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
            float x[UNITS][2][4];   // of lanes behind the last head: whatever the slot holds, not used
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                Four<In>::get(x[u][0], *slot(st, r, u, 0));
                Four<In>::get(x[u][1], *slot(st, r, u, 1));
            }
            if (q_norm || k_norm) {   // the same for all: the lanes of other heads take part in the sum
                float sum = 0.f;
#pragma unroll
                for (int u = 0; u < UNITS; ++u)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum = fmaf(x[u][i / 4][i % 4], x[u][i / 4][i % 4], sum);
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
                if (!is_v && (is_q ? q_norm : k_norm)) {
                    const float inv = rsqrtf(sum * (1.f / D) + a.eps);
#pragma unroll
                    for (int u = 0; u < UNITS; ++u)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float w[4];
                            Four<In>::get(w, is_q ? weight[0][u][k] : weight[1][u][k]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[u][k][i] *= inv * w[i];
                        }
                }
            }
            if (h >= H) continue;
            // heads of the tensor and the head in it
            const int n = is_q ? a.Hq : a.Hkv, at = is_q ? h : is_v ? h - a.Hq - a.Hkv : h - a.Hq;
            Out *dst = static_cast<Out *>(is_q ? a.q : is_v ? a.v : a.k) + ((size_t(p.b) * n + at) * a.T + p.t) * D;
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                float(&p)[4] = x[u][0], (&n)[4] = x[u][1];
                const auto turn = [](float &first, float &second, float co, float si) {
                    const float was = first;
                    first = __fsub_rn(__fmul_rn(was, co), __fmul_rn(second, si));
                    second = __fadd_rn(__fmul_rn(second, co), __fmul_rn(was, si));
                };
                if (!is_v && turns[u]) {
                    if (a.interleaved) {
                        turn(p[0], p[1], c[u][0], s[u][0]); turn(p[2], p[3], c[u][1], s[u][1]);
                        turn(n[0], n[1], c[u][2], s[u][2]); turn(n[2], n[3], c[u][3], s[u][3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) turn(p[i], n[i], c[u][i], s[u][i]);
                    }
                }
                using OutRaw = typename Four<Out>::Raw;
                *reinterpret_cast<OutRaw *>(dst + at0[u]) = Four<Out>::put(p);
                *reinterpret_cast<OutRaw *>(dst + at1[u]) = Four<Out>::put(n);
            }
        }
    };
    Place now{int(blockIdx.x) / a.T, int(blockIdx.x) % a.T}, ahead = now;
    int st = 0;
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) {
        load(ahead, k);
        advance(ahead);
    }
#pragma unroll 1
    for (; now.b < B; advance(now)) {
        load(ahead, (st + ST - 1) % ST);
        advance(ahead);
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        finish(now, st);
        st = st + 1 == ST ? 0 : st + 1;
    }
}

// =========================================================================================
// Logits of a row, in fp32 and rounded once at the end:
//   n = how often the token is in the row's history;  if n > 0:  x = x > 0 ? x / repetition : x * repetition,
//   x = x - (frequency * n + presence);   then x + bias, and -inf where the mask's bit is not set.
// The token is the lowest index of the largest result (a NaN counts as larger than anything), -1 where all are -inf.
//
// One row is bound by latency (5.2 us for 32000 tokens: launch, history, cluster barrier).  64 rows of 128256 bf16 logits with bias, mask and
// 4000 tokens of history take 20.0 us, their bytes 5.4: 3 us until the history is counted, 5.5 for the penalties, which nearly every warp
// has to do for some lane, and 9 for the rest, which is as much issue as it is 84 MB through L2 (a bias is four bytes a token and row).
// A cluster of up to eight CTAs shares a row; each counts the history's tokens
// that fall into its part in shared memory (integer additions, so the order does not matter) and then passes over its part once, 16
// aligned bytes a load whatever the row's alignment.  The first loads are under way while the history is counted.  The CTAs' largest
// values meet in the shared memory of the first, so nothing has to be cleared, kept or launched besides.
struct LogitArgs {
    const void *x;
    void *out;
    int *tokens;                                             // [B] or nullptr
    const int *history, *history_lens;                       // [B, history_cap], [B] (nullptr: all of it)
    const float *repetition, *presence, *frequency;          // [B], or nullptr: the number beside it
    float repetition1, presence1, frequency1;
    const float *bias;                                       // [V] (stride 0) or [B, V], or nullptr
    const uint32_t *mask;                                    // [B, >= (V + 31) / 32], or nullptr
    long long stride_x, stride_out, stride_history, stride_bias, stride_mask;
    int V, history_cap;
    int part;                                                // packs of a CTA, a multiple of 32, see below
};
constexpr int kLogitThreads = 512, kLogitCluster = 8, kLogitAhead = 4;   // kLogitAhead: loads of a thread that are under way at once
constexpr int kLogitBytes = 73728;                                       // of counts

template <class T>
struct LogitIo;
template <>
struct LogitIo<float> {
    static constexpr int N = 4;
    __device__ static float load(const float *p) { return *p; }
    __device__ static void unpack(const uint4 &v, float (&x)[4])
    {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    __device__ static uint4 pack(const float (&x)[4])
    {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    __device__ static float round(float v) { return v; }
    __device__ static void store(float *p, float v) { *p = v; }
};
template <>
struct LogitIo<__half> {
    static constexpr int N = 8;
    __device__ static float load(const __half *p) { return __half2float(*p); }
    __device__ static void unpack(const uint4 &v, float (&x)[8])
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
    __device__ static uint4 pack(const float (&x)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static float round(float v) { return __half2float(__float2half_rn(v)); }
    __device__ static void store(__half *p, float v) { *p = __float2half_rn(v); }
};
template <>
struct LogitIo<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ static float load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
    __device__ static void unpack(const uint4 &v, float (&x)[8])
    {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ static uint4 pack(const float (&x)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static float round(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
    __device__ static void store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
};

// Value and index as one number whose order is that of the choice: larger values first (NaN above all, -0 as +0), then lower indexes.
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t u = __float_as_uint(v + 0.f);
    return v != v ? 0xffffffffu : (u >> 31 ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long rank_of(float v, int index) { return (unsigned long long)key_of(v) << 32 | uint32_t(~index); }
constexpr uint32_t kRankMinusInf = 0x007fffffu;   // key of -inf

__device__ __forceinline__ float max_or_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A pack: the elements of 16 aligned bytes of the row.  A row that starts `skew` elements behind such a boundary has elements
// p * N - skew ... of pack p; of the first and the last one some lie outside.  Count: what an occurrence is counted in, 16 bits where a
// history is short enough for it.
template <class T, class Count>
__global__ void __launch_bounds__(kLogitThreads, 2) process_logits_kernel(const __grid_constant__ LogitArgs a)
{
    using Io = LogitIo<T>;
    constexpr int N = Io::N, PER = 4 / int(sizeof(Count));   // counts in a word
    extern __shared__ __align__(16) uint32_t counts[];
    __shared__ unsigned long long best[kLogitThreads / 32], gathered[kLogitCluster];
    uint32_t rank, ranks;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // that all CTAs of the cluster run is waited for below

    const int b = blockIdx.y;
    const T *x = static_cast<const T *>(a.x) + b * a.stride_x;
    T *out = static_cast<T *>(a.out) + b * a.stride_out;
    const float *bias = a.bias ? a.bias + b * a.stride_bias : nullptr;
    const uint32_t *mask = a.mask ? a.mask + b * a.stride_mask : nullptr;
    const int n_words = (a.V + 31) / 32;
    const int skew = int(reinterpret_cast<uintptr_t>(x) / sizeof(T) % N);
    const bool same = int(reinterpret_cast<uintptr_t>(out) / sizeof(T) % N) == skew;   // else the results are stored one by one
    const bool bias4 = (reinterpret_cast<uintptr_t>(bias) / 4 - skew) % 4 == 0;        // four biases a load
    const int packs = (a.V + skew + N - 1) / N;
    // A row's packs are dealt out 32 at a time, so that every CTA of the cluster gets its share of the frequent tokens, which have the
    // low numbers.  Its l-th pack is number
    const int log_ranks = __ffs(ranks) - 1;
    const auto pack_of = [&](int l) { return ((l >> 5 << log_ranks | int(rank)) << 5) | (l & 31); };
    const float rep = a.repetition ? a.repetition[b] : a.repetition1, pres = a.presence ? a.presence[b] : a.presence1,
                freq = a.frequency ? a.frequency[b] : a.frequency1;
    const int *history = a.history ? a.history + b * a.stride_history : nullptr;
    const int first_id = history && int(threadIdx.x) < a.history_cap ? history[threadIdx.x] : -1;
    const int n_history = !history ? 0 : a.history_lens ? min(max(a.history_lens[b], 0), a.history_cap) : a.history_cap;

    const auto whole = [&](int p) { return p * N >= skew && p * N - skew + N <= a.V; };   // all of a pack lies in the row
    uint32_t top_key = 0;
    int top_at = a.V;
    uint4 top_pack = make_uint4(0, 0, 0, 0);
    // Pack p of the row, the at-th of those that are counted; raw: what it holds, if all of it lies in the row.
    const auto work = [&](auto whole_pack, int p, int at, const uint4 &raw) {
        const int v = p * N - skew;                    // index of the pack's first element
        constexpr bool all = decltype(whole_pack)::value;
        float y[N];
        if constexpr (all) {
            Io::unpack(raw, y);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = v + i >= 0 && v + i < a.V ? Io::load(x + v + i) : 0.f;
        }
        if (n_history) {
            uint32_t w[N / PER], any = 0;
#pragma unroll
            for (int i = 0; i < N / PER; ++i) w[i] = 0;
            if constexpr (N / PER >= 4) {
#pragma unroll
                for (int i = 0; i < N / PER; i += 4) {
                    const uint4 c = *reinterpret_cast<const uint4 *>(counts + at * (N / PER) + i);
                    w[i] = c.x; w[i + 1] = c.y; w[i + 2] = c.z; w[i + 3] = c.w;
                }
            } else {
                const uint2 c = *reinterpret_cast<const uint2 *>(counts + at * (N / PER));
                w[0] = c.x; w[1] = c.y;
            }
#pragma unroll
            for (int i = 0; i < N / PER; ++i) any |= w[i];
            if (any) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t n = PER == 1 ? w[i / PER] : w[i / PER] >> (i % PER * 16) & 0xffffu;
                    if (n) {
                        const float z = y[i] > 0.f ? __fdiv_rn(y[i], rep) : __fmul_rn(y[i], rep);
                        y[i] = __fsub_rn(z, __fadd_rn(__fmul_rn(freq, float(n)), pres));
                    }
                }
            }
        }
        if (bias) {
            if (all && bias4) {
#pragma unroll
                for (int i = 0; i < N; i += 4) {
                    const float4 z = *reinterpret_cast<const float4 *>(bias + v + i);
                    y[i] = __fadd_rn(y[i], z.x); y[i + 1] = __fadd_rn(y[i + 1], z.y);
                    y[i + 2] = __fadd_rn(y[i + 2], z.z); y[i + 3] = __fadd_rn(y[i + 3], z.w);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (all || (v + i >= 0 && v + i < a.V)) y[i] = __fadd_rn(y[i], bias[v + i]);
            }
        }
        if (mask) {
            const int first = max(v, 0);
            const uint32_t w0 = mask[first >> 5], w1 = mask[min((first >> 5) + 1, n_words - 1)];
            const uint32_t bits = __funnelshift_r(w0, w1, first & 31) << (first - v);
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (!(bits >> i & 1)) y[i] = -INFINITY;
        }
        const uint4 packed = Io::pack(y);
        if (all && same) {
            *reinterpret_cast<uint4 *>(out + v) = packed;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (v + i >= 0 && v + i < a.V) Io::store(out + v + i, y[i]);
        }
        if (a.tokens) {   // the pack with the largest element so far, the first of them
            Io::unpack(packed, y);   // as they have been rounded
            if (!all) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (v + i < 0 || v + i >= a.V) y[i] = -INFINITY;
            }
            float most = y[0];
#pragma unroll
            for (int i = 1; i < N; ++i) most = max_or_nan(most, y[i]);
            const uint32_t key = key_of(most);
            if (key > top_key || (key == top_key && v < top_at)) {
                top_key = key;
                top_at = v;
                top_pack = packed;
            }
        }
    };
    constexpr int kPacks = kLogitBytes / int(sizeof(Count)) / N;
    for (int p0 = 0; p0 < a.part; p0 += kPacks) {
        const int p1 = min(a.part, p0 + kPacks);
        uint4 ahead[kLogitAhead];
        const auto fetch = [&](int l) {
#pragma unroll
            for (int u = 0; u < kLogitAhead; ++u) {
                const int q = pack_of(l + u * kLogitThreads);
                ahead[u] = l + u * kLogitThreads < p1 && whole(q) ? *reinterpret_cast<const uint4 *>(x + (q * N - skew)) : make_uint4(0, 0, 0, 0);
            }
        };
        fetch(p0 + threadIdx.x);
        if (history) {   // cleared before the length is known, which is on its way with the first ids
            int id = first_id;
            for (int i = threadIdx.x; i < ((p1 - p0) * N / PER + 3) / 4; i += kLogitThreads) reinterpret_cast<uint4 *>(counts)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
#pragma unroll 8
            for (int i = threadIdx.x; i < n_history; i += kLogitThreads) {
                if (i >= kLogitThreads) id = history[i];
                const uint32_t e = uint32_t(id) + uint32_t(skew), group = e / (32 * N);
                const int l = int(group >> log_ranks << 5 | (e / N & 31)) - p0;   // the CTA's pack that holds it, if it is the CTA's
                if (id >= 0 && id < a.V && (group & (ranks - 1)) == rank && l >= 0 && l < p1 - p0) {
                    const uint32_t at = uint32_t(l) * N + e % N;
                    atomicAdd(&counts[at / PER], 1u << (at % PER * 16));
                }
            }
            __syncthreads();
        }
        for (int base = p0 + threadIdx.x; base < p1; base += kLogitAhead * kLogitThreads) {
            if (base >= p0 + kLogitAhead * kLogitThreads) fetch(base);
#pragma unroll
            for (int u = 0; u < kLogitAhead; ++u) {
                const int l = base + u * kLogitThreads, p = pack_of(l);
                if (l >= p1 || p >= packs) break;
                if (whole(p)) work(std::true_type{}, p, l - p0, ahead[u]);
            }
        }
        // the first and the last pack of the row, where some of their elements lie outside
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            const int p = k ? packs - 1 : 0, group = p >> 5, l = group >> log_ranks << 5 | (p & 31);
            if (whole(p) || (k && packs == 1) || (group & int(ranks - 1)) != int(rank) || l < p0 || l >= p1) continue;
            if (int(threadIdx.x) == (l - p0) % kLogitThreads) work(std::false_type{}, p, l - p0, make_uint4(0, 0, 0, 0));
        }
        __syncthreads();   // the counts are read
    }
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (!a.tokens) return;
    unsigned long long top = 0;
    {
        float y[N];
        Io::unpack(top_pack, y);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (top_at + i >= 0 && top_at + i < a.V) top = max(top, rank_of(y[i], top_at + i));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(kFull, top, o));
    if (threadIdx.x % 32 == 0) best[threadIdx.x / 32] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kLogitThreads / 32; ++i) top = max(top, best[i]);
        uint32_t there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(smem_u32(&gathered[rank])));
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(there), "l"(top) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && threadIdx.x == 0) {
        for (uint32_t i = 0; i < ranks; ++i) top = max(top, gathered[i]);
        a.tokens[b] = uint32_t(top >> 32) <= kRankMinusInf ? -1 : int(~uint32_t(top));
    }
}

}  // namespace adkv

using namespace adkv;

ADKV_DEFINE_TU_STATUS(adkv_tu_status_step)

template <int D, class In, class Out>
static int launch_rope_kernel(RopeArgs a, cudaStream_t s)
{
    constexpr int bytes = rope_stages<D, In>() * rope_slot_bytes<D, In>(), heads = kRopeThreads / (D / 8 / rope_units<D>());
    static_assert(bytes <= 48 * 1024, "");
    constexpr long long places = kSMs * std::min(kRopeCtas, 227 * 1024 / (bytes + 1024));   // CTAs that the chip holds
    const int each = (a.Hq + 2 * a.Hkv + heads - 1) / heads, groups = (each + kRopeRows - 1) / kRopeRows;
    a.rows = (each + groups - 1) / groups;
    const dim3 grid(std::min((long long)a.tokens, std::max(1ll, places / groups)), groups);
    norm_rope_kernel<D, In, Out><<<grid, kRopeThreads, bytes, s>>>(a);
    return launch_status();
}

template <int D>
static int launch_rope(const RopeArgs &a, int in_type, int out_type, cudaStream_t s)
{
    switch (in_type * 4 + out_type) {
    case ADKV_T_F16 * 4 + ADKV_T_F16: return launch_rope_kernel<D, __half, __half>(a, s);
    case ADKV_T_BF16 * 4 + ADKV_T_F16: return launch_rope_kernel<D, __nv_bfloat16, __half>(a, s);
    case ADKV_T_BF16 * 4 + ADKV_T_BF16: return launch_rope_kernel<D, __nv_bfloat16, __nv_bfloat16>(a, s);
    case ADKV_T_F32 * 4 + ADKV_T_F16: return launch_rope_kernel<D, float, __half>(a, s);
    case ADKV_T_F32 * 4 + ADKV_T_F32: return launch_rope_kernel<D, float, float>(a, s);
    default: return ADKV_E_TYPE;
    }
}

static bool aligned_to(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <class T, class Count>
static int launch_logits_kernel(LogitArgs a, int B, cudaStream_t s)
{
    constexpr int N = LogitIo<T>::N, room = kLogitBytes / int(sizeof(Count));   // tokens that can be counted at once
    // CTAs of a row: more while the chip holds them all at once, two an SM, and each has 2048 elements, and while a CTA's part of a row
    // with a history is more than it can count at once
    int cluster = 1;
    while (cluster < kLogitCluster && 2ll * B * cluster <= 2 * kSMs && a.V / (2 * cluster) >= 2048) cluster *= 2;
    while (cluster < kLogitCluster && a.history && a.V / cluster > room) cluster *= 2;
    const int packs = (a.V + 2 * N - 2) / N;   // of the worst alignment
    a.part = ((packs + 31) / 32 + cluster - 1) / cluster * 32;
    const int bytes = a.history ? std::min((a.part * N * int(sizeof(Count)) + 15) / 16 * 16, kLogitBytes) : 0;
    const auto kernel = process_logits_kernel<T, Count>;
    if (bytes > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLogitBytes) != cudaSuccess)
        return launch_status();
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(cluster, B);
    cfg.blockDim = dim3(kLogitThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) return launch_status();
    return launch_status();
}
template <class T>
static int launch_logits(const LogitArgs &a, int B, cudaStream_t s)
{
    return a.history_cap > 65535 ? launch_logits_kernel<T, uint32_t>(a, B, s) : launch_logits_kernel<T, uint16_t>(a, B, s);
}

extern "C" {

int adkv_norm_rope_qkv(const void *qkv, long long stride_b, long long stride_t, int in_type, void *q, void *k, void *v, int out_type,
                       const void *q_weight, const void *k_weight, float eps, const void *cos, const void *sin, long long table_stride,
                       int table_rows, int rot, const void *positions, int positions_per_token, int start, int B, int T, int Hq, int Hkv,
                       int D, int interleaved, void *stream)
{
    if (!qkv || !q || !k || !v || !cos || !sin) return ADKV_E_NULL;
    if (D != 64 && D != 128 && D != 256 && D != 512) return ADKV_E_HEAD_DIM;
    if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || rot <= 0 || rot > D || rot % 8 || table_rows < 0 || start < 0 || stride_b % 4 || stride_t % 4 ||
        (long long)B * T > 0x7fffffffll)
        return ADKV_E_SHAPE;
    if (in_type < ADKV_T_F16 || in_type > ADKV_T_F32 || (out_type != in_type && out_type != ADKV_T_F16)) return ADKV_E_TYPE;
    const unsigned in4 = in_type == ADKV_T_F32 ? 16 : 8, out4 = out_type == ADKV_T_F32 ? 16 : 8;
    if (!aligned_to(qkv, in4) || !aligned_to(q_weight, in4) || !aligned_to(k_weight, in4) || !aligned_to(q, out4) || !aligned_to(k, out4) ||
        !aligned_to(v, out4) || !aligned_to(cos, 4) || !aligned_to(sin, 4) || !aligned_to(positions, 4))
        return ADKV_E_ALIGN;
    if (!positions && B && T && (long long)start + T > table_rows) return ADKV_E_CAPACITY;
    if (B == 0 || T == 0) return 0;
    const RopeArgs a{qkv, stride_b, stride_t, q, k, v, q_weight, k_weight, static_cast<const float *>(cos), static_cast<const float *>(sin),
                     static_cast<const int *>(positions), table_stride, table_rows, rot, positions_per_token, start, B * T, T, Hq, Hkv, interleaved, 0, eps};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (D) {
    case 64: return launch_rope<64>(a, in_type, out_type, s);
    case 128: return launch_rope<128>(a, in_type, out_type, s);
    case 256: return launch_rope<256>(a, in_type, out_type, s);
    default: return launch_rope<512>(a, in_type, out_type, s);
    }
}

int adkv_process_logits(const void *x, long long stride_x, void *out, long long stride_out, int type, void *tokens, const void *history,
                        long long stride_history, int history_cap, const void *history_lens, const void *repetition, float repetition1,
                        const void *presence, float presence1, const void *frequency, float frequency1, const void *bias,
                        long long stride_bias, const void *mask, long long stride_mask, int B, int V, void *stream)
{
    if (!x || !out) return ADKV_E_NULL;
    if (B < 0 || V <= 0 || V > 0x7fff0000 || history_cap < 0 || B > 65535 || (B > 1 && stride_out < V)) return ADKV_E_SHAPE;   // rows of out must lie apart
    if (type < ADKV_T_F16 || type > ADKV_T_F32) return ADKV_E_TYPE;
    const unsigned size = type == ADKV_T_F32 ? 4 : 2;
    if (!aligned_to(x, size) || !aligned_to(out, size) || !aligned_to(tokens, 4) || !aligned_to(history, 4) || !aligned_to(history_lens, 4) ||
        !aligned_to(repetition, 4) || !aligned_to(presence, 4) || !aligned_to(frequency, 4) || !aligned_to(bias, 4) || !aligned_to(mask, 4))
        return ADKV_E_ALIGN;
    if (B == 0) return 0;
    const auto f = [](const void *p) { return static_cast<const float *>(p); };
    const LogitArgs a{x, out, static_cast<int *>(tokens), static_cast<const int *>(history), static_cast<const int *>(history_lens), f(repetition),
                      f(presence), f(frequency), repetition1, presence1, frequency1, f(bias), static_cast<const uint32_t *>(mask), stride_x,
                      stride_out, stride_history, stride_bias, stride_mask, V, history_cap, 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return type == ADKV_T_F16 ? launch_logits<__half>(a, B, s) : type == ADKV_T_BF16 ? launch_logits<__nv_bfloat16>(a, B, s) : launch_logits<float>(a, B, s);
}

}  // extern "C"
