// Log-probabilities of given tokens with the entropy of every row, its top alternatives, and their gradient, for sm_100a.
//
//   y = x / temperature, m = max x, s = sum_v exp((x_v - m) / temperature), t = sum_v exp((x_v - m) / temperature) (x_v - m)
//   ln p_v = (x_v - m) / temperature - ln s        entropy = ln s - t / (temperature s)     (both terms >= 0: no cancellation)
//   d logprob / d x_v = ([v = target] - p_v) / temperature
//   d entropy / d x_v = -p_v (ln p_v + entropy) / temperature
//
// Both directions are pure streams: the forward reads every logit once (the running maximum carries s and t along), the
// gradient reads it once more and writes once. The bound is HBM; per logit the forward issues about six instructions, one of
// them the exponential, which leaves the SM half idle at the rate BF16 logits arrive.
//
// Top alternatives cost nothing per logit of a long row: the maximum that every thread keeps for the softmax anyway gives a
// threshold (the k-th largest of the maxima of 32 groups of threads) that at least k logits reach. A thread also leaves the maximum
// of each eighth of its logits; only those that reach the threshold are read again, a percent of the row, and the few logits that
// reach it are ranked by counting. (Reading all logits of such threads again cost as much as a fifth of the row: 20 alternatives of
// 4096 x 131072 BF16 logits 57 us on top of 166, 21 so.) A row that fits the registers of a few warps is compared with the threshold
// there. Order: larger logit first, equal ones by the lower index. A row with more candidates than the list holds (many equal logits,
// or fewer allowed tokens than alternatives) falls back to one pass per alternative.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "b200loss.h"
#include "kernels.cuh"
#include "loss_internal.h"
#include "tc_common.cuh"

namespace cg = cooperative_groups;

namespace {

using b200attn::launch_pdl;
using b200attn::launch_pdl_cluster;
using b200attn::pdl_launch_dependents;
using b200attn::pdl_wait;

constexpr int kWarpRowThreads = 256; // CTAs of the kernels that give a row to a warp
constexpr int kUnroll = 4;           // 16-byte loads in flight per thread
constexpr int kMaxTop = 32;
constexpr int kSegments = 8;
constexpr int kMaxCluster = 8;
constexpr int kWarpRowVocab = 384;   // rows up to here are handled by one warp each
constexpr int kWarpGradVocab = 256;  // the same in the gradient
constexpr int kSmallRowVecs = 1024;  // gradient: rows of up to so many 16-byte vectors by CTAs of 64 threads, longer ones by 256
constexpr int kMiddleRowVecs = 8192; // forward: up to so many by 128 threads, longer ones by 256
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -1e30f;    // x - m is held above this, so that a masked logit contributes 0 * finite
constexpr float kFloor = -0x1.92p99f; // -9.95e29, a BF16 value: logits enter the sums of a row as at least this (see Stat)
constexpr float kWild = 1e29f;       // maxima beyond this take the exact pass

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Maximum that a NaN passes through: a row that holds one ends as NaN instead of losing it.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// ---------------------------------------------------------------- element access
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kPerVec = 4;
    static constexpr uint32_t kNegInf = 0xff800000u;
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ void store(float* p, float x) { *p = x; }
    static __device__ __forceinline__ void unpack(const uint4& w, float* x) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ uint4 raise(uint4 w) {  // every element to at least kFloor
        w.x = max1(w.x), w.y = max1(w.y), w.z = max1(w.z), w.w = max1(w.w);
        return w;
    }
    static __device__ __forceinline__ uint32_t max1(uint32_t x) { return __float_as_uint(max_nan(__uint_as_float(x), kFloor)); }
    template <int N>
    static __device__ __forceinline__ float largest(const uint4 (&w)[N]) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            float x[4];
            unpack(w[u], x);
            m = max_nan(max_nan(m, max_nan(x[0], x[1])), max_nan(x[2], x[3]));
        }
        return m;
    }
    // Bits of a word for kVecsPerWord vectors: set by vector u for the elements that are not below a threshold (a number that T holds).
    static constexpr int kVecsPerWord = 8;
    static constexpr float kLowestNumber = -0x1.fffffep127f;
    static __device__ __forceinline__ uint32_t reach(const uint4& w, float threshold, int u, uint32_t bits) {
        float x[4];
        unpack(w, x);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (!(x[e] < threshold)) bits |= 1u << (4 * (u % kVecsPerWord) + e);
        return bits;
    }
    static __device__ __forceinline__ int vec_of(int bit) { return bit >> 2; }
    static __device__ __forceinline__ int element_of(int bit) { return bit & 3; }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kPerVec = 8;
    static constexpr uint32_t kNegInf = 0xff80ff80u;
    static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
    static __device__ __forceinline__ void unpack(const uint4& w, float* x) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    // packed pairs: half the instructions of single maxima
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t y;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
        return y;
    }
    static __device__ __forceinline__ uint4 raise(uint4 w) {
        constexpr uint32_t floor2 = 0xf149f149u;  // kFloor, twice
        w.x = max2(w.x, floor2), w.y = max2(w.y, floor2), w.z = max2(w.z, floor2), w.w = max2(w.w, floor2);
        return w;
    }
    template <int N>
    static __device__ __forceinline__ float largest(const uint4 (&w)[N]) {
        uint32_t m = kNegInf;
#pragma unroll
        for (int u = 0; u < N; ++u) m = max2(max2(m, max2(w[u].x, w[u].y)), max2(w[u].z, w[u].w));
        return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    static constexpr int kVecsPerWord = 4;  // (see Elem<float>) the lower elements of the pairs in the lower half
    static constexpr float kLowestNumber = -0x1.fep127f;
    static __device__ __forceinline__ uint32_t reach(const uint4& w, float threshold, int u, uint32_t bits) {
        const __nv_bfloat162 t2 = __float2bfloat162_rn(threshold);
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) bits |= ~__hlt2_mask(*reinterpret_cast<const __nv_bfloat162*>(&v[i]), t2) & (0x00010001u << (4 * (u % kVecsPerWord) + i));
        return bits;
    }
    static __device__ __forceinline__ int vec_of(int bit) { return (bit & 15) >> 2; }
    static __device__ __forceinline__ int element_of(int bit) { return 2 * (bit & 3) + (bit >> 4); }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
};

// A row split into up to 15 bytes of elements in front of the first 16-byte boundary, whole vectors, and the rest.
struct RowSplit {
    int head, vecs, tail;
};
template <typename T>
__device__ __forceinline__ RowSplit split_row(const T* row, int V) {
    RowSplit s;
    const int past = int(reinterpret_cast<uintptr_t>(row) & 15u) / int(sizeof(T));
    s.head = min(past ? Elem<T>::kPerVec - past : 0, V);
    s.vecs = (V - s.head) / Elem<T>::kPerVec;
    s.tail = V - s.head - s.vecs * Elem<T>::kPerVec;
    return s;
}

// ---------------------------------------------------------------- arithmetic
// Packed pairs of FP32: one instruction for two operations.
struct Pair {
    uint64_t v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair add(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair mul(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// A part of a row: its maximum m, s = sum 2^a and t = sum a 2^a with a = c (x - m), c = log2(e) / temperature.
// Logits enter the sums as at least kFloor, which costs one packed maximum and keeps every a and every m finite (a masked logit
// adds 0 * finite, not 0 * inf). That changes nothing unless the row's maximum is below kFloor / 10 or so itself: rows with a
// maximum outside +-kWild (a row of masked logits, of the type's lowest value, of NaN or +inf) are summed again without it.
struct Stat {
    float m, s, t;
};
// `a` with its sums taken relative to the larger maximum M.
__device__ __forceinline__ void rebase(Stat& a, float M, float c) {
    const float d = fmaxf((a.m - M) * c, -1000.f), f = ex2(d);  // 2^-1000 is 0, and s d stays finite
    a.t = fmaf(a.s, d, a.t) * f;
    a.s *= f;
    a.m = M;
}
// What the outputs need of a whole row.
struct RowStat {
    float m, ln_s, entropy;  // ln_s: of the sum relative to m
};
__device__ __forceinline__ RowStat finish(const Stat& a) {
    if (a.m == -INFINITY) return RowStat{a.m, 0.f, 0.f};  // no token is allowed
    const float log2_s = log2f(a.s);
    return RowStat{a.m, log2_s * kLn2, (log2_s - a.t / a.s) * kLn2};
}
// s and t of a row (or of a part of it) whose maximum m is known, in exact steps and with every logit as it is: one element.
__device__ __forceinline__ void add_exact(float x, float m, float c, float& s, float& t) {
    const float a = max_nan(x - m, kLowest) * c, e = ex2(a);
    s += e;
    t = fmaf(e, a, t);
}
__device__ __forceinline__ float warp_add(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ float warp_max_nan(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = max_nan(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}

// Whole numbers in the order of the logits (-0 = +0; NaN above every number, below the all-ones bound of a search), and back.
constexpr uint32_t kKeyNaN = 0xfffffffeu;
__device__ __forceinline__ uint32_t to_key(float x) {
    if (x != x) return kKeyNaN;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_key(uint32_t k) {
    if (k == kKeyNaN) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;  // to_key(-inf)
// Larger = better: the logit, then the lower index.
__device__ __forceinline__ uint64_t candidate(uint32_t key, int index) { return (uint64_t(key) << 32) | uint32_t(~uint32_t(index)); }
__device__ __forceinline__ int index_of(uint64_t c) { return int(~uint32_t(c)); }

struct FwdArgs {
    const void* logits;
    long long row_stride;
    const int* targets;
    int rows, V;
    float inv_temperature;
    float *logprobs, *entropy, *stats;
    int top;
    float* top_logprobs;
    int* top_tokens;
};

// A row without an allowed token (every logit -inf): every log-probability is -inf, the entropy 0.
__device__ __forceinline__ float logprob_of(float x, const RowStat& a, float inv_temperature) {
    return a.m == -INFINITY ? -INFINITY : fmaf(x - a.m, inv_temperature, -a.ln_s);
}
__device__ __forceinline__ void write_row(const FwdArgs& a, int r, const RowStat& st, bool given, float target_x) {
    a.stats[2ll * r] = st.m;
    a.stats[2ll * r + 1] = st.ln_s;
    a.entropy[r] = st.entropy;
    a.logprobs[r] = given ? logprob_of(target_x, st, a.inv_temperature) : 0.f;
}

// ---------------------------------------------------------------- alternatives
// Sorts the warp's keys in descending order (lane 0 the largest).
__device__ __forceinline__ uint32_t warp_sort(uint32_t x, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const uint32_t y = __shfl_xor_sync(0xffffffffu, x, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0);  // this lane keeps the larger one
            x = larger ? max(x, y) : min(x, y);
        }
    return x;
}
// The k-th largest of 32 groups' maxima (lane i's key is that of group i): at least k logits of the row reach it, and where the large ones
// are spread evenly -32 ln(1 - k / 32) do in the mean (31 for 20 alternatives), however long the row. Never -inf: a masked logit is
// only an alternative where fewer tokens are allowed than alternatives asked for, which is left to write_alternatives' last resort.
template <typename T>
__device__ __forceinline__ float threshold_of(uint32_t group, int top, int lane) {
    return from_key(max(__shfl_sync(0xffffffffu, warp_sort(group, lane), top - 1), to_key(Elem<T>::kLowestNumber)));
}
__device__ __forceinline__ void write_alternative(const FwdArgs& a, int r, const RowStat& total, int rank, uint64_t y) {
    a.top_logprobs[(long long)r * a.top + rank] = logprob_of(from_key(uint32_t(y >> 32)), total, a.inv_temperature);
    a.top_tokens[(long long)r * a.top + rank] = index_of(y);
}
// Ranks the n candidates of a row, whose indices are in `cand`, by counting: the threads of a row (one warp or a whole CTA). Where they are
// fewer than alternatives or more than the list holds: one pass over the row per alternative, the best logit below the one before.
template <typename T, int kThreads, int kList>
__device__ __forceinline__ void write_alternatives(const FwdArgs& a, int r, const RowStat& total, const T* row, const RowSplit& sp, int tid, int n, uint64_t* cand,
                                                   uint64_t* s_best) {
    const int lane = tid & 31, warp = tid >> 5;
    if (n >= a.top && n <= kList) {
        const bool few = kThreads == 32 || n <= 32;  // one warp's work
        if (few && warp > 0) return;
        const int step = few ? 32 : kThreads;
        for (int i = tid; i < n; i += step) {
            const int index = int(cand[i]);
            cand[i] = candidate(to_key(Elem<T>::load(row + index)), index);
        }
        if (few) __syncwarp();
        else __syncthreads();
        for (int i = tid; i < n; i += step) {
            const uint64_t y = cand[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += cand[j] > y;
            if (rank < a.top) write_alternative(a, r, total, rank, y);
        }
        return;
    }
    const uint4* vec = reinterpret_cast<const uint4*>(row + sp.head);
    const int singles = sp.head + sp.tail;
    uint64_t before = ~uint64_t(0);
    for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        auto see = [&](float x, int index) {
            const uint64_t y = candidate(to_key(x), index);
            if (y < before && y > best) best = y;
        };
        for (int i = tid; i < sp.vecs; i += kThreads) {
            constexpr int E = Elem<T>::kPerVec;
            float x[E];
            Elem<T>::unpack(__ldg(vec + i), x);
#pragma unroll
            for (int e = 0; e < E; ++e) see(x[e], sp.head + i * E + e);
        }
        if (tid < singles) {
            const int index = tid < sp.head ? tid : a.V - singles + tid;
            see(Elem<T>::load(row + index), index);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t y = __shfl_xor_sync(0xffffffffu, best, o);
            if (y > best) best = y;
        }
        if constexpr (kThreads > 32) {
            __syncthreads();  // the round before has been read
            if (lane == 0) s_best[warp] = best;
            __syncthreads();
            for (int i = 0; i < kThreads / 32; ++i) best = s_best[i] > best ? s_best[i] : best;
        }
        if (tid == 0) write_alternative(a, r, total, k, best);
        before = best;
    }
}

// ---------------------------------------------------------------- forward, one CTA (or one cluster of CTAs) per row
template <typename T, int kThreads, bool CLUSTER>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const FwdArgs a) {
    constexpr int E = Elem<T>::kPerVec, kWarps = kThreads / 32, kMaxCand = kThreads >= 256 ? 1024 : 256, kMaxHot = kThreads >= 256 ? 256 : 128;
    __shared__ float s_max[kWarps], s_sum[kWarps * kMaxCluster], s_sum_a[kWarps * kMaxCluster], s_part_max[kMaxCluster];
    __shared__ uint32_t s_key[kThreads], s_part_key[kMaxCluster][32];
    __shared__ uint64_t s_cand[kMaxCand], s_best[kWarps];
    __shared__ float s_segment[kSegments][kThreads];
    __shared__ int s_hot[kMaxHot];  // segments that hold a candidate: thread + kThreads * segment
    __shared__ int s_nhot, s_ncand;

    pdl_launch_dependents();
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = CLUSTER ? int(cluster.num_blocks()) : 1, part = CLUSTER ? int(cluster.block_rank()) : 0;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float c = a.inv_temperature * kLog2e;
    const Pair c2 = pair(c, c);
    const uint4 nothing = make_uint4(Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf);

    const int r = int(blockIdx.x / unsigned(parts));
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    const RowSplit sp = split_row(row, a.V);
    const int head = sp.head;
    const uint4* vec = reinterpret_cast<const uint4*>(row + head);
    const int begin = int((long long)sp.vecs * part / parts), end = int((long long)sp.vecs * (part + 1) / parts);
    // the single element in front of or behind the vectors that this thread owns, if any
    const int edge = (part == 0 && tid < sp.head) ? tid
                     : (part == parts - 1 && tid >= 16 && tid < 16 + sp.tail) ? sp.head + sp.vecs * E + (tid - 16)
                                                                              : -1;
    uint4 next[kUnroll];  // the next round's loads are under way while this one is added
    auto load_round = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kThreads + tid;
            next[u] = i < end ? __ldg(vec + i) : nothing;
        }
    };
    pdl_wait();
    load_round(begin);
    // needed at the end only: under way with the first round
    const float edge_x = edge >= 0 ? Elem<T>::load(row + edge) : -INFINITY;
    const int target = a.targets[r];
    const bool given = (unsigned)target < (unsigned)a.V;
    Stat st{kFloor, 0.f, 0.f};
    float my_max = edge_x;  // of the logits as they are: what the alternatives are found by, and whether the row is wild
    Pair s2 = pair(0.f, 0.f), t2 = pair(0.f, 0.f);
    // The row's rounds in at most kSegments segments: a thread's maximum is kept for each (alternatives only).
    const int rounds = (end - begin + kThreads * kUnroll - 1) / (kThreads * kUnroll), per_segment = max(1, (rounds + kSegments - 1) / kSegments);
    float segment_max = -INFINITY;
    int segment = 0, left = per_segment;
    for (int i0 = begin; i0 < end; i0 += kThreads * kUnroll) {
        uint4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) w[u] = next[u];
        if (i0 + kThreads * kUnroll < end) load_round(i0 + kThreads * kUnroll);
        const float round_max = Elem<T>::largest(w);
        my_max = max_nan(my_max, round_max);
        if (a.top > 0) {
            segment_max = max_nan(segment_max, round_max);
            if (--left == 0 || i0 + kThreads * kUnroll >= end) {
                s_segment[segment++][tid] = segment_max;
                segment_max = -INFINITY, left = per_segment;
            }
        }
        const float m = max_nan(st.m, round_max);
        if (m != st.m) {  // a new maximum, or NaN
            float sa, sb, ta, tb;
            split(s2, sa, sb), split(t2, ta, tb);
            Stat old{st.m, sa + sb, ta + tb};
            rebase(old, m, c);
            st.m = m;
            s2 = pair(old.s, 0.f), t2 = pair(old.t, 0.f);
        }
        const Pair neg_m = pair(-st.m, -st.m);
        auto add_vec = [&](const uint4& v) {
            float x[E];
            Elem<T>::unpack(Elem<T>::raise(v), x);
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                float a0, a1;
                const Pair arg = mul(add(pair(x[e], x[e + 1]), neg_m), c2);
                split(arg, a0, a1);
                const Pair ex = pair(ex2(a0), ex2(a1));
                s2 = add(s2, ex);
                t2 = fma(ex, arg, t2);
            }
        };
        if (i0 + kThreads * kUnroll <= end) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) add_vec(w[u]);
        } else {  // the last round: not what this warp has nothing of
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (i0 + u * kThreads + warp * 32 < end) add_vec(w[u]);
        }
    }
    const float target_x = given && tid == 0 && part == 0 ? Elem<T>::load(row + target) : 0.f;  // under way with the reductions
    {
        float sa, sb, ta, tb;
        split(s2, sa, sb), split(t2, ta, tb);
        st.s = sa + sb, st.t = ta + tb;
    }
    auto barrier = [&]() {
        if constexpr (CLUSTER) cluster.sync();
        else __syncthreads();
    };
    float row_max = warp_max_nan(my_max);
    if (lane == 0) s_max[warp] = row_max;
    s_key[tid] = to_key(my_max);
    if (tid == 0) s_nhot = 0, s_ncand = 0;
    barrier();
    uint32_t group = 0u;  // the largest key of the row's threads with this lane
    if constexpr (CLUSTER) {  // a warp fetches what a CTA of the row has
        for (int p = warp; p < parts; p += kWarps) {
            const float* from = cluster.map_shared_rank(s_max, p);
            const uint32_t* keys = cluster.map_shared_rank(s_key, p);
            const float x = warp_max_nan(lane < kWarps ? from[lane] : -INFINITY);
            uint32_t k = 0u;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) k = max(k, keys[i * 32 + lane]);
            s_part_key[p][lane] = k;
            if (lane == 0) s_part_max[p] = x;
        }
        __syncthreads();
        for (int p = 0; p < parts; ++p) row_max = max_nan(row_max, s_part_max[p]), group = max(group, s_part_key[p][lane]);
    } else {
#pragma unroll
        for (int i = 0; i < kWarps; ++i) row_max = max_nan(row_max, s_max[i]), group = max(group, s_key[i * 32 + lane]);
    }
    float s = 0.f, t = 0.f;
    if (fabsf(row_max) < kWild) {
        rebase(st, row_max, c);
        s = st.s, t = st.t;
        if (edge >= 0) add_exact(edge_x, row_max, c, s, t);
    } else if (row_max != -INFINITY) {  // (see Stat)
        for (int i = begin + tid; i < end; i += kThreads) {
            float x[E];
            Elem<T>::unpack(__ldg(vec + i), x);
#pragma unroll
            for (int e = 0; e < E; ++e) add_exact(x[e], row_max, c, s, t);
        }
        if (edge >= 0) add_exact(edge_x, row_max, c, s, t);
    }
    s = warp_add(s), t = warp_add(t);
    // what follows goes to the first CTA of the row
    float *sums = s_sum, *sums_a = s_sum_a;
    int* ncand = &s_ncand;
    uint64_t* cand = s_cand;
    if constexpr (CLUSTER) {
        sums = cluster.map_shared_rank(s_sum, 0) + part * kWarps, sums_a = cluster.map_shared_rank(s_sum_a, 0) + part * kWarps;
        ncand = cluster.map_shared_rank(&s_ncand, 0), cand = cluster.map_shared_rank(s_cand, 0);
    }
    if (lane == 0) sums[warp] = s, sums_a[warp] = t;
    if (a.top > 0) {
        const float threshold = threshold_of<T>(group, a.top, lane);
        if (!(my_max < threshold))
            for (int i = 0; i < segment; ++i)  // its own: no other thread has written them
                if (!(s_segment[i][tid] < threshold)) {
                    const int at = atomicAdd(&s_nhot, 1);
                    if (at < kMaxHot) s_hot[at] = tid + kThreads * i;
                }
        __syncthreads();
        const int nhot = s_nhot;
        // every (segment, vector of it) to a thread of its own, several at a time, so that the reads are under way together
        const int per = per_segment * kUnroll, pairs = nhot <= kMaxHot ? nhot * per : 0;
        auto vec_at = [&](int i) {
            const int hot = s_hot[i / per];
            return begin + hot % kThreads + ((hot / kThreads) * per + i % per) * kThreads;
        };
        for (int i0 = tid; i0 < pairs; i0 += kThreads * kUnroll) {
            uint4 w[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int i = i0 + u * kThreads, at = i < pairs ? vec_at(i) : end;
                w[u] = at < end ? __ldg(vec + at) : nothing;
            }
            static_assert(kUnroll <= Elem<T>::kVecsPerWord, "");
            uint32_t bits = 0u;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) bits = Elem<T>::reach(w[u], threshold, u, bits);
            if (bits != 0u) {
                int at = atomicAdd(ncand, __popc(bits));
                for (; bits != 0u && at < kMaxCand; bits &= bits - 1u, ++at) {
                    const int bit = __ffs(bits) - 1;
                    cand[at] = head + vec_at(i0 + Elem<T>::vec_of(bit) * kThreads) * E + Elem<T>::element_of(bit);
                }
            }
        }
        if (edge >= 0 && !(edge_x < threshold)) {
            const int at = atomicAdd(ncand, 1);
            if (at < kMaxCand) cand[at] = edge;
        }
        if (nhot > kMaxHot && tid == 0) atomicAdd(ncand, kMaxCand + 1);  // not looked for
    }
    barrier();
    if (part != 0) return;
    s = t = 0.f;
    for (int i = 0; i < parts * kWarps; ++i) s += s_sum[i], t += s_sum_a[i];
    const RowStat total = finish(Stat{row_max, s, t});
    if (tid == 0) write_row(a, r, total, given, target_x);
    if (a.top > 0) write_alternatives<T, kThreads, kMaxCand>(a, r, total, row, sp, tid, s_ncand, s_cand, s_best);
}

// ---------------------------------------------------------------- forward, rows that fit the registers of a few warps
// kWarps warps to a row (kWarps = 1: four rows to a CTA), N vectors per thread, all loads of a row under way together. With the row in
// registers its maximum is known before the sums, which are then exact in one go, and the alternatives are compared in place: 32
// groups of threads give a threshold (the k-th largest of their maxima) that a few dozen logits of the row reach. Two barriers.
template <typename T, int kWarps, int N>
__global__ void __launch_bounds__(kWarps == 1 ? 128 : 32 * kWarps) token_logprobs_resident_kernel(const FwdArgs a) {
    constexpr int E = Elem<T>::kPerVec, kThreads = 32 * kWarps, kRows = kWarps == 1 ? 4 : 1, kList = 256;
    __shared__ uint64_t s_cand[kRows][kList];
    __shared__ int s_ncand[kRows];
    __shared__ float s_max[kWarps], s_sum[kWarps], s_sum_a[kWarps];
    __shared__ uint32_t s_key[kWarps][32];
    __shared__ uint64_t s_best[kWarps];
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, local = kWarps == 1 ? threadIdx.x >> 5 : 0, warp = kWarps == 1 ? 0 : threadIdx.x >> 5;
    const int tid = warp * 32 + lane;
    auto barrier = [&]() {
        if constexpr (kWarps == 1) __syncwarp();
        else __syncthreads();
    };
    const long long r64 = (long long)blockIdx.x * kRows + local;
    const float c = a.inv_temperature * kLog2e;
    const uint4 nothing = make_uint4(Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf);
    pdl_wait();
    if (r64 >= a.rows) return;
    const int r = int(r64);
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    const RowSplit sp = split_row(row, a.V);
    const int head = sp.head;
    const uint4* vec = reinterpret_cast<const uint4*>(row + head);
    uint4 w[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int i = u * kThreads + tid;
        w[u] = i < sp.vecs ? __ldg(vec + i) : nothing;
    }
    // the single element in front of or behind the vectors that this thread owns, if any
    const int edge = tid < head ? tid : (tid >= 16 && tid < 16 + sp.tail) ? head + sp.vecs * E + (tid - 16) : -1;
    const float edge_x = edge >= 0 ? Elem<T>::load(row + edge) : -INFINITY;
    const int target = a.targets[r];
    const bool given = (unsigned)target < (unsigned)a.V;
    const float target_x = given && tid == 0 ? Elem<T>::load(row + target) : 0.f;

    const float my_max = max_nan(Elem<T>::largest(w), edge_x);
    float m = warp_max_nan(my_max);
    uint32_t group = to_key(my_max);
    if (tid == 0) s_ncand[local] = 0;
    if constexpr (kWarps > 1) {
        if (lane == 0) s_max[warp] = m;
        s_key[warp][lane] = group;
    }
    barrier();
    if constexpr (kWarps > 1) {
#pragma unroll
        for (int i = 0; i < kWarps; ++i) m = max_nan(m, s_max[i]), group = max(group, s_key[i][lane]);
    }
    float s = 0.f, t = 0.f;
    if (fabsf(m) < kWild) {  // (see Stat)
        const Pair c2 = pair(c, c), neg_m = pair(-m, -m);
        Pair s2 = pair(0.f, 0.f), t2 = pair(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            if (u * kThreads + warp * 32 >= sp.vecs) break;
            float x[E];
            Elem<T>::unpack(Elem<T>::raise(w[u]), x);
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                float a0, a1;
                const Pair arg = mul(add(pair(x[e], x[e + 1]), neg_m), c2);
                split(arg, a0, a1);
                const Pair ex = pair(ex2(a0), ex2(a1));
                s2 = add(s2, ex);
                t2 = fma(ex, arg, t2);
            }
        }
        float sb, tb;
        split(s2, s, sb), split(t2, t, tb);
        s += sb, t += tb;
        if (edge >= 0) add_exact(edge_x, m, c, s, t);
    } else if (m != -INFINITY) {  // read again: the elements of the row as numbers are not kept beside their words
        for (int i = tid; i < sp.vecs; i += kThreads) {
            float x[E];
            Elem<T>::unpack(__ldg(vec + i), x);
#pragma unroll
            for (int e = 0; e < E; ++e) add_exact(x[e], m, c, s, t);
        }
        if (edge >= 0) add_exact(edge_x, m, c, s, t);
    }
    s = warp_add(s), t = warp_add(t);
    if constexpr (kWarps > 1) {
        if (lane == 0) s_sum[warp] = s, s_sum_a[warp] = t;
    }
    if (a.top > 0) {
        const float threshold = threshold_of<T>(group, a.top, lane);
        constexpr int kPer = Elem<T>::kVecsPerWord, kWords = (N + kPer - 1) / kPer;
        uint32_t bits[kWords];
        int count = edge >= 0 && !(edge_x < threshold);
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            bits[i] = 0u;
#pragma unroll
            for (int u = i * kPer; u < min(N, (i + 1) * kPer); ++u) bits[i] = Elem<T>::reach(w[u], threshold, u, bits[i]);
            count += __popc(bits[i]);
        }
        if (count > 0) {
            int at = atomicAdd(&s_ncand[local], count);
            if (at + count <= kList) {
                if (edge >= 0 && !(edge_x < threshold)) s_cand[local][at++] = edge;
#pragma unroll
                for (int i = 0; i < kWords; ++i)
                    for (uint32_t left = bits[i]; left != 0u; left &= left - 1u) {
                        const int bit = __ffs(left) - 1;
                        s_cand[local][at++] = head + ((i * kPer + Elem<T>::vec_of(bit)) * kThreads + tid) * E + Elem<T>::element_of(bit);
                    }
            }
        }
    }
    barrier();
    if constexpr (kWarps > 1) {
        s = t = 0.f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) s += s_sum[i], t += s_sum_a[i];
    }
    const RowStat total = finish(Stat{m, s, t});
    if (tid == 0) write_row(a, r, total, given, target_x);
    if (a.top > 0) write_alternatives<T, kThreads, kList>(a, r, total, row, sp, tid, s_ncand[local], s_cand[local], s_best);
}

// ---------------------------------------------------------------- forward, one warp per (short) row
// N: elements per lane, all of them in registers.
template <typename T, int N>
__global__ void __launch_bounds__(kWarpRowThreads) token_logprobs_warp_kernel(const FwdArgs a) {
    constexpr int kWarps = kWarpRowThreads / 32;
    __shared__ uint64_t s_cand[kWarps][32 * N];
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long r64 = (long long)blockIdx.x * kWarps + warp;
    pdl_wait();
    if (r64 >= a.rows) return;
    const int r = int(r64);
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    const float c = a.inv_temperature * kLog2e;
    const int target = a.targets[r];
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i * 32 + lane < a.V ? Elem<T>::load(row + i * 32 + lane) : -INFINITY;
    const bool given = (unsigned)target < (unsigned)a.V;
    const float target_x = given ? Elem<T>::load(row + target) : 0.f;
    float mine = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mine = max_nan(mine, x[i]);
    Stat st{warp_max_nan(mine), 0.f, 0.f};
    if (st.m != -INFINITY) {
#pragma unroll
        for (int i = 0; i < N; ++i) add_exact(x[i], st.m, c, st.s, st.t);
        st.s = warp_add(st.s), st.t = warp_add(st.t);
    }
    const RowStat total = finish(st);
    if (lane == 0) write_row(a, r, total, given, target_x);
    if (a.top == 0) return;

    // alternatives: as above, with the lanes as groups; a row too short for 32 of them, or with too few allowed tokens, has the threshold
    // -inf (every logit is a candidate). The list holds them all.
    const uint32_t group = lane < a.V ? to_key(mine) : 0u;
    const float threshold = from_key(max(__shfl_sync(0xffffffffu, warp_sort(group, lane), a.top - 1), kKeyNegInf));
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool reaches = i * 32 + lane < a.V && !(x[i] < threshold);
        const uint32_t who = __ballot_sync(0xffffffffu, reaches);
        if (reaches) s_cand[warp][n + __popc(who & ((1u << lane) - 1u))] = candidate(to_key(x[i]), i * 32 + lane);
        n += __popc(who);
    }
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
        const uint64_t y = s_cand[warp][i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s_cand[warp][j] > y;
        if (rank < a.top) write_alternative(a, r, total, rank, y);
    }
}

// ---------------------------------------------------------------- gradient
struct BwdArgs {
    const void* logits;
    long long row_stride;
    const int* targets;
    const float *entropy, *stats, *grad_logprobs, *grad_entropy;
    int rows, V;
    float inv_temperature;
    void* dlogits;
    long long d_row_stride;
    int chunks;  // CTAs per row
    float lowest;  // d = x - m is held above this: 2^(c d - l) is 0 there already, and b d a number at every temperature and weight
};

// dx_v = p_v (a + b d) + [v = target] g / temperature with d = x_v - m and p_v = 2^(c d - l): one exponential and two
// multiply-adds per logit once these are known.
struct RowGrad {
    float m, l, a, b, g;
    int target;
    bool zero;  // no gradient reaches the row (or it has no allowed token): written as zeros, whatever its logits hold
};
__device__ __forceinline__ RowGrad row_grad(const BwdArgs& p, int r) {
    RowGrad q;
    q.target = p.targets[r];
    const bool given = (unsigned)q.target < (unsigned)p.V;
    const float g = given ? p.grad_logprobs[r] : 0.f, ge = p.grad_entropy ? p.grad_entropy[r] : 0.f;
    q.m = p.stats[2ll * r];
    const float ln_s = p.stats[2ll * r + 1];
    q.zero = (g == 0.f && ge == 0.f) || q.m == -INFINITY;
    q.l = ln_s * kLog2e;
    q.g = g * p.inv_temperature;
    q.a = -p.inv_temperature * (ge == 0.f ? g : fmaf(ge, p.entropy[r] - ln_s, g));
    q.b = -p.inv_temperature * p.inv_temperature * ge;
    return q;
}
__device__ __forceinline__ float grad_of(const RowGrad& q, float x, float c, float lowest) {  // without the target's own term
    const float d = max_nan(x - q.m, lowest);
    return ex2(fmaf(d, c, -q.l)) * fmaf(d, q.b, q.a);
}

// One CTA per row and chunk of vectors; logits and dlogits are at the same distance from a 16-byte boundary in every row.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(const BwdArgs a) {
    constexpr int E = Elem<T>::kPerVec;
    const int r = int(blockIdx.x / unsigned(a.chunks)), chunk = int(blockIdx.x % unsigned(a.chunks));
    const int tid = threadIdx.x;
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    T* out = static_cast<T*>(a.dlogits) + a.d_row_stride * r;
    const RowSplit sp = split_row(row, a.V);
    const RowGrad q = row_grad(a, r);
    const float c = a.inv_temperature * kLog2e;
    const uint4* src = reinterpret_cast<const uint4*>(row + sp.head);
    uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
    const int begin = chunk * kThreads * kUnroll;
    if (q.zero) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = begin + u * kThreads + tid;
            if (i < sp.vecs) dst[i] = make_uint4(0u, 0u, 0u, 0u);
        }
    } else {
        uint4 w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = begin + u * kThreads + tid;
            if (i < sp.vecs) w[u] = src[i];
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = begin + u * kThreads + tid;
            if (i < sp.vecs) {
                float x[E];
                Elem<T>::unpack(w[u], x);
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = grad_of(q, x[e], c, a.lowest);
                const int at = q.target - (sp.head + i * E);
                if ((unsigned)at < (unsigned)E) {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (e == at) x[e] += q.g;
                }
                dst[i] = Elem<T>::pack(x);
            }
        }
    }
    // the elements outside the vectors
    const int edge = (chunk == 0 && tid < sp.head) ? tid
                     : (chunk == a.chunks - 1 && tid >= 32 && tid < 32 + sp.tail) ? sp.head + sp.vecs * E + (tid - 32)
                                                                                  : -1;
    if (edge >= 0) Elem<T>::store(out + edge, q.zero ? 0.f : grad_of(q, Elem<T>::load(row + edge), c, a.lowest) + (edge == q.target ? q.g : 0.f));
}

// One warp per row: short rows, and rows of dlogits at another distance from a 16-byte boundary than the logits'.
template <typename T>
__global__ void __launch_bounds__(kWarpRowThreads) token_logprobs_bwd_warp_kernel(const BwdArgs a) {
    constexpr int kWarps = kWarpRowThreads / 32;
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long r64 = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    pdl_wait();
    if (r64 >= a.rows) return;
    const int r = int(r64);
    const T* row = static_cast<const T*>(a.logits) + a.row_stride * r;
    T* out = static_cast<T*>(a.dlogits) + a.d_row_stride * r;
    const RowGrad q = row_grad(a, r);
    const float c = a.inv_temperature * kLog2e;
    for (int v0 = 0; v0 < a.V; v0 += 32 * kUnroll) {  // read together, then written: the gradient may go where the logits are
        float x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int v = v0 + u * 32 + lane;
            x[u] = v < a.V && !q.zero ? Elem<T>::load(row + v) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int v = v0 + u * 32 + lane;
            if (v < a.V) Elem<T>::store(out + v, q.zero ? 0.f : grad_of(q, x[u], c, a.lowest) + (v == q.target ? q.g : 0.f));
        }
    }
}

// ---------------------------------------------------------------- host side
int fail(int code, const char* what) {
    b200loss::set_error(what);
    return code;
}
int finish(cudaError_t e, const char* where) {
    if (e == cudaSuccess) return B200LOSS_OK;
    b200loss::set_error(where, cudaGetErrorString(e));
    return B200LOSS_ERR_CUDA;
}

int check_common(const char* null_text, bool any_null, int dtype, int rows, int V, long long row_stride, float temperature) {
    if (dtype != B200LOSS_F32 && dtype != B200LOSS_BF16) return fail(B200LOSS_ERR_ARG, "token_logprobs: dtype must be B200LOSS_F32 or B200LOSS_BF16");
    if (rows < 0 || V <= 0) return fail(B200LOSS_ERR_ARG, "token_logprobs: rows must not be negative and V must be positive");
    if (row_stride < V) return fail(B200LOSS_ERR_ARG, "token_logprobs: row_stride is smaller than V");
    if (!(temperature >= 1e-6f && temperature <= 1e6f)) return fail(B200LOSS_ERR_ARG, "token_logprobs: temperature must be between 1e-6 and 1e6");
    if (rows > 0 && any_null) return fail(B200LOSS_ERR_ARG, null_text);
    return B200LOSS_OK;
}
bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

template <typename T, int kThreads>
cudaError_t launch_rows(const FwdArgs& a, cudaStream_t stream) {
    // Few rows: a cluster of CTAs shares one, so that the row is not read at the speed of one SM. Each CTA keeps at least one
    // full round of loads.
    int parts = 1;
    while (parts < kMaxCluster && (long long)a.rows * parts * 2 <= 296 && a.V / (parts * 2) >= kThreads * Elem<T>::kPerVec) parts *= 2;
    if (parts == 1) return launch_pdl(token_logprobs_kernel<T, kThreads, false>, dim3(unsigned(a.rows)), dim3(kThreads), 0, stream, a);
    return launch_pdl_cluster(token_logprobs_kernel<T, kThreads, true>, dim3(unsigned(a.rows) * unsigned(parts)), dim3(unsigned(parts)), dim3(kThreads), 0, stream, a);
}

template <typename T, int kWarps, int N>
cudaError_t launch_resident(const FwdArgs& a, cudaStream_t stream) {
    constexpr int rows = kWarps == 1 ? 4 : 1, threads = kWarps == 1 ? 128 : 32 * kWarps;
    return launch_pdl(token_logprobs_resident_kernel<T, kWarps, N>, dim3((a.rows + rows - 1) / rows), dim3(threads), 0, stream, a);
}
template <typename T>
cudaError_t launch_forward(const FwdArgs& a, cudaStream_t stream) {
    if (a.V <= kWarpRowVocab) {
        constexpr int rows = kWarpRowThreads / 32;
        auto kern = a.V <= 128 ? token_logprobs_warp_kernel<T, 4> : token_logprobs_warp_kernel<T, 12>;
        return launch_pdl(kern, dim3((a.rows + rows - 1) / rows), dim3(kWarpRowThreads), 0, stream, a);
    }
    // Rows that fit the registers of a few warps. Measured without and with 20 alternatives, here and by the
    // kernel for long rows: BF16 16384 x 2001 14 and 27 us (34 and 86), 8388 x 4000 14 and 26 (23 and 52), 4096 x 8192 14 and 21 (17 and 33),
    // 2097 x 16000 14 and 21 (15 and 23); FP32 5592 x 6000 23 and 38 (27 and 42); one row of 8192 2.3 and 3.7 us (4.0 and 7).
    const int vecs = a.V / Elem<T>::kPerVec;
    if (vecs <= 128) return launch_resident<T, 1, 4>(a, stream);
    if (vecs <= 256) return launch_resident<T, 1, 8>(a, stream);
    // Half the warps with twice the vectors where rows are many: their ends cost less (without and with 20 alternatives, many vectors /
    // many warps: BF16 14894 x 2200 15.4 and 31 / 18.4 and 34 us, 4000 x 3000 6.7 and 12.7 / 7.1 and 12.0; FP32 8000 x 4096 21 and 31 / 24 and 34,
    // 600 x 4096 4.0 and 6.0 / 3.8 and 5.5).
    if (vecs <= 512) return a.rows > 40 * 148 ? launch_resident<T, 1, 16>(a, stream) : launch_resident<T, 2, 8>(a, stream);
    if (vecs <= 1024) return a.rows > 5 * 148 ? launch_resident<T, 2, 16>(a, stream) : launch_resident<T, 4, 8>(a, stream);
    if (vecs <= 2048) return launch_resident<T, 4, 16>(a, stream);
    // Eight warps with 100 registers are two CTAs to an SM, which wait for their loads together: up to two rounds of them (BF16
    // 300 x 32000 7.1 and 10.5 us, 8.2 and 11.6 by the kernel below; 1118 x 30000 15.7 and 24.7, 14.6 and 20.2 below).
    if (vecs <= 4096 && a.rows <= 4 * 148) return launch_resident<T, 8, 16>(a, stream);
    // A thread should have some rounds of its row, and the ends of rows should not fall together on an SM: the shorter the row, the
    // smaller (and the more) the CTAs, unless there are too few rows to fill the card with small ones (and too many for clusters of them).
    // Measured with 128 / 256 threads, BF16, without and with 20 alternatives: 3355 x 20000 28 and 39 / 34 and 51 us, 6001 x 50304 98
    // and 121 / 104 and 137 us, 64 x 32000 4.6 and 7.9 / 5.3 and 8.2 us, 600 x 50257 18 and 24 / 15 and 21 us, 671 x 100000 40 and 46 / 31 and 35 us.
    return vecs <= kMiddleRowVecs && (a.rows > 5 * 148 || a.rows <= 148) ? launch_rows<T, 128>(a, stream) : launch_rows<T, 256>(a, stream);
}

template <typename T, int kThreads>
cudaError_t launch_gradient(BwdArgs a, cudaStream_t stream) {
    constexpr int per_cta = kThreads * kUnroll * Elem<T>::kPerVec;
    a.chunks = int((a.V + (long long)per_cta - 1) / per_cta);
    if ((long long)a.rows * a.chunks > 0x7fffffffLL) return cudaErrorInvalidValue;
    // launched the ordinary way: its many short CTAs pay more for the dependency wait than the overlap gives (8192 x 3000: 21 us, 17 so)
    token_logprobs_bwd_kernel<T, kThreads><<<unsigned(a.rows) * unsigned(a.chunks), kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_backward(const BwdArgs& a, cudaStream_t stream) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.logits), d = reinterpret_cast<uintptr_t>(a.dlogits);
    const bool same_phase = ((x ^ d) & 15u) == 0 && ((a.row_stride - a.d_row_stride) * (long long)sizeof(T)) % 16 == 0;
    if (a.V <= kWarpGradVocab || !same_phase) {
        constexpr int rows = kWarpRowThreads / 32;
        return launch_pdl(token_logprobs_bwd_warp_kernel<T>, dim3((a.rows + rows - 1) / rows), dim3(kWarpRowThreads), 0, stream, a);
    }
    return a.V <= kSmallRowVecs * Elem<T>::kPerVec ? launch_gradient<T, 64>(a, stream) : launch_gradient<T, 256>(a, stream);
}

}  // namespace

extern "C" {

int b200loss_token_logprobs(const void* logits, int dtype, long long row_stride, const int* targets, int rows, int V,
                            float temperature, float* logprobs, float* entropy, float* stats, int top, float* top_logprobs,
                            int* top_tokens, void* stream) {
    const bool any_null = !logits || !targets || !logprobs || !entropy || !stats || (top > 0 && (!top_logprobs || !top_tokens));
    int rc = check_common("b200loss_token_logprobs: NULL pointer", any_null, dtype, rows, V, row_stride, temperature);
    if (rc) return rc;
    if (top < 0 || top > kMaxTop || top > V) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs: top must be between 0 and min(32, V)");
    if (rows == 0) return B200LOSS_OK;
    if (misaligned(logits, dtype == B200LOSS_F32 ? 4 : 2)) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs: logits are not aligned to their type");
    if (rows > 0x7fffffff / kMaxCluster) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs: too many rows");
    const FwdArgs a{logits, row_stride, targets, rows, V, 1.0f / temperature, logprobs, entropy, stats, top, top_logprobs, top_tokens};
    return finish(dtype == B200LOSS_F32 ? launch_forward<float>(a, (cudaStream_t)stream) : launch_forward<__nv_bfloat16>(a, (cudaStream_t)stream),
                  "b200loss_token_logprobs");
}

int b200loss_token_logprobs_backward(const void* logits, int dtype, long long row_stride, const int* targets, const float* entropy,
                                     const float* stats, const float* grad_logprobs, const float* grad_entropy, int rows, int V,
                                     float temperature, void* dlogits, long long d_row_stride, void* stream) {
    const bool any_null = !logits || !targets || !entropy || !stats || !grad_logprobs || !dlogits;
    int rc = check_common("b200loss_token_logprobs_backward: NULL pointer", any_null, dtype, rows, V, row_stride, temperature);
    if (rc) return rc;
    if (d_row_stride < V) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs_backward: d_row_stride is smaller than V");
    if (rows == 0) return B200LOSS_OK;
    const size_t size = dtype == B200LOSS_F32 ? 4 : 2;
    if (rows > 0x7fffffff / kMaxCluster) return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs_backward: too many rows");
    if (misaligned(logits, size) || misaligned(dlogits, size))
        return fail(B200LOSS_ERR_ARG, "b200loss_token_logprobs_backward: logits or dlogits are not aligned to their type");
    BwdArgs a{logits, row_stride, targets, entropy, stats, grad_logprobs, grad_entropy, rows, V, 1.0f / temperature, dlogits, d_row_stride, 1, -200.f * temperature * kLn2};
    return finish(dtype == B200LOSS_F32 ? launch_backward<float>(a, (cudaStream_t)stream) : launch_backward<__nv_bfloat16>(a, (cudaStream_t)stream),
                  "b200loss_token_logprobs_backward");
}

}  // extern "C"
