// Attention of one new query token per sequence over a cache of keys and values (sampling), sm_100a.
//
//   out[b, h] = softmax(scale * q[b, h] K[b, :len_b, h / G]^T) V[b, :len_b, h / G],   G = H / Hkv query heads to a key head
//
// Every key and value is read once and used for G heads only, so the bound is HBM, and what counts is bytes in flight and the shape
// of the requests. cp.async brings the rows of the next steps into shared memory, three steps per warp (192 KB per SM), a row by
// neighbouring lanes: the first version loaded every lane's 16-byte operands straight into registers (64 bytes of a row per
// request) and stayed at 4.7 TB/s however much was in flight; whole rows per request reach 5.8 TB/s. The operands of mma.sync
// m16n8k16, whose 16 rows are the heads of a group, are then read with 16-byte loads:
//   * Q K^T: the contraction index may be permuted freely as long as both operands agree, so lane (g, t) = (lane / 4, lane % 4)
//     takes 16 contiguous bytes of key g (dims 32c + 8t .. +7), which are its B fragments of two products; Q is read the same way.
//   * P V: the scores' accumulator layout is the A layout of the next product (keys 2t, 2t+1 and 2t+8, 2t+9 of 16). Lane (g, t)
//     takes dims 64e + 8g .. +7 of those four keys, 16 bytes each; pairs of keys are interleaved with a byte permute, and the
//     output columns are permuted with it: lane (g, t) ends with dims 64e + 16t .. +15 of head g.
// Groups of up to 8 heads leave rows 8-15 of the products empty (their accumulators are never kept).
//
// A CTA of four warps takes one split of one (sequence, key head); warp w takes the 16-key tiles w, w + 4, ... of it with its
// own running maximum and sum, and the warps meet in shared memory. The splits of a sequence are equal parts of ITS length
// (read on the device), so a long capacity with short lengths costs nothing. Up to eight splits are a cluster and join through
// distributed shared memory; more of them go to a workspace, which a second kernel joins. Either adds in a fixed order: results do
// not depend on timing.
#include <cooperative_groups.h>

#include "kernels.cuh"
#include "tc_common.cuh"

namespace b200attn {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 16;                      // keys per warp and step
constexpr int kStages = 3;                     // steps of K and V in flight per warp
constexpr int kRound = kTile * kWarps;         // keys of a CTA and step; a split is a multiple of it
constexpr int kLeastPart = 2 * kRound;         // keys of a split at least: fewer cost more to set up and to join than to read (the CTAs of a cluster are there anyway)
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoKey = -1e30f;               // running maximum before the first key (finite: differences of it are numbers)

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Asynchronous 16-byte copy to shared memory; zeros when `live` is false (nothing is read then).
__device__ __forceinline__ void copy16(uint4* dst, const __nv_bfloat16* src, bool live) {
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Keys of one split of a sequence of `len` keys (the last one may be shorter; splits past the end are empty).
__device__ __forceinline__ int chunk_of(int len, int splits, int least) {
    const int c = (len + splits - 1) / splits;
    return max(least, (c + kRound - 1) / kRound * kRound);
}
__device__ __forceinline__ int length_of(const DecodeArgs& a, int b) { return min(max(a.lengths[b], 0), a.T); }

__device__ __forceinline__ void write_out(const DecodeArgs& a, int b, int h, int D, int e, float M, float L, float x0, float x1) {
    const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);  // no keys: zeros; NaN stays NaN
    *reinterpret_cast<uint32_t*>(a.out + ((long long)b * a.H + h) * D + e) = pack_bf16x2(x0 * inv, x1 * inv);
    if (e == 0) a.lse[(long long)b * a.H + h] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// R = 8: the block of heads has at most 8; R = 16: up to 16. CLUSTER: the splits of a sequence are the CTAs of a cluster.
template <int D, int R, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 2) attn_decode_kernel(const DecodeArgs a) {
    constexpr int kRowsPerLane = R / 8;  // head g, and head g + 8
    constexpr int kSets = D / 32;        // 16-byte pieces of a key per lane
    constexpr int kHalves = D / 64;
    extern __shared__ __align__(16) float s_sums[];
    float (*s_o)[R][D] = reinterpret_cast<float (*)[R][D]>(s_sums);  // [warp][head][dim]
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];
    __shared__ float2 s_ml[CLUSTER ? R : 1];                              // this CTA's maximum and sum per head
    float2 (*s_part)[D / 2] = reinterpret_cast<float2 (*)[D / 2]>(s_sums + kWarps * R * D);  // and its output sums, [head][dim pair]

    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.y, b = blockIdx.z;
    const int kvh = blockIdx.x / a.head_blocks, block = blockIdx.x % a.head_blocks;
    const int h0 = kvh * a.G + block * R;          // first query head of this CTA
    const int rows = min(R, a.G - block * R);      // heads of it
    pdl_wait();
    const int len = length_of(a, b);
    const int chunk = chunk_of(len, a.splits, CLUSTER ? kRound : kLeastPart);
    const int begin = split * chunk, end = min(len, begin + chunk);
    if (!CLUSTER && begin >= end && a.splits > 1) return;  // an empty split is never joined

    uint32_t qf[kSets][2][4];  // A fragments of the two steps of every set
#pragma unroll
    for (int c = 0; c < kSets; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[c][i >> 2][i & 3] = 0u;
#pragma unroll
        for (int x = 0; x < kRowsPerLane; ++x) {
            if (g + 8 * x < rows) {
                const uint4 w = __ldg(reinterpret_cast<const uint4*>(a.q + (long long)b * a.q_stride + (long long)(h0 + g + 8 * x) * D + c * 32 + t * 8));
                qf[c][0][x] = w.x, qf[c][0][2 + x] = w.y, qf[c][1][x] = w.z, qf[c][1][2 + x] = w.w;
            }
        }
    }
    const __nv_bfloat16* kbase = a.k + (long long)b * a.k_batch + (long long)kvh * a.k_head;
    const __nv_bfloat16* vbase = a.v + (long long)b * a.v_batch + (long long)kvh * a.v_head;
    const float scale_log2 = a.scale * kLog2e;

    float o[kHalves][8][2 * kRowsPerLane];
#pragma unroll
    for (int e = 0; e < kHalves; ++e)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int x = 0; x < 2 * kRowsPerLane; ++x) o[e][j][x] = 0.f;
    float m[kRowsPerLane], l[kRowsPerLane];
#pragma unroll
    for (int x = 0; x < kRowsPerLane; ++x) m[x] = kNoKey, l[x] = 0.f;

    // A stage of this warp: 16 rows of K, then 16 rows of V, of kChunks 16-byte chunks. A row is copied by neighbouring lanes (whole
    // 128-byte lines go to L2). Chunks are exchanged inside a row so that eight lanes that read together meet eight bank groups:
    // K rows g, g + 1 at chunks 4c + t, V rows 2t at chunks 8e + g.
    constexpr int kChunks = D / 8, kRowsPerCopy = 32 / kChunks, kCopies = kTile / kRowsPerCopy;
    constexpr int kStage = 2 * kTile * kChunks;  // in 16-byte chunks
    uint4* ring = reinterpret_cast<uint4*>(s_sums) + warp * kStages * kStage;
    const int crow = lane / kChunks, cchunk = lane % kChunks;  // this lane's row and chunk of a copy's first rows
    int k_next = begin + warp * kTile;
    const __nv_bfloat16* kp = kbase + (long long)(k_next + crow) * a.k_row + cchunk * 8;
    const __nv_bfloat16* vp = vbase + (long long)(k_next + crow) * a.v_row + cchunk * 8;
    auto issue = [&](int stage) {
        if (k_next < end) {
            uint4* at = ring + stage * kStage;
            const bool whole = k_next + kTile <= end;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int row = i * kRowsPerCopy + crow;
                const bool live = whole || k_next + row < end;
                copy16(at + row * kChunks + (cchunk ^ ((row & 1) << 2)), live ? kp + i * kRowsPerCopy * a.k_row : kbase, live);
            }
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int row = i * kRowsPerCopy + crow;
                const bool live = whole || k_next + row < end;
                copy16(at + (kTile + row) * kChunks + (cchunk ^ (((row >> 1) & 3) << 1)), live ? vp + i * kRowsPerCopy * a.v_row : vbase, live);
            }
            k_next += kRound, kp += kRound * a.k_row, vp += kRound * a.v_row;
        }
        copy_commit();  // also where there is nothing left: the groups are counted
    };
    int k0 = begin + warp * kTile, stage = 0;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);
    for (; k0 < end; k0 += kRound) {
        copy_wait<kStages - 2>();
        __syncwarp();  // every lane's copies of this stage are there, and the stage before has been read by all
        issue(stage == 0 ? kStages - 1 : stage - 1);
        const uint4* at = ring + stage * kStage;
        stage = stage == kStages - 1 ? 0 : stage + 1;
        float s[2][4];
        {
            // four chains of products instead of two: a chain's length is what a lone warp waits for
            float s2[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[n][x] = s2[n][x] = 0.f;
#pragma unroll
            for (int c = 0; c < kSets; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const uint4 w = at[(8 * n + g) * kChunks + ((4 * c + t) ^ ((g & 1) << 2))];
                    mma16816(s[n], qf[c][0], w.x, w.y);
                    mma16816(s2[n], qf[c][1], w.z, w.w);
                }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[n][x] += s2[n][x];
        }
        uint32_t pf[4] = {0u, 0u, 0u, 0u};
        float alpha[kRowsPerLane];
        bool moved = false;
#pragma unroll
        for (int x = 0; x < kRowsPerLane; ++x) {
            float mx = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float& v = s[n][2 * x + y];
                    v = k0 + 8 * n + 2 * t + y < end ? v * scale_log2 : -INFINITY;
                    mx = fmaxf(mx, v);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m[x], mx);
            alpha[x] = fast_exp2(m[x] - m_new);
            moved |= m_new > m[x];
            m[x] = m_new;
            float p[2][2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int y = 0; y < 2; ++y) p[n][y] = fast_exp2(s[n][2 * x + y] - m_new);
            l[x] = l[x] * alpha[x] + ((p[0][0] + p[0][1]) + (p[1][0] + p[1][1]));
            // P enters its product in BF16, as in the other tensor-core paths; the sum l is of the FP32 values
            pf[x] = pack_bf16x2(p[0][0], p[0][1]);
            pf[2 + x] = pack_bf16x2(p[1][0], p[1][1]);
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int e = 0; e < kHalves; ++e)
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int x = 0; x < 2 * kRowsPerLane; ++x) o[e][j][x] *= alpha[x >> 1];
        }
#pragma unroll
        for (int e = 0; e < kHalves; ++e) {
            uint32_t w[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 x = at[(kTile + 2 * t + (i & 1) + 8 * (i >> 1)) * kChunks + ((8 * e + g) ^ (t << 1))];
                w[i][0] = x.x, w[i][1] = x.y, w[i][2] = x.z, w[i][3] = x.w;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                const uint32_t b0 = __byte_perm(w[0][j >> 1], w[1][j >> 1], sel), b1 = __byte_perm(w[2][j >> 1], w[3][j >> 1], sel);
                float acc[4] = {o[e][j][0], o[e][j][1], 0.f, 0.f};
                if (kRowsPerLane == 2) acc[2] = o[e][j][2 * kRowsPerLane - 2], acc[3] = o[e][j][2 * kRowsPerLane - 1];
                mma16816(acc, pf, b0, b1);
                o[e][j][0] = acc[0], o[e][j][1] = acc[1];
                if (kRowsPerLane == 2) o[e][j][2 * kRowsPerLane - 2] = acc[2], o[e][j][2 * kRowsPerLane - 1] = acc[3];
            }
        }
    }
    // the warps of the CTA meet, over the stages: every warp leaves its sums relative to its own maximum
    copy_wait<0>();
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kRowsPerLane; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        if (t == 0) s_m[warp][g + 8 * x] = m[x], s_l[warp][g + 8 * x] = l[x];
#pragma unroll
        for (int e = 0; e < kHalves; ++e)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    *reinterpret_cast<float4*>(&s_o[warp][g + 8 * x][e * 64 + 16 * t + 8 * y + j]) =
                        make_float4(o[e][j][2 * x + y], o[e][j + 1][2 * x + y], o[e][j + 2][2 * x + y], o[e][j + 3][2 * x + y]);
    }
    __syncthreads();
    for (int i = tid; i < rows * (D / 2); i += kThreads) {
        const int row = i / (D / 2), e = (i % (D / 2)) * 2;
        float M = kNoKey;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][row]);
        float L = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {  // a warp without keys has zeros
            const float f = fast_exp2(s_m[w][row] - M);
            L += s_l[w][row] * f;
            x0 = fmaf(s_o[w][row][e], f, x0), x1 = fmaf(s_o[w][row][e + 1], f, x1);
        }
        const int h = h0 + row;
        if constexpr (CLUSTER) {
            s_part[row][e / 2] = make_float2(x0, x1);
            if (e == 0) s_ml[row] = make_float2(M, L);
        } else if (a.splits == 1) {
            write_out(a, b, h, D, e, M, L, x0, x1);
        } else {
            const long long part = ((long long)b * a.H + h) * a.splits + split;
            *reinterpret_cast<float2*>(a.part_o + part * D + e) = make_float2(x0, x1);
            if (e == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = make_float2(M, L);
        }
    }
    if constexpr (CLUSTER) {  // every CTA joins its share of the outputs
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        for (int i = split * kThreads + tid; i < rows * (D / 2); i += a.splits * kThreads) {
            const int row = i / (D / 2), e = i % (D / 2);
            float2 ml[kMaxCluster], x[kMaxCluster];
            float M = kNoKey, L = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
            for (int p = 0; p < kMaxCluster; ++p) {
                if (p >= a.splits) break;
                ml[p] = *cluster.map_shared_rank(&s_ml[row], p);
                x[p] = *cluster.map_shared_rank(&s_part[row][e], p);
                M = fmaxf(M, ml[p].x);
            }
#pragma unroll
            for (int p = 0; p < kMaxCluster; ++p) {
                if (p >= a.splits) break;
                const float f = fast_exp2(ml[p].x - M);
                L = fmaf(ml[p].y, f, L), x0 = fmaf(x[p].x, f, x0), x1 = fmaf(x[p].y, f, x1);
            }
            write_out(a, b, h0 + row, D, 2 * e, M, L, x0, x1);
        }
        cluster.sync();  // the others have read this CTA's shared memory
    }
}

// One CTA per (sequence, head): joins the splits that hold keys. The sums are added in an order that depends on their number only.
constexpr int kJoinThreads = 512;  // a warp reads a split's sums at once; each has few splits, all under way together
constexpr int kMaxSplits = 256;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) attn_decode_join_kernel(const DecodeArgs a) {
    constexpr int kGroups = kJoinThreads / 32, kVec = D / 32;
    __shared__ float s_f[kMaxSplits];
    __shared__ float s_x[kGroups][D];
    __shared__ float s_red[2][kJoinThreads / 32];
    pdl_launch_dependents();
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    const int len = length_of(a, b), chunk = chunk_of(len, a.splits, kLeastPart), n = (len + chunk - 1) / chunk;
    const long long part = ((long long)b * a.H + h) * a.splits;
    // thread i weighs split i
    const float2 ml = tid < n ? reinterpret_cast<const float2*>(a.part_ml)[part + tid] : make_float2(kNoKey, 0.f);
    float M = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0) s_red[0][warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) M = fmaxf(M, s_red[0][w]);
    const float f = fast_exp2(ml.x - M);
    if (tid < kMaxSplits) s_f[tid] = f;
    float L = ml.y * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) s_red[1][warp] = L;
    __syncthreads();
    L = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) L += s_red[1][w];
    float x[kVec];
#pragma unroll
    for (int c = 0; c < kVec; ++c) x[c] = 0.f;
#pragma unroll 8
    for (int i = warp; i < n; i += kGroups) {
        const float* from = a.part_o + (part + i) * D + lane * kVec;
        float y[kVec];
        if constexpr (kVec == 4) *reinterpret_cast<float4*>(y) = *reinterpret_cast<const float4*>(from);
        else *reinterpret_cast<float2*>(y) = *reinterpret_cast<const float2*>(from);
#pragma unroll
        for (int c = 0; c < kVec; ++c) x[c] = fmaf(y[c], s_f[i], x[c]);
    }
#pragma unroll
    for (int c = 0; c < kVec; ++c) s_x[warp][lane * kVec + c] = x[c];
    __syncthreads();
    if (tid < D / 2) {
        float x0 = 0.f, x1 = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) x0 += s_x[i][2 * tid], x1 += s_x[i][2 * tid + 1];
        write_out(a, b, h, D, 2 * tid, M, L, x0, x1);
    }
}

template <int D, int R>
cudaError_t launch(const DecodeArgs& a, cudaStream_t stream) {
    constexpr int stages = kWarps * kStages * kTile * D * 2 * 2, sums = (kWarps + 1) * R * D * int(sizeof(float));
    constexpr int smem = stages > sums ? stages : sums;
    const bool cluster = a.splits > 1 && a.splits <= kMaxCluster;
    auto kern = cluster ? attn_decode_kernel<D, R, true> : attn_decode_kernel<D, R, false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid(a.Hkv * a.head_blocks, a.splits, a.B);
    e = cluster ? launch_pdl_cluster(kern, grid, dim3(1, a.splits, 1), dim3(kThreads), smem, stream, a)
                : launch_pdl(kern, grid, dim3(kThreads), smem, stream, a);
    if (e != cudaSuccess || a.splits == 1 || cluster) return e;
    return launch_pdl(attn_decode_join_kernel<D>, dim3(a.H, a.B), dim3(kJoinThreads), 0, stream, a);
}

}  // namespace

bool decode_needs_workspace(int splits) { return splits > kMaxCluster; }
int decode_splits(int B, int T, int H, int Hkv, int d) {
    const int G = H / Hkv, R = G <= 8 ? 8 : 16;
    const long long items = (long long)B * Hkv * ((G + R - 1) / R);
    // What a CTA costs beside its keys (some 4 us from launch to join) is paid once per round of the CTAs that the card holds, so: one
    // round, or as many full ones as it takes for a split of the longest sequence the cache can hold to have no more than 1280 keys
    // (768 of 64 dims), up to four; sequences differ in length, and short splits even that out. One sequence alone needs no evening
    // out. Measured against six CTAs per SM whatever the lengths (us, that / this): 65 sequences up to 392 keys, 8 key heads, d 128 20.5 /
    // 11.5, 86 up to 989, 1 key head 17.7 / 8.5, 47 up to 1166, 4 key heads 30 / 19, 64 up to 4096, 8 key heads 69 / 69, one of 131,000
    // 76.7 / 73.6 (a round and a part of the next: 79.6), 16 up to 16384, 4 key heads, d 64 21.8 / 20.8; 18 up to 4035, 4 key heads, d 128
    // the other way: 16.0 / 18.8.
    const long long resident = (d == 64 ? 4 : 2) * 148, keys = d == 64 ? 768 : 1280, alone = resident / items > 1 ? resident / items : 1;
    long long want = (T + keys - 1) / keys;
    if (want > 4 * resident / items) want = 4 * resident / items;
    if (want < alone || B == 1) want = alone;
    const long long rounds = (want * items + resident - 1) / resident;
    long long splits = rounds * resident / items;
    const long long most = (T + kLeastPart - 1) / kLeastPart;
    if (splits > most) splits = most;
    if (splits > kMaxSplits) splits = kMaxSplits;
    return splits < 1 ? 1 : int(splits);
}

cudaError_t launch_attn_decode(DecodeArgs a, cudaStream_t stream) {
    a.G = a.H / a.Hkv;
    const int R = a.G <= 8 ? 8 : 16;
    a.head_blocks = (a.G + R - 1) / R;
    if (a.Hkv * (long long)a.head_blocks > 65535 || a.B > 65535) return cudaErrorInvalidValue;
    if (a.d == 64) return R == 8 ? launch<64, 8>(a, stream) : launch<64, 16>(a, stream);
    if (a.d == 128) return R == 8 ? launch<128, 8>(a, stream) : launch<128, 16>(a, stream);
    return cudaErrorInvalidValue;
}

}  // namespace b200attn
