// Attention of one new query token per sequence over a cache of keys and values (sampling), sm_100a.
//
//   out[b, h] = softmax(scale * q[b, h] K[b, :len_b, h / G]^T) V[b, :len_b, h / G],   G = H / Hkv query heads to a key head
//
// Every key and value is read once and used for G heads only, so the bound is HBM and nothing needs staging: the operands of
// the products go from global memory straight into the registers of mma.sync m16n8k16, whose 16 rows are the heads of a group.
//   * Q K^T: the contraction index may be permuted freely as long as both operands agree, so lane (g, t) = (lane / 4, lane % 4)
//     takes 16 contiguous bytes of key g (dims 32c + 8t .. +7), which are its B fragments of two steps; Q is read the same way.
//   * P V: the scores' accumulator layout is the A layout of the next product (keys 2t, 2t+1 and 2t+8, 2t+9 of 16). Lane (g, t)
//     takes dims 64e + 8g .. +7 of those four keys, 16 bytes each; pairs of keys are interleaved with a byte permute, and the
//     output columns are permuted with it: lane (g, t) ends with dims 64e + 16t .. +15 of head g.
// Groups of up to 8 heads leave rows 8-15 of the products empty (their accumulators are never kept).
//
// A CTA of eight warps takes one split of one (sequence, key head); warp w takes the 16-key tiles w, w + 8, ... of it with its
// own running maximum and sum, and the warps meet in shared memory. The splits of a sequence are equal parts of ITS length
// (read on the device), so a long capacity with short lengths costs nothing. With more than one split the parts go to a
// workspace and a second kernel joins them in a fixed order: results do not depend on timing.
#include "kernels.cuh"
#include "tc_common.cuh"

namespace b200attn {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = 16;                      // keys per warp and step
constexpr int kMinChunk = kTile * kWarps;      // keys of a split, at least: one tile for every warp
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoKey = -1e30f;               // running maximum before the first key (finite: differences of it are numbers)

__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Streaming 16-byte load (every key and value is read once).
__device__ __forceinline__ uint4 load_stream(const __nv_bfloat16* p) {
    uint4 w;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(p));
    return w;
}

// Keys of one split of a sequence of `len` keys (the last one may be shorter; splits past the end are empty).
__device__ __forceinline__ int chunk_of(int len, int splits) {
    const int c = (len + splits - 1) / splits;
    return max(kMinChunk, (c + kTile - 1) / kTile * kTile);
}
__device__ __forceinline__ int length_of(const DecodeArgs& a, int b) { return min(max(a.lengths[b], 0), a.T); }

// R = 8: the block of heads has at most 8; R = 16: up to 16.
template <int D, int R>
__global__ void __launch_bounds__(kThreads) attn_decode_kernel(const DecodeArgs a) {
    constexpr int kRowsPerLane = R / 8;  // head g, and head g + 8
    constexpr int kSets = D / 32;        // 16-byte pieces of a key per lane
    constexpr int kHalves = D / 64;
    extern __shared__ __align__(16) float s_sums[];
    float (*s_o)[R][D] = reinterpret_cast<float (*)[R][D]>(s_sums);  // [warp][head][dim]
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];

    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, b = blockIdx.z;
    const int kvh = blockIdx.y / a.head_blocks, block = blockIdx.y % a.head_blocks;
    const int h0 = kvh * a.G + block * R;          // first query head of this CTA
    const int rows = min(R, a.G - block * R);      // heads of it
    pdl_wait();
    const int len = length_of(a, b);
    const int chunk = chunk_of(len, a.splits);
    const int begin = split * chunk, end = min(len, begin + chunk);
    if (begin >= end && !(split == 0 && a.splits == 1)) return;  // an empty split is never joined

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

    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 kf[2][kSets];
    auto load_keys = [&](int k0) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int key = k0 + 8 * n + g;
            const __nv_bfloat16* p = kbase + (long long)key * a.k_row + t * 8;
#pragma unroll
            for (int c = 0; c < kSets; ++c) kf[n][c] = key < end ? load_stream(p + c * 32) : zero;
        }
    };
    int k0 = begin + warp * kTile;
    if (k0 < end) load_keys(k0);
    for (; k0 < end; k0 += kTile * kWarps) {
        uint4 vf[kHalves][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = k0 + 2 * t + (i & 1) + 8 * (i >> 1);
            const __nv_bfloat16* p = vbase + (long long)key * a.v_row + g * 8;
#pragma unroll
            for (int e = 0; e < kHalves; ++e) vf[e][i] = key < end ? load_stream(p + e * 64) : zero;
        }
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int x = 0; x < 4; ++x) s[n][x] = 0.f;
#pragma unroll
            for (int c = 0; c < kSets; ++c) {
                mma16816(s[n], qf[c][0], kf[n][c].x, kf[n][c].y);
                mma16816(s[n], qf[c][1], kf[n][c].z, kf[n][c].w);
            }
        }
        if (k0 + kTile * kWarps < end) load_keys(k0 + kTile * kWarps);
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
            const uint32_t w[4][4] = {{vf[e][0].x, vf[e][0].y, vf[e][0].z, vf[e][0].w}, {vf[e][1].x, vf[e][1].y, vf[e][1].z, vf[e][1].w},
                                      {vf[e][2].x, vf[e][2].y, vf[e][2].z, vf[e][2].w}, {vf[e][3].x, vf[e][3].y, vf[e][3].z, vf[e][3].w}};
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
    // the warps of the CTA meet: every warp leaves its sums relative to its own maximum
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
        if (a.splits == 1) {
            const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);  // no keys: zeros; NaN stays NaN
            *reinterpret_cast<uint32_t*>(a.out + ((long long)b * a.H + h) * D + e) = pack_bf16x2(x0 * inv, x1 * inv);
            if (e == 0) a.lse[(long long)b * a.H + h] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        } else {
            const long long part = ((long long)b * a.H + h) * a.splits + split;
            *reinterpret_cast<float2*>(a.part_o + part * D + e) = make_float2(x0, x1);
            if (e == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = make_float2(M, L);
        }
    }
}

// One CTA per (sequence, head): joins the splits that hold keys, in their order.
template <int D>
__global__ void __launch_bounds__(D / 2) attn_decode_join_kernel(const DecodeArgs a) {
    pdl_launch_dependents();
    const int h = blockIdx.x, b = blockIdx.y, e = threadIdx.x * 2;
    pdl_wait();
    const int len = length_of(a, b), chunk = chunk_of(len, a.splits), n = (len + chunk - 1) / chunk;
    const long long part = ((long long)b * a.H + h) * a.splits;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + part;
    float M = kNoKey;
    for (int i = 0; i < n; ++i) M = fmaxf(M, ml[i].x);
    float L = 0.f, x0 = 0.f, x1 = 0.f;
    for (int i = 0; i < n; ++i) {
        const float f = fast_exp2(ml[i].x - M);
        const float2 x = *reinterpret_cast<const float2*>(a.part_o + (part + i) * D + e);
        L += ml[i].y * f;
        x0 = fmaf(x.x, f, x0), x1 = fmaf(x.y, f, x1);
    }
    const float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);
    *reinterpret_cast<uint32_t*>(a.out + ((long long)b * a.H + h) * D + e) = pack_bf16x2(x0 * inv, x1 * inv);
    if (e == 0) a.lse[(long long)b * a.H + h] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

template <int D, int R>
cudaError_t launch(const DecodeArgs& a, cudaStream_t stream) {
    constexpr int smem = kWarps * R * D * int(sizeof(float));
    cudaError_t e = cudaFuncSetAttribute(attn_decode_kernel<D, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(attn_decode_kernel<D, R>, dim3(a.splits, a.Hkv * a.head_blocks, a.B), dim3(kThreads), smem, stream, a);
    if (e != cudaSuccess || a.splits == 1) return e;
    return launch_pdl(attn_decode_join_kernel<D>, dim3(a.H, a.B), dim3(D / 2), 0, stream, a);
}

}  // namespace

int decode_splits(int B, int T, int H, int Hkv) {
    const int G = H / Hkv, R = G <= 8 ? 8 : 16;
    const long long items = (long long)B * Hkv * ((G + R - 1) / R);
    // enough CTAs for several rounds of the card (sequences differ in length), of at least two tiles per warp each
    long long splits = (148 * 8 + items - 1) / items;
    const long long most = (T + 2 * kMinChunk - 1) / (2 * kMinChunk);
    if (splits > most) splits = most;
    if (splits > 256) splits = 256;
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
