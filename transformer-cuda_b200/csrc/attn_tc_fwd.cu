// Causal attention forward on the sm_100a tensor cores (tcgen05), BF16 operands, FP32
// accumulation and FP32 softmax statistics. Computes what tiled_causal_attention_forward of
// sarimahsan/transformer-cuda computes (src/kernels/attention.cu:518-657): O = softmax(scale*QK^T
// + causal mask) V with the row maximum m and the un-normalised row sum l exported.
//
// One CTA owns one 128-row query tile of one (batch, head) slab and walks the key/value tiles
// 0..diagonal (tiles above the diagonal are never loaded). Ten warps, three roles:
//
//   warps 0-7  softmax: query row r (TMEM lane r) is shared by two threads, (r, 0) in warps 0-3 and
//              (r, 1) in warps 4-7, which take key columns [0,64) and [64,128) of the tile. S_j is
//              read from TMEM with tcgen05.ld; the two halves of a row exchange their partial row
//              maximum through shared memory, turn their columns into P_j = exp2(S_j*scale*log2e - m)
//              in BF16 and write them back over their own S columns in TMEM, where the P.V MMA reads
//              them as its A operand. Row sums stay per thread and meet in the epilogue. The same
//              threads rescale the O accumulator in TMEM when the running maximum has moved by more
//              than 2^8, and run the epilogue.
//   warp 8     TMA producer: Q once, then a ring of K and V tiles (cp.async.bulk.tensor, 128-byte
//              swizzle, no multicast), each signalled through an mbarrier with expect_tx.
//   warp 9     MMA issuer: S_j = Q K_j^T (both operands K-major in shared memory) into one of three
//              TMEM score buffers, and O += P_j V_j (A from TMEM, V as an MN-major shared-memory
//              operand, so no transpose is materialised). QK^T runs two tiles ahead of P.V: MMAs
//              execute in issue order, so with only one tile of lead every QK^T would queue behind a
//              P.V that is itself waiting for the softmax warps.
//
// TMEM columns: [0,128) [128,256) [256,384) S/P buffers 0-2, [384,384+D) O.
// Every mbarrier wait has an iteration limit (tc_common.cuh); a wait that gives up sets the fault
// word and the kernel still runs to its end and frees its TMEM.
#include "kernels.cuh"
#include "ragged_items.cuh"
#include "tc_common.cuh"


namespace b200attn {
namespace {

constexpr int kBM = 128;                 // query rows per CTA
constexpr int kBN = 128;                 // key/value rows per tile
constexpr int kAtomBytes = 128 * 128;    // one TMA box: 128 rows x 64 bf16, 128-byte swizzled
constexpr int kSoftmaxThreads = 256;
constexpr int kThreads = 320;
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kHalfCols = kBN / 2;       // key columns per softmax thread
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <int D>
struct FwdCfg {
    static constexpr int kAtoms = D / 64;
    static constexpr int kTileBytes = kAtoms * kAtomBytes;
    static constexpr int kKStages = 3;  // K is consumed two tiles ahead of V
    static constexpr int kVStages = (D == 64) ? 4 : 3;
    static constexpr int kSBuffers = 3;
    static constexpr int kSmemBytes = kTileBytes * (1 + kKStages + kVStages);  // dynamic buffer is declared 1024-aligned
    static constexpr uint32_t kTmemCols = 512;
    static constexpr uint32_t kColS = 0, kColO = 384;  // score buffer b at columns 128*b
};

struct FwdBarriers {
    uint64_t q_full;
    uint64_t k_full[4], v_full[4], k_empty[4], v_empty[4];
    uint64_t s_full[3], p_full[3];
    uint64_t o_done;
};

// RAGGED: packed sequences with grouped heads, where the card is not full; every CTA finds its tile in the offsets.
template <int D, bool OUT_F32, bool RAGGED>
__global__ void __launch_bounds__(kThreads, 1) attn_fwd_tc_kernel(const __grid_constant__ TcFwdArgs a) {
    using Cfg = FwdCfg<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;
    uint8_t* sK = smem + Cfg::kTileBytes;
    uint8_t* sV = sK + Cfg::kKStages * Cfg::kTileBytes;

    __shared__ FwdBarriers bars;
    __shared__ uint32_t tmem_base_slot;
    __shared__ uint32_t abort_flag;
    __shared__ float s_xchg[2][2][kBM];  // [tile parity][half][row]: partial row maxima, then row sums

    const int tid = threadIdx.x;
    const int warp = tid >> 5;
    const int lane = tid & 31;
    pdl_launch_dependents();

    const int n_q_tiles = (a.T + kBM - 1) / kBM;
    // CTA order: the last query tile of a slab is the longest. Longest-first across all slabs when the
    // problem fits in L2 (shortest tail), else slab by slab (resident CTAs share K/V tiles in L2).
    int bh = 0, qt = 0, hh = 0, bb = 0, hk = 0;  // hh, bb: head and batch coordinates of the 4-D tensor maps; hk: key head
    int row0 = 0, valid = kBM;                   // RAGGED: first row of the sequence, rows of this tile that belong to it
    if constexpr (!RAGGED) {
        bh = a.tile_major_order ? int(blockIdx.x % a.BH) : int(blockIdx.x / n_q_tiles);
        qt = n_q_tiles - 1 - (a.tile_major_order ? int(blockIdx.x / a.BH) : int(blockIdx.x % n_q_tiles));
        hh = bh % a.H, bb = bh / a.H, hk = hh;
    }

    if (tid == 0) {
        mbar_init(&bars.q_full, 1);
        for (int s = 0; s < 4; ++s) {
            mbar_init(&bars.k_full[s], 1);
            mbar_init(&bars.v_full[s], 1);
            mbar_init(&bars.k_empty[s], 1);
            mbar_init(&bars.v_empty[s], 1);
        }
        for (int b = 0; b < 3; ++b) {
            mbar_init(&bars.s_full[b], 1);
            mbar_init(&bars.p_full[b], kSoftmaxThreads);
        }
        mbar_init(&bars.o_done, 1);
        abort_flag = 0;
        if ((smem_u32(smem) & 1023u) != 0 && a.fault_word) atomicCAS(a.fault_word, 0u, kFaultWaitTimeout | 0xA10u);
        mbar_fence_init();
    }
    if (warp == kProducerWarp) {
        if (RAGGED && lane == 0) {  // under the set-up
            tma_prefetch_desc(&a.map_q);
            tma_prefetch_desc(&a.map_k);
            tma_prefetch_desc(&a.map_v);
        }
        tmem_alloc(&tmem_base_slot, Cfg::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_slot;
    // barriers, TMEM and the tensor maps are set up: from here on global memory is touched, so wait for the
    // kernel in front of this one in the stream (returns at once for an ordinary launch)
    pdl_wait();
    if constexpr (RAGGED) {
        const int4 w = ragged_find(a.ragged.offsets, a.ragged.n, a.T, int(blockIdx.x / unsigned(a.H)), lane);
        if (w.z == 0) {  // the host knows an upper bound only
            __syncthreads();
            if (warp == kProducerWarp) tmem_dealloc(tmem, Cfg::kTmemCols);
            return;
        }
        bh = hh = int(blockIdx.x % unsigned(a.H)), hk = hh / a.ragged.group;
        row0 = w.x, qt = w.z - 1, valid = min(kBM, w.y - qt * kBM);
    }
    const int n_kv = qt + 1;  // key tiles 0..qt; qt is the diagonal tile

    if (warp == kProducerWarp) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            if (!RAGGED) {
                tma_prefetch_desc(&a.map_q);
                tma_prefetch_desc(&a.map_k);
                tma_prefetch_desc(&a.map_v);
            }
            mbar_expect_tx(&bars.q_full, Cfg::kTileBytes);
            for (int at = 0; at < Cfg::kAtoms; ++at)
                tma_load_4d(sQ + at * kAtomBytes, &a.map_q, &bars.q_full, at * 64, row0 + qt * kBM, hh, bb);
            for (int j = 0; j < n_kv; ++j) {
                const int ks = j % Cfg::kKStages, kround = j / Cfg::kKStages;
                if (kround > 0) mbar_wait(&bars.k_empty[ks], (kround - 1) & 1, &abort_flag, a.fault_word, 0x10);
                mbar_expect_tx(&bars.k_full[ks], Cfg::kTileBytes);
                for (int at = 0; at < Cfg::kAtoms; ++at)
                    tma_load_4d(sK + ks * Cfg::kTileBytes + at * kAtomBytes, &a.map_k, &bars.k_full[ks], at * 64, row0 + j * kBN, hk, bb);
                const int vs = j % Cfg::kVStages, vround = j / Cfg::kVStages;
                if (vround > 0) mbar_wait(&bars.v_empty[vs], (vround - 1) & 1, &abort_flag, a.fault_word, 0x11);
                mbar_expect_tx(&bars.v_full[vs], Cfg::kTileBytes);
                for (int at = 0; at < Cfg::kAtoms; ++at)
                    tma_load_4d(sV + vs * Cfg::kTileBytes + at * kAtomBytes, &a.map_v, &bars.v_full[vs], at * 64, row0 + j * kBN, hk, bb);
            }
        }
        __syncwarp();
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t idesc_qk = make_idesc_bf16(kBM, kBN, 0, 0);
        constexpr uint32_t idesc_pv = make_idesc_bf16(kBM, D, 0, 1);
        const uint64_t q_desc = make_smem_desc_sw128(smem_u32(sQ), 0, 1024);
        mbar_wait(&bars.q_full, 0, &abort_flag, a.fault_word, 0x20);
        // S[j % 3] = Q K_j^T. The buffer is free: P_{j-3} V_{j-3} was issued before, and MMAs run in order.
        auto issue_qk = [&](int j) {
            const int ks = j % Cfg::kKStages;
            mbar_wait(&bars.k_full[ks], (j / Cfg::kKStages) & 1, &abort_flag, a.fault_word, 0x21);
            tc_fence_after();
            if (elect_one()) {
                const uint64_t k_desc = make_smem_desc_sw128(smem_u32(sK + ks * Cfg::kTileBytes), 0, 1024);
                const uint32_t d_tmem = tmem + Cfg::kColS + (j % Cfg::kSBuffers) * 128;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * kAtomBytes + (kk & 3) * 32;
                    tc_mma_ss(d_tmem, desc_advance(q_desc, off), desc_advance(k_desc, off), idesc_qk, kk > 0);
                }
                tc_commit(&bars.k_empty[ks]);
                tc_commit(&bars.s_full[j % Cfg::kSBuffers]);
            }
            __syncwarp();
        };
        issue_qk(0);
        if (n_kv > 1) issue_qk(1);
        for (int j = 0; j < n_kv; ++j) {
            if (j + 2 < n_kv) issue_qk(j + 2);  // does not depend on the softmax of tile j
            // O += P_j V_j
            const int vs = j % Cfg::kVStages;
            const int b = j % Cfg::kSBuffers;
            mbar_wait(&bars.v_full[vs], (j / Cfg::kVStages) & 1, &abort_flag, a.fault_word, 0x22);
            if constexpr (RAGGED) {  // keys behind the sequence have P = 0, whatever their values hold
                if (j == qt && valid < kBN) zero_tile_rows<128>(sV + vs * Cfg::kTileBytes, Cfg::kAtoms, valid, lane);
            }
            mbar_wait(&bars.p_full[b], (j / Cfg::kSBuffers) & 1, &abort_flag, a.fault_word, 0x23);
            tc_fence_after();
            if (elect_one()) {
                // V tile: rows = key index (the MMA's K), 64-column atoms along the head dim (its N)
                const uint64_t v_desc = make_smem_desc_sw128(smem_u32(sV + vs * Cfg::kTileBytes), kAtomBytes, 1024);
                const uint32_t p_tmem = tmem + Cfg::kColS + b * 128;
                // keys 0-63 of the tile are packed in columns [0,32) of the buffer, keys 64-127 in [64,96)
#pragma unroll
                for (int kk = 0; kk < kBN / 16; ++kk)
                    tc_mma_ts(tmem + Cfg::kColO, p_tmem + (kk >> 2) * kHalfCols + (kk & 3) * 8,
                              desc_advance(v_desc, kk * 2048), idesc_pv, (j > 0) || (kk > 0));
                tc_commit(&bars.v_empty[vs]);
                tc_commit(&bars.o_done);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------ softmax + correction + epilogue
        const int r = tid & 127;                              // query row inside the tile, TMEM lane
        const int half = tid >> 7;                            // which 64 key columns of a tile
        const uint32_t lane_base = uint32_t(warp & 3) * 32u;  // this warp's TMEM lane quadrant
        const int c_begin = half * kHalfCols;
        const float scale_log2 = a.scale * kLog2e;
        // Exponents are taken relative to m_ref, which follows the true running maximum m_true only
        // when that has moved by more than kRescaleThreshold (in log2 units): P stays below
        // 2^threshold, and the O accumulator in TMEM has to be rescaled only on those rare moves.
        // Both threads of a row see the same maxima and so take the same decisions.
        constexpr float kRescaleThreshold = 8.0f;
        float m_true = -INFINITY;  // running maximum of scale*log2e*s over the whole row
        float m_ref = -INFINITY;   // reference the exponentials and l_run are relative to
        float l_run = 0.f;         // this thread's share of the row sum
        for (int j = 0; j < n_kv; ++j) {
            const int sb = j % Cfg::kSBuffers;
            const uint32_t s_col = Cfg::kColS + sb * 128 + c_begin;
            mbar_wait(&bars.s_full[sb], (j / Cfg::kSBuffers) & 1, &abort_flag, a.fault_word, 0x30);
            tc_fence_after();
            uint32_t sv[kHalfCols];
#pragma unroll
            for (int c = 0; c < kHalfCols; c += 32) tmem_ld32(tmem_addr(tmem, lane_base, s_col + c), &sv[c]);
            tmem_wait_ld();
            if (j == qt) {  // diagonal tile: key c is visible to query r iff c <= r
#pragma unroll
                for (int c = 0; c < kHalfCols; ++c)
                    if (c_begin + c > r) sv[c] = 0xff800000u;  // -inf
            }
            // four independent chains instead of one running maximum of 64 dependent instructions
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kHalfCols; c += 4) {
#pragma unroll
                for (int y = 0; y < 4; ++y) mx4[y] = fmaxf(mx4[y], __uint_as_float(sv[c + y]));
            }
            float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            // row maximum over both halves (the buffer alternates with the tile parity, so one barrier per tile is enough)
            s_xchg[j & 1][half][r] = mx;
            named_bar_sync(1, kSoftmaxThreads);
            mx = fmaxf(mx, s_xchg[j & 1][half ^ 1][r]);
            m_true = fmaxf(m_true, mx * scale_log2);
            const bool move = (j == 0) || (m_true - m_ref > kRescaleThreshold);
            float alpha = 1.0f;
            if (move) {
                alpha = fast_exp2(m_ref - m_true);  // 0 on the first tile
                m_ref = m_true;
            }
            // scale-and-shift and row sums on packed pairs (fma2 / add2): five instructions per pair of scores instead of seven
            float2 sum2[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
            uint32_t pk[kHalfCols / 2];
            const float neg_ref = -m_ref;
#pragma unroll
            for (int c = 0; c < kHalfCols; c += 2) {
                const float2 arg = fma2(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1]), scale_log2, neg_ref);
                const float p0 = mixed_exp2(arg.x, c);
                const float p1 = mixed_exp2(arg.y, c + 1);
                sum2[(c >> 1) & 3] = add2(sum2[(c >> 1) & 3], p0, p1);
                pk[c >> 1] = pack_bf16x2(p0, p1);
            }
            l_run = l_run * alpha + (((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y)) + ((sum2[2].x + sum2[2].y) + (sum2[3].x + sum2[3].y)));
            // each half packs its P into the first 32 columns of its OWN 64 score columns
            tmem_st32(tmem_addr(tmem, lane_base, s_col), pk);
            if (j > 0 && __any_sync(0xffffffffu, move)) {
                // bring this thread's half of the O accumulator to the new reference (rows that did not move
                // use alpha = 1); O is complete up to tile j-1 once its P.V has retired
                mbar_wait(&bars.o_done, (j - 1) & 1, &abort_flag, a.fault_word, 0x31);
                tc_fence_after();
#pragma unroll
                for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
                    uint32_t ov[32];
                    tmem_ld32(tmem_addr(tmem, lane_base, Cfg::kColO + c), ov);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                    tmem_st32(tmem_addr(tmem, lane_base, Cfg::kColO + c), ov);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars.p_full[sb]);
        }
        // ---- epilogue: O / l
        // the two halves of a row add up their sums (buffer parity n_kv & 1 was last used two tiles ago)
        s_xchg[n_kv & 1][half][r] = l_run;
        named_bar_sync(1, kSoftmaxThreads);
        l_run += s_xchg[n_kv & 1][half ^ 1][r];
        mbar_wait(&bars.o_done, (n_kv - 1) & 1, &abort_flag, a.fault_word, 0x32);
        tc_fence_after();
        const float inv_l = 1.0f / l_run;
        const int row_g = row0 + qt * kBM + r;
        const bool in_range = RAGGED ? r < valid : row_g < a.T;
        const long long stat_idx = (long long)bh * a.T + row_g;
        if (in_range && half == 0) {
            // exported statistics are relative to the true row maximum
            if (a.m_out) a.m_out[stat_idx] = m_true * kLn2;
            if (a.l_out) a.l_out[stat_idx] = l_run * exp2f(m_ref - m_true);
            if (a.lse_out) a.lse_out[stat_idx] = (m_ref + log2f(l_run)) * kLn2;
        }
#pragma unroll
        for (int c = half * (D / 2); c < (half + 1) * (D / 2); c += 32) {
            uint32_t ov[32];
            tmem_ld32(tmem_addr(tmem, lane_base, Cfg::kColO + c), ov);
            tmem_wait_ld();
            if constexpr (OUT_F32) {
                if (in_range) {
                    float* dst = reinterpret_cast<float*>(a.out) + ((long long)bh * a.T + row_g) * D + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(dst + i) =
                            make_float4(__uint_as_float(ov[i]) * inv_l, __uint_as_float(ov[i + 1]) * inv_l,
                                        __uint_as_float(ov[i + 2]) * inv_l, __uint_as_float(ov[i + 3]) * inv_l);
                }
            } else {
                // stage BF16 rows in the (now idle) Q buffer, swizzled the way the TMA store expects
                uint8_t* atom = sQ + (c >> 6) * kAtomBytes;
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint4 w;
                    w.x = pack_bf16x2(__uint_as_float(ov[i]) * inv_l, __uint_as_float(ov[i + 1]) * inv_l);
                    w.y = pack_bf16x2(__uint_as_float(ov[i + 2]) * inv_l, __uint_as_float(ov[i + 3]) * inv_l);
                    w.z = pack_bf16x2(__uint_as_float(ov[i + 4]) * inv_l, __uint_as_float(ov[i + 5]) * inv_l);
                    w.w = pack_bf16x2(__uint_as_float(ov[i + 6]) * inv_l, __uint_as_float(ov[i + 7]) * inv_l);
                    if (RAGGED && valid < kBM) {  // the rows behind the sequence are not this tile's to write
                        if (in_range)
                            *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.out) + (long long)row_g * a.ragged.out_stride +
                                                      (long long)hh * D + c + i) = w;
                    } else {
                        *reinterpret_cast<uint4*>(atom + swz128(r, ((c & 63) + i) >> 3)) = w;
                    }
                }
            }
        }
        if (!OUT_F32 && !(RAGGED && valid < kBM)) {
            fence_proxy_async_smem();
            named_bar_sync(1, kSoftmaxThreads);
            if (tid == 0) {
                for (int at = 0; at < Cfg::kAtoms; ++at) tma_store_4d(&a.map_o, sQ + at * kAtomBytes, at * 64, row0 + qt * kBM, hh, bb);
                tma_store_commit();
                tma_store_wait_read();  // the staging tile must outlive the bulk read; the write completes with the grid
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kProducerWarp) tmem_dealloc(tmem, Cfg::kTmemCols);
}

template <int D, bool OUT_F32>
cudaError_t launch_fwd(const TcFwdArgs& a, cudaStream_t stream) {
    using Cfg = FwdCfg<D>;
    auto kern = attn_fwd_tc_kernel<D, OUT_F32, false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
    if (e != cudaSuccess) return e;
    const int n_q_tiles = (a.T + kBM - 1) / kBM;
    const long long blocks = (long long)n_q_tiles * a.BH;
    return launch_pdl(kern, dim3((unsigned int)blocks), dim3(kThreads), Cfg::kSmemBytes, stream, a);
}

template <int D>
cudaError_t launch_fwd_ragged(const TcFwdArgs& a, cudaStream_t stream) {
    using Cfg = FwdCfg<D>;
    auto kern = attn_fwd_tc_kernel<D, false, true>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes);
    if (e != cudaSuccess) return e;
    return launch_pdl(kern, dim3((unsigned int)(a.ragged.capacity * a.H)), dim3(kThreads), Cfg::kSmemBytes, stream, a);
}

}  // namespace

cudaError_t launch_attn_fwd_ragged(const TcFwdArgs& a, cudaStream_t stream) {
    // Where the card is not full the chain of a tile's steps is what counts, and this variant (eight softmax warps, scores made two
    // tiles ahead) has the shorter one; sequences of one or two tiles gain from two CTAs per SM again as soon as the tiles outnumber
    // the SMs clearly. Measured, two small CTAs / one large, d = 128: one sequence of 4000, 2 heads 58 / 37 us; two of 1538, 8 heads
    // (208 CTAs) 30 / 21 us; one of 1700, 20 heads (280) 34 / 27 us; twenty of 60-300, 6 heads (270) 12.3 / 14.5 us.
    const long long ctas = (long long)a.ragged.capacity * a.H;
    if (a.ragged.items == nullptr && (ctas <= 222 || a.T >= 256ll * a.ragged.n)) {
        if (a.d == 64) return launch_fwd_ragged<64>(a, stream);
        if (a.d == 128) return launch_fwd_ragged<128>(a, stream);
    }
    return launch_attn_fwd_ragged_short(a, stream);
}

cudaError_t launch_attn_fwd_tc(const TcFwdArgs& a, cudaStream_t stream) {
    if (a.BH == 0 || a.T == 0) return cudaSuccess;
    // Few key tiles per CTA: the two-CTAs-per-SM variant hides the per-CTA prologue and epilogue better.
    // Two small CTAs per SM (attn_tc_fwd_short.cu) against one large CTA with eight softmax warps (this file),
    // measured on a B200, forward TFLOP/s: d=64 T=1024 363 vs 248, T=4096 557 vs 462, T=8192 620 vs 524;
    // d=128 T=512 509 vs 352, T=2048 807 vs 716, T=4096 963 vs 930, T=8192 equal.
    if (a.d == 64 || a.T <= 4096) return launch_attn_fwd_tc_short(a, stream);
    if (a.d == 128) return a.out_is_f32 ? launch_fwd<128, true>(a, stream) : launch_fwd<128, false>(a, stream);
    return cudaErrorInvalidValue;
}

}  // namespace b200attn
