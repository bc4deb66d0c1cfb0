// srf_grouped_fp8.cu -- the grouped layer on 8-bit (e4m3) samples and weights, on tcgen05 / TMEM.
//
//   y[r][n] = act( sum_b sx[b][r] sw[g][n/128][b] * sum_{k in block b} x[r][k] W[g][n][k] ),   blocks of 128 inputs
//
// Inside a block the tensor core sums products of 8-bit values in fp32 (TMEM); the scales differ from block to block, so
// every block's sum is taken out of TMEM, scaled and added in fp32 registers.  A stage of the operand ring is one block
// (128 bytes of every row), its four instructions start a new accumulator, and two warpgroups -- each half of the tile's
// columns -- follow one block behind.  The rest is as in srf_grouped.cu.
//
// Measured (several B200): 32773 samples in 8 groups, 4096 -> 2048: 297-307 us a call (1.8 PFLOP/s), 270 us alone with the
// tensor pipe busy for 57 % of the time.  What bounds it is the accumulators' turn-over: a block's instructions take 512
// cycles, reading its sums out of TMEM 455, and the two hand-overs between the issuing thread and the 16 scaling warps of a
// pair some 700, shared by the two accumulators that TMEM holds: 835 cycles a block.  The scales themselves cost 2 %.  Narrower
// tiles with more accumulators or more warps were slower (192 columns and three sets of warps 333 us, 128 columns and four
// accumulators 370), as were single CTAs (330 us alone).  Few samples: 131 samples in 32 groups of 2048 x 2048, 135 MB, 31-33
// us (floor 20.6): whole tiles only, 1.73 an SM round up to 2, which makes 23.8 of them; the rest is start-up and the hand-over
// of every block.
#include <cstring>
#include "srf_layers.cuh"
#include "srf_tile.cuh"

namespace srf {

using namespace tile;

namespace {

constexpr int kThreads = 384;                 // TMA, MMA, TMEM owner, spare, 8 scaling warps
constexpr int kBM = 128, kBK = 128;
constexpr uint32_t kTmemCols = 512;
constexpr int kABytes = kBM * kBK;
constexpr int kStoreBytes = 8 * 4096;         // staging of the scaling warps
constexpr int kScaleAhead = 4;                // blocks whose scales are on their way
constexpr int kScaleBytes = 8 * kScaleAhead * 128;
constexpr int kSmemMin = 120 * 1024;          // a second CTA that allocates TMEM must never share the SM

struct Fp8Args {
    const uint64_t* offsets;
    unsigned char* out;
    const float* x_scales;        // [blocks of n_in][n_rows]
    const float* w_scales;        // [group][blocks of n_out][blocks of n_in]
    uint64_t out_row_bytes;
    uint32_t n_rows, n_groups, n_in, n_out;
    int bf16, f32, relu;
    unsigned int* error_flags;
};

// CG CTAs share a tile of CG*128 x BN outputs; each holds 128 rows of A and BN/CG rows of B per stage.
template <int BN, int CG> __host__ __device__ constexpr int n_stages() { return BN / CG == 256 ? 3 : BN / CG == 128 ? 5 : 7; }
template <int BN> __host__ __device__ constexpr int n_accs() { return BN == 256 ? 2 : 4; }
template <int BN, int CG> __host__ __device__ constexpr int smem_bytes() {
    const int b = 1024 + n_stages<BN, CG>() * (kABytes + BN / CG * kBK) + kStoreBytes + kScaleBytes + 512;
    return b < kSmemMin ? kSmemMin : b;
}

// Copies of one lane's own values into shared memory, in groups that complete in order.  Copies of 4 bytes exist through L1 only;
// they are ordinary loads for memory order, so the wait for the kernel in front (a quantisation that writes the scales)
// orders them.
__device__ __forceinline__ void copy_async4(float* dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

// Two scales whose product is no normal number, as two factors of about the same exponent with the same product: a block's
// sum (0 or 2^-18 .. 2^25) times one and then the other leaves the range only where the result does.  Powers of two are moved
// between them, so neither is rounded.  A scale of 0, infinity or NaN has the product it has.
__device__ __forceinline__ void balance_scales(float sx, float sw, float* before, float* scale) {
    const float ax = fabsf(sx), aw = fabsf(sw), inf = __int_as_float(0x7f800000);
    if (ax > 0.f && ax < inf && aw > 0.f && aw < inf) {
        const int k = (ilogbf(sw) - ilogbf(sx)) / 2;
        *before = ldexpf(sx, k);
        *scale = ldexpf(sw, -k);
    }
}
// Neither subnormal (its bits would be lost), nor 0 or infinite (which it may have become), nor NaN.
__device__ __forceinline__ bool normal(float v) { return fabsf(v) >= 1.17549435e-38f && fabsf(v) <= 3.40282347e38f; }

template <int BN, int CG>
__global__ void __launch_bounds__(kThreads, 1)
k_grouped_fp8(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Fp8Args p) {
    constexpr int kStages = n_stages<BN, CG>(), kAccs = n_accs<BN>();
    constexpr int kBRows = BN / CG, kBBytes = kBRows * kBK;
    constexpr int kCols = BN / 2;                 // columns of one set of scaling warps
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char* sm_a = smem;
    unsigned char* sm_b = smem + kStages * kABytes;
    unsigned char* sm_store = sm_b + kStages * kBBytes;
    float* sm_scale = reinterpret_cast<float*>(sm_store + kStoreBytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm_store + kStoreBytes + kScaleBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 2 * kAccs);
    volatile uint32_t* failed = tmem_slot + 1;
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * kStages;
    const uint32_t bar_acc_full = bar_empty + 8 * kStages, bar_acc_empty = bar_acc_full + 8 * kAccs;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const uint32_t tiles_n = (p.n_out + BN - 1) / BN;
    const uint32_t blocks_k = (p.n_in + kBK - 1) / kBK, blocks_n = (p.n_out + 127) / 128;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) { mbar_init(bar_full + 8 * i, CG); mbar_init(bar_empty + 8 * i, 1); }
        for (int i = 0; i < kAccs; ++i) { mbar_init(bar_acc_full + 8 * i, 1); mbar_init(bar_acc_empty + 8 * i, 8 * CG); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *failed = 0;
        tma_prefetch_map(&map_a);
        tma_prefetch_map(&map_b);
    }
    if (warp == 2) tmem_alloc<CG>(smem_u32(tmem_slot), kTmemCols);
    tc_fence_before();
    if (CG == 2) cluster_sync(); else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_for_inputs();
    let_next_start();

    bool bad = false, ok = true;
    GroupWalk walk;
    uint32_t at = blockIdx.x / CG, group = 0, tn = 0, m = 0;
    Span span = {0, 0};
    auto next_tile = [&]() -> bool {
        constexpr uint32_t kHeight = CG * kBM;
        uint32_t local;
        if (!walk.find(at, p.offsets, p.n_groups, p.n_rows,
                       [&](const Span& s) { return (s.end - s.begin + kHeight - 1) / kHeight * tiles_n; }, &group, &span, &local, &bad))
            return false;
        tile_place(local, (span.end - span.begin + kHeight - 1) / kHeight, tiles_n, &m, &tn);
        m = span.begin + m * kHeight + rank * kBM;
        at += gridDim.x / CG;
        return true;
    };

    if (warp < 4) {
        if (BN == 256) regs_for_issue();
        if (warp == 0) {
            // ---- operand loads: one thread ----
            const uint32_t lead_full = CG == 2 ? leader_addr(bar_full) : bar_full;
            const uint32_t a0 = smem_u32(sm_a), b0 = smem_u32(sm_b);
            Ring<kStages> at_stage;
            uint32_t issued = 0;
            while (ok && next_tile()) {
                // single CTAs load only the rows that the group has (what lies in the others' place is never stored)
                const uint32_t boxes = CG == 2 || span.end - m >= (uint32_t)kBM ? kBM / kRowBox : (span.end - m + kRowBox - 1) / kRowBox;
                const uint32_t bytes = boxes * (kRowBox * kBK) + kBBytes;
                if (elect_one()) {
                    Ring<kStages> r = at_stage;
                    for (uint32_t k = 0; k < blocks_k; ++k) {
                        if (r.round > 0 && !mbar_wait_one(bar_empty + 8 * r.slot, (r.round - 1) & 1, failed)) { ok = false; break; }
                        const uint32_t bar = lead_full + 8 * r.slot;
                        pair_expect<CG>(bar, bytes);
                        if (CG == 2) tma_2d<CG>(a0 + r.slot * kABytes, &map_a, bar, (int)(k * kBK), (int)m);
                        else
                            for (uint32_t i = 0; i < boxes; ++i)
                                tma_2d<CG>(a0 + r.slot * kABytes + i * (kRowBox * kBK), &map_a, bar, (int)(k * kBK), (int)(m + i * kRowBox));
                        tma_3d<CG>(b0 + r.slot * kBBytes, &map_b, bar, (int)(k * kBK), (int)(tn * BN + rank * kBRows), (int)group);
                        ++issued;
                        r.step();
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                at_stage.skip(blocks_k);
            }
            // Copies may still be on their way when another warp gave up: they must land before the CTA (or pair) leaves.
            if ((!ok || *failed) && rank == 0) drain_ring<kStages>(bar_full, issued);
        } else if (warp == 1 && rank == 0) {
            // ---- matrix instructions: one thread; four to a block, each block its own accumulator ----
            constexpr uint32_t idesc = idesc_shape(CG * kBM, BN);      // e4m3 is format 0
            const uint64_t desc_a = operand_desc(smem_u32(sm_a), 16, 1024), desc_b = operand_desc(smem_u32(sm_b), 16, 1024);
            Ring<kStages> at_stage;
            Ring<kAccs> at_acc;
            while (ok && next_tile()) {
                if (elect_one()) {
                    Ring<kStages> r = at_stage;
                    Ring<kAccs> acc = at_acc;
                    for (uint32_t k = 0; k < blocks_k; ++k) {
                        if (acc.round > 0 && !mbar_wait_one(bar_acc_empty + 8 * acc.slot, (acc.round - 1) & 1, failed)) { ok = false; break; }
                        if (!mbar_wait_one(bar_full + 8 * r.slot, r.round & 1, failed)) { ok = false; break; }
                        tc_fence_after();
                        const uint64_t da = desc_at(desc_a, r.slot * kABytes), db = desc_at(desc_b, r.slot * kBBytes);
                        const uint32_t d = tmem + acc.slot * BN;
#pragma unroll
                        for (uint32_t q = 0; q < 4; ++q) mma_f8<CG>(d, desc_at(da, q * 32), desc_at(db, q * 32), idesc, q != 0);
                        mma_commit<CG>(bar_acc_full + 8 * acc.slot);
                        mma_commit<CG>(bar_empty + 8 * r.slot);
                        r.step();
                        acc.step();
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                at_stage.skip(blocks_k);
                at_acc.skip(blocks_k);
            }
        }
    } else {
        // ---- scale, sum, store ----
        if (BN == 256) regs_for_sums();
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        unsigned char* stage = sm_store + (warp - 4) * 4096;
        const uint32_t lead_acc_empty = CG == 2 ? leader_addr(bar_acc_empty) : bar_acc_empty;
        uint32_t acc = 0, acc_round = 0;
        while (ok && next_tile()) {
            const uint32_t row0 = m + quarter * 32;
            const uint32_t row = row0 + lane < span.end ? row0 + lane : span.end - 1;      // behind the group: the scales of its last sample
            const uint32_t col0 = tn * BN + half * kCols;
            const uint32_t wb = col0 / 128 < blocks_n ? col0 / 128 : blocks_n - 1;
            const float* sx = p.x_scales + row;
            const float* sw = p.w_scales + ((size_t)group * blocks_n + wb) * blocks_k;
            uint64_t sum[kCols / 2];
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) sum[i] = 0ull;
            // The sample's scales come through a ring in shared memory, every lane its own, four blocks ahead, and the matrix's one
            // per lane, 32 blocks at a time.  (Loaded into registers one block ahead, 250 of 920 cycles a block went into
            // waiting for L2; further ahead, the registers spilled.)
            float* ring = sm_scale + (warp - 4) * (kScaleAhead * 32) + lane;
            const float* sx_ahead = sx;
#pragma unroll
            for (uint32_t u = 0; u < kScaleAhead; ++u) {
                if (u < blocks_k) copy_async4(ring + u * 32, sx_ahead);
                copy_async_group();
                sx_ahead += p.n_rows;
            }
            float sw_lane = 0.f;
            for (uint32_t k = 0; k < blocks_k; ++k) {
                if ((k & 31) == 0) sw_lane = k + lane < blocks_k ? __ldcg(sw + k + lane) : 0.f;
                copy_async_wait<kScaleAhead - 1>();
                float* slot = ring + (k % kScaleAhead) * 32;
                const float scale_x = *slot, scale_w = __shfl_sync(0xffffffffu, sw_lane, k & 31);
                float scale = scale_x * scale_w;
                if (k + kScaleAhead < blocks_k) copy_async4(slot, sx_ahead);
                copy_async_group();
                sx_ahead += p.n_rows;
                if (!mbar_wait(bar_acc_full + 8 * acc, acc_round & 1, failed)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d = tmem + acc * BN + half * kCols + ((uint32_t)(quarter * 32) << 16);
                // a piece of 32 columns is on its way while the one before it is scaled and added
                uint32_t r[2][32];
                tmem_ld32(d, r[0]);
                // Where a sample of the warp needs a second factor, the block's sums take it in TMEM (1 for the other samples), so that
                // the way below stays as it is (32773 samples, 4096 -> 2048: 298 us with this test, 296 without; the factor as a branch
                // in the loop below 331, a second loop beside it 387).
                if (__any_sync(0xffffffffu, !normal(scale))) {
                    float before = 1.f;
                    if (!normal(scale)) balance_scales(scale_x, scale_w, &before, &scale);
                    tmem_ld_wait(r[0]);
#pragma unroll 1
                    for (int c = 0; c < kCols; c += 32) {
                        tmem_ld32(d + c, r[0]);
                        tmem_ld_wait(r[0]);
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[0][i] = __float_as_uint(__uint_as_float(r[0][i]) * before);
                        tmem_st32(d + c, r[0]);
                    }
                    tmem_st_wait();
                    tmem_ld32(d, r[0]);
                }
                const uint64_t scale2 = pair_of(__float_as_uint(scale), __float_as_uint(scale));
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) {
                    tmem_ld_wait(r[c & 1]);
                    if (c + 1 < kCols / 32) {
                        tmem_ld32(d + 32 * (c + 1), r[(c + 1) & 1]);
                    } else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) pair_arrive_read<CG>(lead_acc_empty + 8 * acc);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) fma2(sum[16 * c + i], pair_of(r[c & 1][2 * i], r[c & 1][2 * i + 1]), scale2);
                }
                if (++acc == kAccs) { acc = 0; ++acc_round; }
            }
            if (!ok) break;
            RowStore rs;
            rs.bf16 = p.bf16 != 0;
            rs.f32 = p.f32 != 0;
            rs.gate = nullptr;
            rs.gate_row_bytes = 0;
            rs.row_bytes = p.out_row_bytes;
            rs.rows = row0 >= span.end ? 0u : span.end - row0 < 32 ? span.end - row0 : 32u;
            unsigned char* out = p.out + row0 * p.out_row_bytes;
            if (p.relu) {
#pragma unroll
                for (int i = 0; i < kCols / 2; ++i) sum[i] = pair_of(__float_as_uint(relu(lo_of(sum[i]))), __float_as_uint(relu(hi_of(sum[i]))));
            }
            const uint32_t cols = col0 >= p.n_out ? 0u : p.n_out - col0 < (uint32_t)kCols ? p.n_out - col0 : (uint32_t)kCols;
            if (p.f32) {
#pragma unroll
                for (int c = 0; c < kCols; c += 32) {
                    if ((uint32_t)c >= cols) continue;
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        const uint64_t v0 = sum[c / 2 + 2 * u], v1 = sum[c / 2 + 2 * u + 1];
                        stage_unit(stage, lane, u, make_uint4((uint32_t)v0, (uint32_t)(v0 >> 32), (uint32_t)v1, (uint32_t)(v1 >> 32)));
                    }
                    rs.bytes = (cols - c < 32u ? cols - c : 32u) * 4u;
                    rs.out = out + (size_t)(col0 + c) * 4;
                    store_rows(rs, stage);
                }
            } else {
                constexpr int kPer = kCols < 64 ? kCols : 64;
#pragma unroll
                for (int c = 0; c < kCols; c += kPer) {
                    if ((uint32_t)c >= cols) continue;
#pragma unroll
                    for (int u = 0; u < kPer / 8; ++u) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = pack16(lo_of(sum[c / 2 + 4 * u + e]), hi_of(sum[c / 2 + 4 * u + e]), rs.bf16);
                        stage_unit(stage, lane, u, make_uint4(w[0], w[1], w[2], w[3]));
                    }
                    rs.bytes = (cols - c < (uint32_t)kPer ? cols - c : (uint32_t)kPer) * 2u;
                    rs.out = out + (size_t)(col0 + c) * 2;
                    store_rows(rs, stage);
                }
            }
        }
    }
    if ((bad || (!ok && lane == 0)) && p.error_flags) atomicOr(p.error_flags, (ok ? 0u : 2u) | (bad ? 16u : 0u));
    tc_fence_before();
    if (CG == 2) cluster_sync(); else __syncthreads();      // a pair's barriers and accumulators serve both CTAs to the end
    if (warp == 2) tmem_free<CG>(tmem, kTmemCols);
}

}  // namespace

const char* launch_grouped_matmul_fp8(const srf_grouped_t& p, const uint64_t* offsets, const void* x, const float* x_scales,
                                      const void* w, const float* w_scales, void* y, unsigned int* error_flags,
                                      cudaStream_t stream) {
    if (!p.n_rows) return nullptr;
    const int sms = sm_count();
    const TileShape t = pick_tile(p, p.n_out, sms, 64, 256);
    CUtensorMap a, b;
    if (!make_operand_map(&a, x, SRF_TYPE_E4M3, p.n_in, p.n_rows, p.ld_x, 0, 0, t.cg == 2 ? kBM : kRowBox) ||
        !make_operand_map(&b, w, SRF_TYPE_E4M3, p.n_in, p.n_out, p.ld_w, p.n_groups, p.group_stride, t.bn / t.cg))
        return "the driver refused an operand's tensor map";
    Fp8Args k;
    memset(&k, 0, sizeof(k));
    k.offsets = offsets; k.out = (unsigned char*)y; k.x_scales = x_scales; k.w_scales = w_scales; k.n_rows = (uint32_t)p.n_rows;
    k.n_groups = p.n_groups; k.n_in = p.n_in; k.n_out = p.n_out;
    k.f32 = p.out_type == SRF_TYPE_F32; k.bf16 = p.out_type == SRF_TYPE_BF16; k.relu = p.activation == SRF_ACT_RELU;
    k.out_row_bytes = p.ld_y * (k.f32 ? 4 : 2); k.error_flags = error_flags;
    const uint32_t grid = tile_grid(p, p.n_out, t, sms);
    if (t.cg == 2) return launch_layer(k_grouped_fp8<256, 2>, smem_bytes<256, 2>(), kThreads, 2, dim3(grid), stream, a, b, k);
    switch (t.bn) {
    case 256: return launch_layer(k_grouped_fp8<256, 1>, smem_bytes<256, 1>(), kThreads, 1, dim3(grid), stream, a, b, k);
    case 128: return launch_layer(k_grouped_fp8<128, 1>, smem_bytes<128, 1>(), kThreads, 1, dim3(grid), stream, a, b, k);
    default: return launch_layer(k_grouped_fp8<64, 1>, smem_bytes<64, 1>(), kThreads, 1, dim3(grid), stream, a, b, k);
    }
}

}  // namespace srf
