// srf_grouped.cu -- matrix products grouped by ragged sample lists, 16-bit values, on tcgen05 / TMEM.
//
// The samples of a frame or batch are sorted by region; group g owns samples offsets[g] .. offsets[g+1] and a matrix
// W[g] (n_out x n_in, row-major like the network's own layers).  Three products, all D = A B^T summed over k:
//
//   layer        y[r][n]  = act(sum_k x[r][k]  W[g][n][k])    A = samples, k = inputs    B = W[g]
//   input grad   dx[r][k] = sum_n dy[r][n] W[g][n][k]         A = samples, k = outputs   B = W[g], read down its columns
//   weight grad  dW[g][n][k] = sum_r dy[r][n] x[r][k]         A, B = both sample arrays, read down their columns
//
// One persistent CTA per SM: a TMA warp fills a ring of 64-deep operand stages, one thread issues tcgen05.mma
// (128 x BN outputs a CTA, fp32 accumulators in TMEM, two to four of them), two sets of four warps take finished
// accumulators to memory, every other tile each, while the next ones fill.  Operands that are read down their columns
// stay as they lie in memory: the tensor core takes them MN-major.  Tiles are dealt round-robin; every warp finds its
// tiles itself from the offsets (GroupWalk), so no launch, workspace or host read prepares them.
//
// Large layers run on pairs of CTAs (CG = 2): one instruction computes 256 x 256 outputs on two SMs, each of which
// loads its own 128 rows of A and half of B, so that an operand byte from L2 serves twice as many products.  Their tiles
// are 160 to 256 columns wide, in steps of 32, so that the columns divide evenly: 656 columns are three tiles of 224 (66
// groups of 1057 samples, 780 -> 656: 84.7 us against 88.7).
//
// The tensor core's additions to an accumulator truncate, so that a long sum's error grows with its length: 2-norm 2.5e-6 at 2048
// products of mixed signs, 9.7e-6 at 8192, 7.7e-5 at 65536; sums of one sign fall short by 1.3e-5, 5.3e-5 and 4.3e-4 of themselves.
// That is little beside a rounding to bf16, or to fp16 up to 8192 products, but not what a result in fp32 should have.  LONG
// kernels therefore start a new accumulator every 512 products (6.4e-7; 2.8e-6 for one sign) and add those in registers, rounded;
// both sets of epilogue warps work on every tile then, half of its columns each.  The rounded additions of m such runs, one by one,
// have an error of their own that grows with sqrt(m): weight gradients have 4.8e-7 at 2^14 samples, 5.8e-7 at 2^18, 8.4e-7 at 2^20
// where one worker owns a whole sum (shorter where the sum is cut), and some 4e-6 at 2^24.
//
// Measured (several B200): 32801 samples in 16 groups, 2048 -> 2043: 178 us alone (1.54 PFLOP/s, tensor pipe 93 %), 214-224 us a
// call under the power limit (single CTAs 241), with results in fp32 238-243; 160 samples in 64 groups, 2048 -> 1408: 63-68 us,
// 5.4-5.9 TB/s of matrices; 1048613 samples 32 -> 64: 41-43 us, bound by the pace of the epilogue's chain (one tile of 128 x 64
// every 1500 cycles an SM; DRAM moves 21 us' worth); weight gradient of 16389 x 2048 x 2048: 126 us alone and 27-33 for its
// joins.
//
// A tile's rows behind its group's end hold the next group's samples: harmless in the first two products (an output row
// depends on its own sample alone and those rows are not stored).  In the weight gradient they would be summed, so the
// rows of the last stage of a group are zeroed in shared memory, in both operands (a NaN of the next group must not
// meet a zero).
#include <cstring>
#include "srf_layers.cuh"
#include "srf_tile.cuh"

namespace srf {

using namespace tile;

namespace {

enum Mode { kLayer = 0, kInputGrad = 1, kWeightGrad = 2 };

constexpr int kThreads = 384;                 // TMA, MMA, TMEM owner, spare, two sets of 4 epilogue warps (four sets: 2 % slower
                                              // for 1048613 samples 32 -> 64, narrow gradients 6 %)
constexpr int kBM = 128, kBK = 64;
constexpr uint32_t kChunk = 8;                // stages to an accumulator in LONG kernels
constexpr uint32_t kTmemCols = 512;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kStoreBytes = 8 * 4096;         // staging of the epilogue warps
constexpr int kSmemMin = 120 * 1024;          // a second CTA that allocates TMEM must never share the SM

struct GroupedArgs {
    const uint64_t* offsets;
    unsigned char* out;
    const unsigned char* gate;
    float* partial;               // weight gradient: two tiles of partial sums per worker
    uint64_t out_row_bytes, out_group_bytes, gate_row_bytes;
    uint32_t n_rows, n_groups;
    uint32_t out_rows;            // weight gradient: n_out
    uint32_t out_cols;            // n_out, n_in, n_in
    uint32_t depth;               // summed length of the first two products
    uint32_t width;               // columns of a pair's tile
    uint32_t n_workers;           // weight gradient: even shares of the work
    int bf16, f32, relu;
    unsigned int* error_flags;
};

// CG CTAs share a tile of CG*128 x BN outputs; each holds 128 rows of A and BN/CG rows of B per stage.
template <int BN, int CG> __host__ __device__ constexpr int n_stages() { return BN / CG == 256 ? 4 : BN / CG == 128 ? 6 : 8; }
template <int BN> __host__ __device__ constexpr int n_accs() { return BN == 256 ? 2 : 4; }
template <int BN, int CG> __host__ __device__ constexpr int smem_bytes() {
    const int b = 1024 + n_stages<BN, CG>() * (kABytes + BN / CG * kBK * 2) + kStoreBytes + 512;
    return b < kSmemMin ? kSmemMin : b;
}

// Units of work of a group: whole output tiles for the first two products; for the weight gradient, whose work is cut evenly
// across the CTAs (see below), the 64-sample stages of an output tile and kTileUnits in front of them, for what a tile costs
// beside its stages: counted without, groups of few samples -- many shallow tiles -- held their CTAs up (both gradients of
// 16389 x 2048 x 2048 in groups of 200 to 5000 samples: 324 us, with 4 units 307, 8 304, 14 302).  Weight gradients alone, ragged
// groups, units 0 / 4 / 8 / 14: 262144 x 64 x 64 in 1024 groups 80 / 74 / 74 / 74 us (in 16: 31 each), 65536 x 256 x 512 in 64
// groups 68 / 62 / 61 / 59, 16389 x 1024 x 1024 in 100 groups 252 / 201 / 186 / 179.
constexpr uint32_t kTileUnits = 14;
template <int MODE, int CG>
__device__ __forceinline__ uint32_t group_units(const Span& s, uint32_t tiles_across) {
    const uint32_t rows = s.end - s.begin;
    return (MODE == kWeightGrad ? (rows ? (rows + kBK - 1) / kBK + kTileUnits : 0u) : (rows + CG * kBM - 1) / (CG * kBM)) * tiles_across;
}

// One stretch of summed stages of one output tile.
struct Piece {
    uint32_t group;
    Span span;
    uint32_t m;            // first output row: sample (first two products) or row of W (weight gradient)
    uint32_t n;            // output column tile
    uint32_t k0;           // first stage
    uint32_t k_stages;     // stages
    bool whole;            // the piece is the tile's whole sum
    bool first;            // the piece holds the tile's first stage
    uint32_t worker;
};

// The pieces of this CTA (or pair), one after the other; every warp walks them for itself.
//
// Weight gradient: the stages of all tiles are one line of `units` that n_workers share out evenly, so ragged groups
// balance by themselves and a narrow layer (one tile per group) still fills every SM.  CTA c works for the workers c,
// c + CTAs, ...: with more workers than CTAs, all CTAs are in the same part of the line at a time and find that part's
// samples in L2.  A tile that a boundary cuts is summed from the workers' partial sums, in the workers' order, by a second
// kernel: the same result on every run.
__device__ __forceinline__ uint32_t first_unit(uint32_t units, uint32_t worker, uint32_t n_workers) {
    const uint32_t q = units / n_workers, r = units - q * n_workers;
    return worker * q + (worker < r ? worker : r);
}

template <int MODE, int CG>
struct Pieces {
    GroupWalk walk;
    uint32_t at, stop, step, units, worker;
    // first two products: pieces start, start + every, ... of those dealt to this CTA
    __device__ __forceinline__ void init(const GroupedArgs& p, uint32_t n_units, uint32_t start, uint32_t every) {
        const uint32_t self = blockIdx.x / CG, all = gridDim.x / CG;
        if (MODE == kWeightGrad) {
            units = n_units;
            worker = self;
            at = first_unit(units, worker, p.n_workers);
            stop = first_unit(units, worker + 1, p.n_workers);
        } else {
            at = self + start * all;
            step = every * all;
        }
    }
    __device__ __forceinline__ bool next(const GroupedArgs& p, uint32_t tiles_m, uint32_t tiles_n, Piece* o, bool* bad) {
        const uint32_t across = MODE == kWeightGrad ? tiles_m * tiles_n : tiles_n;
        for (;;) {
            if (MODE == kWeightGrad) {
                while (at >= stop) {
                    worker += gridDim.x / CG;
                    if (worker >= p.n_workers) return false;
                    at = first_unit(units, worker, p.n_workers);
                    stop = first_unit(units, worker + 1, p.n_workers);
                }
            }
            uint32_t local;
            if (!walk.find(at, p.offsets, p.n_groups, p.n_rows, [&](const Span& s) { return group_units<MODE, CG>(s, across); },
                           &o->group, &o->span, &local, bad))
                return false;
            const uint32_t rows = o->span.end - o->span.begin;
            uint32_t m;
            if (MODE == kWeightGrad) {
                const uint32_t deep = (rows + kBK - 1) / kBK, cost = deep + kTileUnits;
                const uint32_t t = local / cost, v = local - t * cost;
                const uint32_t end = cost - v < stop - at ? cost : v + (stop - at);        // units of the tile up to which this worker goes
                at += end - v;
                if (end <= kTileUnits) continue;                                          // none of its stages
                tile_place(t, tiles_m, tiles_n, &m, &o->n);
                o->m = m * (CG * kBM);
                o->k0 = v > kTileUnits ? v - kTileUnits : 0;
                o->k_stages = end - kTileUnits - o->k0;
                o->first = o->k0 == 0;
                o->whole = o->k_stages == deep;
                o->worker = worker;
            } else {
                tile_place(local, (rows + CG * kBM - 1) / (CG * kBM), tiles_n, &m, &o->n);
                o->m = o->span.begin + m * (CG * kBM);
                o->k0 = 0;
                o->k_stages = (p.depth + kBK - 1) / kBK;
                o->first = o->whole = true;
                at += step;
            }
            return true;
        }
    }
};

// Units of all groups (warp-collective).
template <int MODE, int CG>
__device__ __forceinline__ uint32_t all_units(const GroupedArgs& p, uint32_t across, bool* bad) {
    uint32_t sum = 0;
    for (uint32_t g = threadIdx.x & 31; g < p.n_groups; g += 32) sum += group_units<MODE, CG>(group_span(p.offsets, g, p.n_rows, bad), across);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
}

// Zeroes rows [r0, r1) of the blocks of 64 columns of an operand stage (128 bytes a row).
__device__ __forceinline__ void zero_rows(unsigned char* stage, int blocks, int r0, int r1) {
    const int units = (r1 - r0) * 8;
    for (int i = threadIdx.x & 31; i < units * blocks; i += 32) {
        const int blk = i / units, u = i - blk * units;
        *reinterpret_cast<uint4*>(stage + blk * 8192 + r0 * 128 + u * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
}

template <int MODE, int BN, int CG, bool LONG>
__global__ void __launch_bounds__(kThreads, 1)
k_grouped(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GroupedArgs p) {
    constexpr int kStages = n_stages<BN, CG>(), kAccs = n_accs<BN>();
    constexpr int kBRows = BN / CG, kBBytes = kBRows * kBK * 2;
    constexpr bool kAColumns = MODE == kWeightGrad, kBColumns = MODE != kLayer;     // read down the columns: MN-major
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char* sm_a = smem;
    unsigned char* sm_b = smem + kStages * kABytes;
    unsigned char* sm_store = sm_b + kStages * kBBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm_store + kStoreBytes);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 2 * kAccs + 1);
    volatile uint32_t* failed = tmem_slot + 1;
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * kStages;
    const uint32_t bar_acc_full = bar_empty + 8 * kStages, bar_acc_empty = bar_acc_full + 8 * kAccs;
    const uint32_t bar_tail = bar_acc_empty + 8 * kAccs;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const uint32_t width = CG == 2 ? p.width : BN;                 // columns of a tile
    const uint32_t tiles_n = (p.out_cols + width - 1) / width;
    const uint32_t tiles_m = MODE == kWeightGrad ? (p.out_rows + CG * kBM - 1) / (CG * kBM) : 0;

    // Barriers of a pair: `full` and `acc_empty` are those of rank 0, where the instructions are issued; `empty` and
    // `acc_full` are signalled in both CTAs.
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) { mbar_init(bar_full + 8 * i, CG); mbar_init(bar_empty + 8 * i, 1); }
        for (int i = 0; i < kAccs; ++i) { mbar_init(bar_acc_full + 8 * i, 1); mbar_init(bar_acc_empty + 8 * i, (LONG ? 8 : 4) * CG); }
        mbar_init(bar_tail, 1);
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
    Pieces<MODE, CG> pieces;
    const bool storing = !LONG && warp >= 4;       // the two sets of epilogue warps take every other piece
    pieces.init(p, MODE == kWeightGrad ? all_units<MODE, CG>(p, tiles_m * tiles_n, &bad) : 0, storing ? (warp - 4) >> 2 : 0, storing ? 2 : 1);
    Piece t;

    if (warp < 4) {
        if (LONG && BN == 256) regs_for_issue();
        if (warp == 0) {
            // ---- operand loads: one thread, but for the zeroing of a group's last stage ----
            const uint32_t lead_full = CG == 2 ? leader_addr(bar_full) : bar_full;
            const uint32_t a0 = smem_u32(sm_a), b0 = smem_u32(sm_b);
            Ring<kStages> at;
            uint32_t issued = 0, tails = 0;
            while (ok && pieces.next(p, tiles_m, tiles_n, &t, &bad)) {
                const int am = (int)(t.m + rank * kBM), bn = (int)(t.n * width + rank * (width / CG));
                // weight gradient: the group's last stage, if it is of this piece and not a full one
                const uint32_t deep = t.span.end - t.span.begin;
                const bool tail = MODE == kWeightGrad && (t.k0 + t.k_stages) * kBK > deep;
                // single CTAs load only the rows that the group has (what lies in the others' place is never stored)
                const uint32_t boxes = MODE == kWeightGrad || CG == 2 || t.span.end - t.m >= (uint32_t)kBM ? kBM / kRowBox : (t.span.end - t.m + kRowBox - 1) / kRowBox;
                const uint32_t bytes = boxes * (kABytes / (kBM / kRowBox)) + (MODE == kLayer ? width / CG * (kBK * 2) : kBBytes);
                if (elect_one()) {
                    Ring<kStages> r = at;
                    for (uint32_t k = 0; k < t.k_stages; ++k) {
                        if (r.round > 0 && !mbar_wait_one(bar_empty + 8 * r.slot, (r.round - 1) & 1, failed)) { ok = false; break; }
                        const bool last = tail && k + 1 == t.k_stages;
                        const uint32_t a = a0 + r.slot * kABytes, b = b0 + r.slot * kBBytes, bar = last ? bar_tail : lead_full + 8 * r.slot;
                        if (last) mbar_expect(bar_tail, bytes);
                        else pair_expect<CG>(bar, bytes);
                        const int kk = (int)((t.k0 + k) * kBK);
                        if (kAColumns) {
#pragma unroll
                            for (int i = 0; i < kBM / 64; ++i) tma_2d<CG>(a + i * 8192, &map_a, bar, am + 64 * i, (int)t.span.begin + kk);
                        } else if (CG == 2) {
                            tma_2d<CG>(a, &map_a, bar, kk, am);
                        } else {
                            for (uint32_t i = 0; i < boxes; ++i) tma_2d<CG>(a + i * (kRowBox * 128), &map_a, bar, kk, am + (int)(i * kRowBox));
                        }
                        if (MODE == kLayer) {
                            tma_3d<CG>(b, &map_b, bar, kk, bn, (int)t.group);
                        } else if (MODE == kInputGrad) {
#pragma unroll
                            for (int i = 0; i < kBRows / 64; ++i) tma_3d<CG>(b + i * 8192, &map_b, bar, bn + 64 * i, kk, (int)t.group);
                        } else {
#pragma unroll
                            for (int i = 0; i < kBRows / 64; ++i) tma_2d<CG>(b + i * 8192, &map_b, bar, bn + 64 * i, (int)t.span.begin + kk);
                        }
                        ++issued;
                        r.step();
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                at.skip(t.k_stages);
                if (tail) {
                    // When the last stage has landed, zero the next group's samples up to the next 16 (an instruction's
                    // depth), then report the stage.
                    const uint32_t q = at.slot ? at.slot - 1 : kStages - 1;
                    ok = mbar_wait(bar_tail, tails++ & 1, failed);
                    const int r0 = (int)(deep - (t.k0 + t.k_stages - 1) * kBK), r1 = (r0 + 15) & ~15;
                    zero_rows(sm_a + q * kABytes, kBM / 64, r0, r1);
                    zero_rows(sm_b + q * kBBytes, kBRows / 64, r0, r1);
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0 && ok) pair_arrive<CG>(lead_full + 8 * q);
                    __syncwarp();
                }
            }
            // Copies may still be on their way when another warp gave up: they must land before the CTA (or pair) leaves.
            if ((!ok || *failed) && rank == 0) drain_ring<kStages>(bar_full, issued);
        } else if (warp == 1 && rank == 0) {
            // ---- matrix instructions: one thread ----
            const uint32_t idesc = idesc_shape(CG * kBM, width) | (p.bf16 ? (1u << 7) | (1u << 10) : 0u) | (kAColumns ? 1u << 15 : 0u) | (kBColumns ? 1u << 16 : 0u);
            const uint64_t desc_a = operand_desc(smem_u32(sm_a), kAColumns ? 8192 : 16, 1024), desc_b = operand_desc(smem_u32(sm_b), kBColumns ? 8192 : 16, 1024);
            constexpr uint32_t kStepA = kAColumns ? 2048 : 32, kStepB = kBColumns ? 2048 : 32;      // bytes of 16 summed indices
            Ring<kStages> at;
            Ring<kAccs> acc;
            while (ok && pieces.next(p, tiles_m, tiles_n, &t, &bad)) {
                if (elect_one()) {
                    Ring<kStages> r = at;
                    Ring<kAccs> to = acc;
                    const uint32_t deep = t.span.end - t.span.begin;
                    for (uint32_t k0 = 0; ok && k0 < t.k_stages; k0 += LONG ? kChunk : t.k_stages) {
                        // one accumulator
                        const uint32_t k1 = LONG && t.k_stages - k0 > kChunk ? k0 + kChunk : t.k_stages;
                        if (to.round > 0 && !mbar_wait_one(bar_acc_empty + 8 * to.slot, (to.round - 1) & 1, failed)) { ok = false; break; }
                        const uint32_t d = tmem + to.slot * BN;
                        for (uint32_t k = k0; k < k1; ++k) {
                            if (!mbar_wait_one(bar_full + 8 * r.slot, r.round & 1, failed)) { ok = false; break; }
                            tc_fence_after();
                            const uint64_t da = desc_at(desc_a, r.slot * kABytes), db = desc_at(desc_b, r.slot * kBBytes);
                            const uint32_t rows = deep - (t.k0 + k) * kBK;
                            if (MODE == kWeightGrad && rows < (uint32_t)kBK) {
                                pair_acquire<CG>();                // the other CTA zeroed rows of its operands
                                for (uint32_t q = 0; q < (rows + 15) / 16; ++q) mma_f16<CG>(d, desc_at(da, q * kStepA), desc_at(db, q * kStepB), idesc, ((k - k0) | q) != 0);
                            } else {
#pragma unroll
                                for (uint32_t q = 0; q < kBK / 16; ++q) mma_f16<CG>(d, desc_at(da, q * kStepA), desc_at(db, q * kStepB), idesc, ((k - k0) | q) != 0);
                            }
                            mma_commit<CG>(bar_empty + 8 * r.slot);
                            r.step();
                        }
                        if (ok) mma_commit<CG>(bar_acc_full + 8 * to.slot);
                        to.step();
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                at.skip(t.k_stages);
                acc.skip(LONG ? (t.k_stages + kChunk - 1) / kChunk : 1);
            }
        }
    } else if (LONG) {
        // ---- accumulators to sums, finished sums to memory ----
        if (BN == 256) regs_for_sums();
        constexpr int kCols = BN / 2;                 // columns of one set
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        unsigned char* stage = sm_store + (warp - 4) * 4096;
        const uint32_t lead_acc_empty = CG == 2 ? leader_addr(bar_acc_empty) : bar_acc_empty;
        Ring<kAccs> acc;
        while (ok && pieces.next(p, tiles_m, tiles_n, &t, &bad)) {
            uint64_t sum[kCols / 2];
#pragma unroll
            for (int i = 0; i < kCols / 2; ++i) sum[i] = 0ull;
            for (uint32_t k = 0; k < t.k_stages; k += kChunk) {
                if (!mbar_wait(bar_acc_full + 8 * acc.slot, acc.round & 1, failed)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d = tmem + acc.slot * BN + half * kCols + ((uint32_t)(quarter * 32) << 16);
                uint32_t r[2][32];
                tmem_ld32(d, r[0]);
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) {
                    tmem_ld_wait(r[c & 1]);
                    if (c + 1 < kCols / 32) {
                        tmem_ld32(d + 32 * (c + 1), r[(c + 1) & 1]);
                    } else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) pair_arrive_read<CG>(lead_acc_empty + 8 * acc.slot);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) add2(sum[16 * c + i], pair_of(r[c & 1][2 * i], r[c & 1][2 * i + 1]));
                }
                acc.step();
            }
            if (!ok) break;
            const bool partial = MODE == kWeightGrad && !t.whole;
            const uint32_t row0 = t.m + rank * kBM + quarter * 32, end = MODE == kWeightGrad ? p.out_rows : t.span.end;
            const uint32_t col0 = t.n * width + half * kCols, room = width - half * kCols;      // 32 columns at least
            RowStore rs;
            rs.bf16 = p.bf16 != 0;
            rs.f32 = partial || p.f32;
            rs.gate = nullptr;
            rs.gate_row_bytes = p.gate_row_bytes;
            rs.rows = row0 >= end ? 0u : end - row0 < 32 ? end - row0 : 32u;
            unsigned char* out;
            if (partial) {
                // slot 0: the tile began with an earlier worker; slot 1: it goes on with the next one
                out = reinterpret_cast<unsigned char*>(p.partial + (((size_t)t.worker * 2 + (t.first ? 1 : 0)) * CG + rank) * kBM * BN) +
                      ((size_t)quarter * 32 * BN + half * kCols) * 4;
                rs.row_bytes = BN * 4;
            } else {
                out = p.out + (MODE == kWeightGrad ? t.group * p.out_group_bytes : 0ull) + row0 * p.out_row_bytes + (size_t)col0 * (rs.f32 ? 4 : 2);
                rs.row_bytes = p.out_row_bytes;
            }
            const uint32_t cols = col0 >= p.out_cols ? 0u : min(min(p.out_cols - col0, (uint32_t)kCols), room);
            if (rs.f32) {
#pragma unroll
                for (int c = 0; c < kCols; c += 32) {
                    if ((uint32_t)c >= cols) continue;
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        float v[4] = {lo_of(sum[c / 2 + 2 * u]), hi_of(sum[c / 2 + 2 * u]), lo_of(sum[c / 2 + 2 * u + 1]), hi_of(sum[c / 2 + 2 * u + 1])};
                        if (MODE == kLayer && p.relu) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = relu(v[e]);
                        }
                        stage_unit(stage, lane, u, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
                    }
                    rs.bytes = (cols - c < 32u ? cols - c : 32u) * 4u;
                    rs.out = out + (size_t)c * 4;
                    if (MODE == kInputGrad && p.gate) {
                        uint4 hv[8];
                        rs.gate = p.gate + row0 * p.gate_row_bytes + (size_t)(col0 + c) * 2;
                        load_gate(rs, hv);
                        store_rows<true>(rs, stage, hv);
                    } else {
                        store_rows(rs, stage);
                    }
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
                        for (int e = 0; e < 4; ++e) {
                            const float lo = lo_of(sum[c / 2 + 4 * u + e]), hi = hi_of(sum[c / 2 + 4 * u + e]);
                            w[e] = MODE == kLayer && p.relu ? pack16_relu(lo, hi, rs.bf16) : pack16(lo, hi, rs.bf16);
                        }
                        stage_unit(stage, lane, u, make_uint4(w[0], w[1], w[2], w[3]));
                    }
                    rs.bytes = (cols - c < (uint32_t)kPer ? cols - c : (uint32_t)kPer) * 2u;
                    rs.out = out + (size_t)c * 2;
                    if (MODE == kInputGrad && p.gate) {
                        uint4 hv[8];
                        rs.gate = p.gate + row0 * p.gate_row_bytes + (size_t)(col0 + c) * 2;
                        load_gate(rs, hv);
                        store_rows<true>(rs, stage, hv);
                    } else {
                        store_rows(rs, stage);
                    }
                }
            }
        }
    } else {
        // ---- finished accumulators to memory ----
        const int quarter = warp & 3, set = (warp - 4) >> 2;
        unsigned char* stage = sm_store + (warp - 4) * 4096;
        const uint32_t lead_acc_empty = CG == 2 ? leader_addr(bar_acc_empty) : bar_acc_empty;
        uint32_t acc = set, acc_round = 0;
        while (pieces.next(p, tiles_m, tiles_n, &t, &bad)) {
            RowStore rs;
            rs.bf16 = p.bf16 != 0;
            rs.gate = nullptr;
            rs.gate_row_bytes = p.gate_row_bytes;
            const bool gated = MODE == kInputGrad && p.gate;
            rs.f32 = p.f32;
            const uint32_t row0 = t.m + rank * kBM + quarter * 32;
            rs.rows = row0 >= t.span.end ? 0u : t.span.end - row0 < 32 ? t.span.end - row0 : 32u;
            const uint32_t col0 = t.n * width;
            const uint32_t cols = p.out_cols - col0 < width ? p.out_cols - col0 : width;
            unsigned char* out = p.out + row0 * p.out_row_bytes;
            rs.row_bytes = p.out_row_bytes;
            const uint32_t per = rs.f32 ? 32u : 64u, size = rs.f32 ? 4u : 2u;
            auto piece = [&](uint32_t c) {
                rs.bytes = (cols - c < per ? cols - c : per) * size;
                rs.out = out + (size_t)(col0 + c) * size;
                if (gated) rs.gate = p.gate + row0 * p.gate_row_bytes + (size_t)(col0 + c) * 2;
            };
            uint4 hv[8];
            piece(0);
            if (gated) load_gate(rs, hv);                  // on its way while the sums finish
            if (!mbar_wait(bar_acc_full + 8 * acc, acc_round & 1, failed)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d = tmem + acc * BN + ((uint32_t)(quarter * 32) << 16);
            for (uint32_t c = 0; c < cols; c += per) {
                uint32_t r[32];
                if (rs.f32) {
                    tmem_ld32(d + c, r);
                    tmem_ld_wait(r);
                    if (p.relu)
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(relu(__uint_as_float(r[i])));
#pragma unroll
                    for (int u = 0; u < 8; ++u) stage_unit(stage, lane, u, make_uint4(r[4 * u], r[4 * u + 1], r[4 * u + 2], r[4 * u + 3]));
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (c + 32u * h < cols) {
                            tmem_ld32(d + c + 32 * h, r);
                            tmem_ld_wait(r);
                            uint32_t o[16];
                            pack32(r, o, rs.bf16, p.relu != 0);
#pragma unroll
                            for (int u = 0; u < 4; ++u) stage_unit(stage, lane, 4 * h + u, make_uint4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]));
                        }
                    }
                }
                if (c + per >= cols) {             // the accumulator is read: a later tile may have it
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) pair_arrive_read<CG>(lead_acc_empty + 8 * acc);
                }
                if (gated) {
                    store_rows<true>(rs, stage, hv);
                    if (c + per < cols) {
                        piece(c + per);
                        load_gate(rs, hv);
                    }
                } else {
                    store_rows(rs, stage);
                    piece(c + per);
                }
            }
            acc += 2;
            if (acc >= kAccs) { acc -= kAccs; ++acc_round; }
        }
    }
    if ((bad || (!ok && lane == 0)) && p.error_flags) atomicOr(p.error_flags, (ok ? 0u : 2u) | (bad ? 16u : 0u));
    tc_fence_before();
    if (CG == 2) cluster_sync(); else __syncthreads();      // a pair's barriers and accumulators serve both CTAs to the end
    if (warp == 2) tmem_free<CG>(tmem, kTmemCols);
}

// Second kernel of the weight gradient: sums the partial sums of every output tile that a boundary between two workers
// cuts, in a fixed order of the workers, and writes the zeros of groups without samples.  A block takes a slice of a tile:
// LANES threads share a quad of sums, each taking every LANES-th worker.
//
// BY_TILE: blocks (tile, slice).  Otherwise, where there are more tiles than boundaries, blocks (v, slice) with v <
// n_workers - 1 for the boundary behind worker v, which take the tile when this boundary is the first to cut it, and
// blocks (n_workers - 1 + g, slice) for the zeros of group g.
constexpr int kJoinThreads = 256;
template <int BN, int CG, int LANES> __host__ __device__ constexpr int join_slices() { return CG * kBM * BN / 4 / (LANES == 1 ? 512 : kJoinThreads / LANES); }

template <int BN, int CG, int LANES, bool BY_TILE>
__global__ void __launch_bounds__(kJoinThreads) k_weight_grad_join(const GroupedArgs p) {
    constexpr uint32_t kSlices = join_slices<BN, CG, LANES>(), kQuads = CG * kBM * BN / 4 / kSlices;
    const uint32_t width = CG == 2 ? p.width : BN;
    const uint32_t tiles_n = (p.out_cols + width - 1) / width, tiles_m = (p.out_rows + CG * kBM - 1) / (CG * kBM);
    const uint32_t across = tiles_m * tiles_n, slice = blockIdx.y, n = p.n_workers;
    wait_for_inputs();
    let_next_start();
    bool bad = false;
    if (!BY_TILE && blockIdx.x >= n - 1) {
        const uint32_t g = blockIdx.x - (n - 1);
        const Span s = group_span(p.offsets, g, p.n_rows, &bad);
        if (s.end > s.begin) return;
        for (uint32_t row = slice; row < p.out_rows; row += kSlices) {
            unsigned char* o = p.out + g * p.out_group_bytes + row * p.out_row_bytes;
            for (uint32_t col = threadIdx.x; col < p.out_cols; col += kJoinThreads) {
                if (p.f32) reinterpret_cast<float*>(o)[col] = 0.f;
                else reinterpret_cast<uint16_t*>(o)[col] = 0;
            }
        }
        return;
    }
    __shared__ uint32_t sh[6];         // first and last worker of the tile, its group, m, n; no samples
    if (threadIdx.x < 32) {
        auto units_of = [&](const Span& q) { return group_units<kWeightGrad, CG>(q, across); };
        uint32_t group = 0, local = 0, v0 = 1, v1 = 0, tm = 0, tn = 0, empty = 0;
        if (BY_TILE) {
            // units of all groups, and of those in front of this one
            group = blockIdx.x / across;
            uint32_t all = 0, before = 0;
            for (uint32_t g = threadIdx.x; g < p.n_groups; g += 32) {
                const uint32_t u = units_of(group_span(p.offsets, g, p.n_rows, &bad));
                all += u;
                before += g < group ? u : 0;
            }
            all = __reduce_add_sync(0xffffffffu, all);
            before = __reduce_add_sync(0xffffffffu, before);
            const Span s = group_span(p.offsets, group, p.n_rows, &bad);
            const uint32_t t = blockIdx.x - group * across, deep = (s.end - s.begin + kBK - 1) / kBK;
            tile_place(t, tiles_m, tiles_n, &tm, &tn);
            if (!deep) {
                empty = 1;
            } else {
                const uint32_t q = all / n, r = all - q * n;
                auto owner = [&](uint32_t u) { return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q; };
                const uint32_t u0 = before + t * (deep + kTileUnits) + kTileUnits, a = owner(u0), b = owner(u0 + deep - 1);
                if (a < b) { v0 = a; v1 = b; }
            }
        } else {
            const uint32_t units = all_units<kWeightGrad, CG>(p, across, &bad);
            const uint32_t u = first_unit(units, blockIdx.x + 1, n);       // first unit behind the boundary
            GroupWalk walk;
            Span s = {0, 0};
            if (u > 0 && u < units && walk.find(u, p.offsets, p.n_groups, p.n_rows, units_of, &group, &s, &local, &bad)) {
                const uint32_t deep = (s.end - s.begin + kBK - 1) / kBK, t = local / (deep + kTileUnits);
                const uint32_t u0 = u - (local - t * (deep + kTileUnits)) + kTileUnits, before = first_unit(units, blockIdx.x, n);
                // the boundary cuts the tile's stages (the first of which is unit u0), and the one in front of it does not
                if (u > u0 && before <= u0) {
                    v0 = blockIdx.x;
                    v1 = v0 + 1;
                    while (v1 + 1 < n && first_unit(units, v1 + 1, n) < u0 + deep) ++v1;
                    tile_place(t, tiles_m, tiles_n, &tm, &tn);
                }
            }
        }
        if (threadIdx.x == 0) { sh[0] = v0; sh[1] = v1; sh[2] = group; sh[3] = tm; sh[4] = tn; sh[5] = empty; }
    }
    __syncthreads();
    const uint32_t v0 = sh[0], v1 = sh[1], empty = sh[5], part = threadIdx.x % LANES;
    if (v0 > v1 && !empty) return;
    for (uint32_t i = threadIdx.x / LANES; i < kQuads; i += kJoinThreads / LANES) {
        const uint32_t at = slice * kQuads + i, row = at / (BN / 4), col = at % (BN / 4) * 4;
        const uint32_t orow = sh[3] * (CG * kBM) + row, ocol = sh[4] * width + col;
        const bool inside = orow < p.out_rows && ocol < p.out_cols && col < width;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (inside && !empty) {
            const float4* q = reinterpret_cast<const float4*>(p.partial + (size_t)row * BN + col);
            constexpr size_t kSlot = (size_t)CG * kBM * BN / 4;
#pragma unroll 4
            for (uint32_t v = v0 + part; v <= v1; v += LANES) {
                const float4 e = __ldcg(q + (2 * (size_t)v + (v == v0 ? 1 : 0)) * kSlot);
                sum.x += e.x; sum.y += e.y; sum.z += e.z; sum.w += e.w;
            }
        }
#pragma unroll
        for (int d = LANES / 2; d; d >>= 1) {
            sum.x += __shfl_xor_sync(0xffffffffu, sum.x, d);
            sum.y += __shfl_xor_sync(0xffffffffu, sum.y, d);
            sum.z += __shfl_xor_sync(0xffffffffu, sum.z, d);
            sum.w += __shfl_xor_sync(0xffffffffu, sum.w, d);
        }
        if (!inside || part) continue;
        unsigned char* o = p.out + sh[2] * p.out_group_bytes + orow * p.out_row_bytes;
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
        if (p.f32 && ocol + 4 <= p.out_cols) {
            reinterpret_cast<float4*>(o)[ocol / 4] = sum;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (ocol + e >= p.out_cols) continue;
                if (p.f32) reinterpret_cast<float*>(o)[ocol + e] = f[e];
                else reinterpret_cast<uint16_t*>(o)[ocol + e] = (uint16_t)pack16(f[e], 0.f, p.bf16 != 0);
            }
        }
    }
}

// Width of a pair's tiles: as many tiles as 256 columns each would make, evenly.
uint32_t pair_width(uint32_t cols) {
    const uint32_t tiles = (cols + 255) / 256, even = ((cols + tiles - 1) / tiles + 31) / 32 * 32;
    return even < 160 ? 160 : even;
}

// Shape and shares of the weight gradient.
struct WeightGradPlan { int bn, cg; uint32_t width; uint64_t across; uint32_t grid, workers; };
WeightGradPlan plan_weight_grad(const srf_grouped_t& p, int sms) {
    WeightGradPlan w;
    w.cg = p.n_out > 128 && p.n_in > 128 ? 2 : 1;
    w.bn = p.n_in <= 64 ? 64 : p.n_in <= 128 ? 128 : 256;
    w.width = w.cg == 2 ? pair_width(p.n_in) : w.bn;
    w.across = (uint64_t)((p.n_out + w.cg * kBM - 1) / (w.cg * kBM)) * ((p.n_in + w.width - 1) / w.width);
    const uint64_t filled = p.n_groups < p.n_rows ? p.n_groups : p.n_rows;
    const uint64_t units = (max_row_tiles(p, kBK) + filled * kTileUnits) * w.across, teams = sms / w.cg;
    const uint64_t busy = units < teams ? units : teams;
    // All teams together walk the samples once per tile of a group that a team works on; samples beyond what L2 holds are
    // taken in two parts (16389 x 2048 x 2048 with its input gradient: 355 us in one, 305 in two, 310 in three, 329 in
    // four -- every part cuts as many tiles again).  Weight gradients alone, in one / two parts: 131072 x 768 x 768 in 16 groups
    // 195 / 143 us, 65536 x 1024 x 1024 in one 154 / 156, 262144 x 512 x 512 in 4 (4 tiles) 199 / 199; fewer tiles, 262144 x
    // 256 x 256 in 16 groups, 75 / 83; fewer bytes, 4096 x 2048 x 2048 in 8, 66 / 73.
    const uint64_t bytes = p.n_rows * (p.n_in + p.n_out) * 2;
    const uint64_t parts = w.across >= 8 && bytes > (64ull << 20) ? 2 : 1;
    w.grid = (uint32_t)busy * w.cg;
    w.workers = (uint32_t)(busy * parts);
    if (!w.workers) w.workers = 1;
    return w;
}

// Whether sums of `depth` products take a LONG kernel.  One accumulator is off by up to 1.3e-5 of the sum at 2048 products of one
// sign, 5.3e-5 at 8192, 4.3e-4 at 65536 (a LONG kernel 2.8e-6 at all of them): too much for an fp32 result; a ninth of fp16's half
// step of 4.9e-4 at 8192, but all of it at 65536; at most a ninth of bf16's 3.9e-3 at any depth.
bool long_sums(const srf_grouped_t& p, uint32_t depth) {
    return p.out_type == SRF_TYPE_F32 ? depth > kChunk * kBK : p.out_type == SRF_TYPE_F16 && depth > 8192;
}

template <int MODE, int BN, int CG, bool LONG>
const char* launch(const CUtensorMap& a, const CUtensorMap& b, const GroupedArgs& args, uint32_t grid, cudaStream_t stream) {
    static_assert(smem_bytes<BN, CG>() <= 227 * 1024, "shared memory of one SM");
    return launch_layer(k_grouped<MODE, BN, CG, LONG>, smem_bytes<BN, CG>(), kThreads, CG, dim3(grid), stream, a, b, args);
}

template <int MODE>
const char* launch_long(const CUtensorMap& a, const CUtensorMap& b, const GroupedArgs& k, TileShape t, uint32_t grid, cudaStream_t stream) {
    if (t.cg == 2) return launch<MODE, 256, 2, true>(a, b, k, grid, stream);
    switch (t.bn) {
    case 256: return launch<MODE, 256, 1, true>(a, b, k, grid, stream);
    case 128: return launch<MODE, 128, 1, true>(a, b, k, grid, stream);
    default: return launch<MODE, 64, 1, true>(a, b, k, grid, stream);
    }
}

}  // namespace

uint64_t max_row_tiles(const srf_grouped_t& p, uint64_t height) {
    const uint64_t busy = p.n_groups < p.n_rows ? p.n_groups : p.n_rows;
    return p.n_rows / height + busy;
}

TileShape pick_tile(const srf_grouped_t& p, uint32_t cols, int sms, int smallest, int cols_step) {
    // Pairs: groups of two 256-row tiles at least, and a tile for every SM.  32768 samples 1024 -> 1024 on single CTAs / pairs,
    // even groups of 128: 123 / 125 us, 256: 84 / 81 (uneven ones waste half of a pair's last tile), 512: 73 / 64, 2048: 64 / 55;
    // fewer tiles, 4 groups 1024 -> 256: 32 tiles 16.4 / 18.5, 128 tiles 30.7 / 28.9, 256 tiles (1024 -> 1024) 41.0 / 35.8.
    if (cols > 128 && p.n_rows / p.n_groups >= 512 && p.n_rows / 256 * ((cols + 255) / 256) >= (uint64_t)sms) return {cols_step == 32 ? (int)pair_width(cols) : 256, 2};
    // Otherwise the width that costs least: rounds of tiles over the SMs, times a tile's share of loads -- its columns, its
    // samples, and as much as 32 columns for what every tile costs (16 to 64 choose alike; 160 samples in 64 groups, 2048 -> 1408,
    // cold: 79.9 us, with 128 82.0; 3000 in 128, 512 -> 304: 19.7, with none 20.5, with 128 21.6).
    const uint64_t busy = p.n_groups < p.n_rows ? p.n_groups : p.n_rows;
    const uint64_t mean = (p.n_rows + busy - 1) / busy;
    const uint64_t row_tiles = mean <= 128 ? busy : p.n_rows / 128 + busy / 2;
    int best = smallest;
    uint64_t least = ~0ull;
    for (int bn = smallest; bn <= 256; bn *= 2) {
        const uint64_t tiles = row_tiles * ((cols + bn - 1) / bn);
        const uint64_t cost = (tiles + sms - 1) / sms * (bn + (mean < 128 ? mean : 128) + 32);
        if (cost <= least) { least = cost; best = bn; }
        if ((uint32_t)bn >= cols) break;
    }
    return {best, 1};
}

uint32_t tile_grid(const srf_grouped_t& p, uint32_t cols, TileShape t, int sms) {
    const uint64_t tiles = max_row_tiles(p, t.cg * 128) * ((cols + t.bn - 1) / t.bn), teams = sms / t.cg;
    return (uint32_t)(tiles < teams ? tiles : teams) * t.cg;
}

int sm_count() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

bool make_operand_map(void* map, const void* base, int type, uint64_t cols, uint64_t rows, uint64_t ld, uint64_t n_matrices,
                      uint64_t matrix_stride, uint32_t box_rows) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    if (!encode) return false;
    const uint64_t size = type == SRF_TYPE_E4M3 ? 1 : 2;
    const cuuint32_t rank = n_matrices ? 3 : 2;
    const cuuint64_t dims[3] = {cols, rows, n_matrices};
    const cuuint64_t strides[2] = {ld * size, matrix_stride * size};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / size), box_rows, 1};
    const cuuint32_t step[3] = {1, 1, 1};
    const CUtensorMapDataType dt = type == SRF_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : type == SRF_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    return encode(reinterpret_cast<CUtensorMap*>(map), dt, rank, const_cast<void*>(base), dims, strides, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

const char* launch_grouped_matmul(const srf_grouped_t& p, const uint64_t* offsets, const void* x, const void* w, void* y,
                                  unsigned int* error_flags, cudaStream_t stream) {
    if (!p.n_rows) return nullptr;
    const int sms = sm_count();
    const TileShape t = pick_tile(p, p.n_out, sms, long_sums(p, p.n_in) ? 64 : 32, 32);
    CUtensorMap a, b;
    if (!make_operand_map(&a, x, p.type, p.n_in, p.n_rows, p.ld_x, 0, 0, t.cg == 2 ? kBM : kRowBox) ||
        !make_operand_map(&b, w, p.type, p.n_in, p.n_out, p.ld_w, p.n_groups, p.group_stride, t.bn / t.cg))
        return "the driver refused an operand's tensor map";
    GroupedArgs k;
    memset(&k, 0, sizeof(k));
    k.offsets = offsets; k.out = (unsigned char*)y; k.n_rows = (uint32_t)p.n_rows; k.n_groups = p.n_groups;
    k.f32 = p.out_type == SRF_TYPE_F32; k.bf16 = p.type == SRF_TYPE_BF16; k.relu = p.activation == SRF_ACT_RELU;
    k.out_row_bytes = p.ld_y * (k.f32 ? 4 : 2); k.out_cols = p.n_out; k.depth = p.n_in; k.width = t.bn; k.error_flags = error_flags;
    const uint32_t grid = tile_grid(p, p.n_out, t, sms);
    if (long_sums(p, p.n_in)) return launch_long<kLayer>(a, b, k, t, grid, stream);
    if (t.cg == 2) return launch<kLayer, 256, 2, false>(a, b, k, grid, stream);
    switch (t.bn) {
    case 256: return launch<kLayer, 256, 1, false>(a, b, k, grid, stream);
    case 128: return launch<kLayer, 128, 1, false>(a, b, k, grid, stream);
    case 64: return launch<kLayer, 64, 1, false>(a, b, k, grid, stream);
    default: return launch<kLayer, 32, 1, false>(a, b, k, grid, stream);
    }
}

const char* launch_grouped_input_grad(const srf_grouped_t& p, const uint64_t* offsets, const void* dy, const void* w,
                                      const void* gate, void* dx, unsigned int* error_flags, cudaStream_t stream) {
    if (!p.n_rows) return nullptr;
    const int sms = sm_count();
    const TileShape t = pick_tile(p, p.n_in, sms, 64, 32);
    CUtensorMap a, b;
    if (!make_operand_map(&a, dy, p.type, p.n_out, p.n_rows, p.ld_y, 0, 0, t.cg == 2 ? kBM : kRowBox) ||
        !make_operand_map(&b, w, p.type, p.n_in, p.n_out, p.ld_w, p.n_groups, p.group_stride, kBK))
        return "the driver refused an operand's tensor map";
    GroupedArgs k;
    memset(&k, 0, sizeof(k));
    k.offsets = offsets; k.out = (unsigned char*)dx; k.gate = (const unsigned char*)gate; k.n_rows = (uint32_t)p.n_rows; k.n_groups = p.n_groups;
    k.f32 = p.out_type == SRF_TYPE_F32; k.bf16 = p.type == SRF_TYPE_BF16;
    k.out_row_bytes = p.ld_x * (k.f32 ? 4 : 2); k.gate_row_bytes = p.ld_x * 2; k.out_cols = p.n_in; k.depth = p.n_out; k.width = t.bn;
    k.error_flags = error_flags;
    const uint32_t grid = tile_grid(p, p.n_in, t, sms);
    if (long_sums(p, p.n_out)) return launch_long<kInputGrad>(a, b, k, t, grid, stream);
    if (t.cg == 2) return launch<kInputGrad, 256, 2, false>(a, b, k, grid, stream);
    switch (t.bn) {
    case 256: return launch<kInputGrad, 256, 1, false>(a, b, k, grid, stream);
    case 128: return launch<kInputGrad, 128, 1, false>(a, b, k, grid, stream);
    default: return launch<kInputGrad, 64, 1, false>(a, b, k, grid, stream);
    }
}

size_t grouped_weight_grad_workspace(const srf_grouped_t& p, int n_sms) {
    const WeightGradPlan w = plan_weight_grad(p, n_sms);
    return (size_t)w.workers * 2 * w.cg * kBM * w.bn * sizeof(float);
}

namespace {

template <int BN, int CG>
const char* weight_grad(const CUtensorMap& a, const CUtensorMap& b, const GroupedArgs& k, const WeightGradPlan& w, cudaStream_t stream) {
    if (w.grid) {
        const char* why = launch<kWeightGrad, BN, CG, true>(a, b, k, w.grid, stream);
        if (why) return why;
    }
    // Few tiles: all of them, and eight threads to a quad (each tile may have many partial sums); many tiles: the boundaries.
    const uint64_t tiles = w.across * k.n_groups;
    constexpr int kFine = join_slices<BN, CG, 8>(), kCoarse = join_slices<BN, CG, 1>();
    if (tiles * kFine <= 4096) return launch_layer(k_weight_grad_join<BN, CG, 8, true>, 0, kJoinThreads, 1, dim3((uint32_t)tiles, kFine), stream, k);
    if (tiles <= w.workers) return launch_layer(k_weight_grad_join<BN, CG, 1, true>, 0, kJoinThreads, 1, dim3((uint32_t)tiles, kCoarse), stream, k);
    return launch_layer(k_weight_grad_join<BN, CG, 1, false>, 0, kJoinThreads, 1, dim3(k.n_workers - 1 + k.n_groups, kCoarse), stream, k);
}

}  // namespace

const char* launch_grouped_weight_grad(const srf_grouped_t& p, const uint64_t* offsets, const void* dy, const void* x, void* dw,
                                       void* workspace, unsigned int* error_flags, cudaStream_t stream) {
    const WeightGradPlan w = plan_weight_grad(p, sm_count());
    GroupedArgs k;
    memset(&k, 0, sizeof(k));
    k.offsets = offsets; k.out = (unsigned char*)dw; k.partial = (float*)workspace; k.n_rows = (uint32_t)p.n_rows; k.n_groups = p.n_groups;
    k.f32 = p.out_type == SRF_TYPE_F32; k.bf16 = p.type == SRF_TYPE_BF16;
    k.out_row_bytes = p.ld_w * (k.f32 ? 4 : 2); k.out_group_bytes = p.group_stride * (k.f32 ? 4 : 2);
    k.out_rows = p.n_out; k.out_cols = p.n_in; k.width = w.width; k.n_workers = w.workers; k.error_flags = error_flags;
    CUtensorMap a, b;
    memset(&a, 0, sizeof(a));
    memset(&b, 0, sizeof(b));
    if (w.grid && (!make_operand_map(&a, dy, p.type, p.n_out, p.n_rows, p.ld_y, 0, 0, kBK) ||
                   !make_operand_map(&b, x, p.type, p.n_in, p.n_rows, p.ld_x, 0, 0, kBK)))
        return "the driver refused an operand's tensor map";
    if (w.cg == 2) return weight_grad<256, 2>(a, b, k, w, stream);
    switch (w.bn) {
    case 256: return weight_grad<256, 1>(a, b, k, w, stream);
    case 128: return weight_grad<128, 1>(a, b, k, w, stream);
    default: return weight_grad<64, 1>(a, b, k, w, stream);
    }
}

}  // namespace srf
