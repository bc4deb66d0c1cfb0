// srf_tile.cuh -- what the layer kernels (srf_grouped.cu, srf_grouped_fp8.cu) share: bounded barriers, TMA loads,
// tcgen05 wrappers, the walk over the output tiles of ragged groups, and the store of a finished tile.
//
// Shared-memory operands lie as a TMA load with 128-byte swizzle leaves them: rows of 128 bytes, eight rows to an atom
// of 1024 bytes whose 16-byte units are permuted by the row's number.  An operand whose long side is the summed axis
// (K-major) has one row per output row or column; one whose long side is the output axis (MN-major) has one row per
// summed index and a separate block of rows for every 64 output rows or columns.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace srf {
namespace tile {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0;
}
// Longest wait on one barrier, in cycles (about four seconds).  The longest wait that real work causes is for one accumulator:
// 1024 stages of a sum of 65536 products, well under a millisecond.
constexpr long long kWaitCycles = 8000000000ll;

// Bounded wait of one thread.  `failed` (shared memory) tells the CTA's other warps that one of them gave up.
__device__ __forceinline__ bool mbar_wait_one(uint32_t bar, uint32_t parity, volatile uint32_t* failed) {
    if (mbar_test(bar, parity)) return true;
    const long long t0 = clock64();
    for (uint32_t i = 1; i < (1u << 31); ++i) {
        if (mbar_test(bar, parity)) return true;
        if ((i & 63u) == 0 && (*failed != 0 || clock64() - t0 > kWaitCycles)) break;
    }
    *failed = 1;
    return false;
}
// The same for a whole warp, with one answer for all its lanes: a phase that one lane saw complete is complete.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* failed) {
    if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
    const bool done = mbar_wait_one(bar, parity, failed);
    return __any_sync(0xffffffffu, done);
}

// One lane of a converged warp, the same one every time.  The compiler knows that a single thread is behind it, which the
// instructions with uniform operands (TMA, tcgen05) are issued faster for than behind `lane == 0`.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}

// Programmatic dependent launch: a kernel's blocks may be set up while the kernel in front of it in the stream still runs.
// Nothing in global memory is touched in front of wait_for_inputs(), which returns when that kernel has completed and its
// writes are visible.  Loads behind it are ordinary ones (through L2 where nothing is read twice) or TMA's, never the
// read-only path: the data was not read-only while this kernel was on the GPU.
__device__ __forceinline__ void wait_for_inputs() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Place in a ring of `N` slots, advanced by all lanes of a warp alike.
template <int N>
struct Ring {
    uint32_t slot = 0, round = 0;
    __device__ __forceinline__ void step() { if (++slot == N) { slot = 0; ++round; } }
    __device__ __forceinline__ void skip(uint32_t n) {
        const uint32_t to = slot + n, turns = to / N;
        round += turns;
        slot = to - turns * N;
    }
};

// ---- pairs of CTAs (CG = 2): two SMs work on one tile, the CTA of rank 0 issues for both ----

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
// The address of this CTA's barrier `bar` in the CTA of rank 0.
__device__ __forceinline__ uint32_t leader_addr(uint32_t bar) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(bar));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// After a wait on arrivals of the pair's other CTA: what it wrote before them is visible.
template <int CG>
__device__ __forceinline__ void pair_acquire() {
    if (CG == 2) asm volatile("fence.acq_rel.cluster;" ::: "memory");
}
// Arrivals on the pair's barriers, which live in the CTA of rank 0; `leader` from leader_addr().  The one that announces
// bytes is relaxed: it publishes nothing, and a release per stage made the load warp wait for memory (1450 cycles a
// stage against 512 of matrix instructions).
template <int CG>
__device__ __forceinline__ void pair_expect(uint32_t leader, uint32_t bytes) {
    if (CG == 1) mbar_expect(leader, bytes);
    else asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" :: "r"(leader), "r"(bytes) : "memory");
}
template <int CG>
__device__ __forceinline__ void pair_arrive(uint32_t leader) {
    if (CG == 1) mbar_arrive(leader);
    else asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(leader) : "memory");
}

// "I have read this accumulator": nothing of this thread's is published (tcgen05.fence orders the reads), so relaxed, and
// no wait for its stores in flight.
template <int CG>
__device__ __forceinline__ void pair_arrive_read(uint32_t leader) {
    if (CG == 1) mbar_arrive(leader);
    else asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" :: "r"(leader) : "memory");
}

// TMA loads into this CTA's shared memory; the bytes are counted on the pair's barrier.
template <int CG>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    if (CG == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
                     :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    if (CG == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];"
                     :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" :: "l"(map) : "memory");
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Descriptor of a shared-memory operand with 128-byte swizzle.  K-major: `sbo` = 1024 (eight rows), lbo unused.
// MN-major: `sbo` = 1024 (eight summed indices), `lbo` = bytes between blocks of 64 output rows.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 | (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// The same operand `bytes` further on (a multiple of 16; the address field does not overflow inside shared memory).
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
                     :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
                     :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
                     :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
                     :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the barrier -- of both CTAs of a pair -- when the instructions issued so far are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     :: "r"(bar), "h"((uint16_t)3) : "memory");
}
// Waits (bounded) for the copies of a ring's last stages that nobody else will wait for; one warp of rank 0.
template <int N>
__device__ __forceinline__ void drain_ring(uint32_t bar_full, uint32_t issued) {
    issued = __reduce_max_sync(0xffffffffu, issued);
    for (uint32_t i = 0; i < issued && i < N; ++i) {
        const uint32_t q = issued - 1 - i;
        uint32_t none = 0;
        mbar_wait(bar_full + 8 * (q % N), (q / N) & 1, &none);
    }
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
    if (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(slot), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(base), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(base), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
// Completes the loads issued so far; `r` passes through, so that nothing that uses it can be moved in front.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
    asm volatile("" : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                      "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}

// The other way: 32 columns of this warp's 32 rows, in place when tmem_st_wait() has returned.
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n"
                 :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                    "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                    "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                    "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
                    "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Instruction descriptor bits common to both kinds: fp32 accumulator, m x n outputs.
__host__ __device__ constexpr uint32_t idesc_shape(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

// ---- ragged groups ----

// Samples [begin, end) of group g.  Offsets that point behind the buffers or run backwards are cut to what is there
// (every access stays in bounds) and reported through *bad.  n_rows < 2^31.
struct Span { uint32_t begin, end; };
__device__ __forceinline__ Span group_span(const uint64_t* __restrict__ offsets, uint32_t g, uint32_t n_rows, bool* bad) {
    Span s = {0, n_rows};
    if (offsets) {
        const uint64_t b = __ldcg((const unsigned long long*)offsets + g), e = __ldcg((const unsigned long long*)offsets + g + 1);
        if (b > e || e > n_rows) *bad = true;
        s.end = e < n_rows ? (uint32_t)e : n_rows;
        s.begin = b < s.end ? (uint32_t)b : s.end;
    }
    return s;
}

// Walks the groups in windows of 32, one group per lane: unit u of the concatenation of all groups' units belongs to
// the group whose running sum first exceeds u.  Units are asked for in ascending order, so a window is never revisited.
// `units(span)` gives a group's number of units; all groups together have less than 2^32 (arrays end at 2^40 bytes).
struct GroupWalk {
    uint32_t base = 0;       // units in front of the window
    uint32_t incl = 0;       // lane: units of the window up to and with this lane's group
    uint32_t own = 0;        // lane: units of this lane's group
    uint32_t total = 0;      // units of the window
    uint32_t g0 = 0;
    Span span = {0, 0};
    bool loaded = false;

    // Warp-collective.  False when there is no unit u.
    template <class Units>
    __device__ __forceinline__ bool find(uint32_t u, const uint64_t* offsets, uint32_t n_groups, uint32_t n_rows, Units units,
                                         uint32_t* group, Span* where, uint32_t* local, bool* bad) {
        const uint32_t lane = threadIdx.x & 31;
        for (;;) {
            if (!loaded) {
                if (g0 >= n_groups) return false;
                span = {0, 0};
                own = 0;
                if (g0 + lane < n_groups) {
                    span = group_span(offsets, g0 + lane, n_rows, bad);
                    own = units(span);
                }
                incl = own;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, d);
                    if ((int)lane >= d) incl += v;
                }
                total = __shfl_sync(0xffffffffu, incl, 31);
                loaded = true;
            }
            if (u - base < total) break;
            base += total;
            g0 += 32;
            loaded = false;
        }
        const int src = __ffs((int)__ballot_sync(0xffffffffu, incl > u - base)) - 1;
        where->begin = __shfl_sync(0xffffffffu, span.begin, src);
        where->end = __shfl_sync(0xffffffffu, span.end, src);
        *group = g0 + (uint32_t)src;
        *local = u - base - __shfl_sync(0xffffffffu, incl - own, src);
        return true;
    }
};

// Output tile `local` of a group of mt x nt tiles -> (m, n).  Tiles run down bands of 16 row tiles, so that the tiles
// in flight at one time share both operands in L2.
__device__ __forceinline__ void tile_place(uint32_t local, uint32_t mt, uint32_t nt, uint32_t* m, uint32_t* n) {
    const uint32_t band = local / (16u * nt);
    const uint32_t m0 = band * 16;
    const uint32_t height = mt - m0 < 16 ? mt - m0 : 16;
    const uint32_t r = local - m0 * nt;
    *n = r / height;
    *m = m0 + r - *n * height;
}

// ---- storing a finished piece of a tile ----

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
    uint32_t r;
    if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// The same with negative values clamped to zero and NaN kept, in one instruction.
__device__ __forceinline__ uint32_t pack16_relu(float lo, float hi, bool bf16) {
    uint32_t r;
    if (bf16) asm("cvt.rn.relu.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.relu.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 32 sums (as bits) -> 32 values of 16 bits.
__device__ __forceinline__ void pack32(const uint32_t (&r)[32], uint32_t (&o)[16], bool bf16, bool clamp) {
    if (clamp) {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = pack16_relu(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), bf16);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = pack16(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), bf16);
    }
}
// NaN stays NaN.
__device__ __forceinline__ float relu(float v) {
    asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(v));
    return v;
}

// x > 0 for a 16-bit value of either type: sign clear, not zero, not NaN.
__device__ __forceinline__ bool positive16(uint32_t h, bool bf16) {
    return h > 0u && h <= (bf16 ? 0x7f80u : 0x7c00u);
}

// Rows are written through a warp's 4 KB of shared memory so that every store instruction covers four whole 128-byte
// lines (a thread holds one row; storing from registers would touch 32 lines with 16 bytes each).  16-byte units are
// permuted by the row's number, which keeps both directions free of bank conflicts.
struct RowStore {
    unsigned char* out;        // the tile's first row, first column of the piece
    uint64_t row_bytes;        // between output rows
    const unsigned char* gate; // or NULL: 16-bit values, same place; a value that is not > 0 shuts the output
    uint64_t gate_row_bytes;
    uint32_t rows;             // rows of this warp's 32 that exist
    uint32_t bytes;            // bytes of the piece's 128 that exist
    bool bf16, f32;
};

__device__ __forceinline__ void stage_unit(unsigned char* stage, int row, int unit, uint4 v) {
    *reinterpret_cast<uint4*>(stage + row * 128 + ((unit ^ (row & 7)) << 4)) = v;
}

// Shuts outputs whose gate is not > 0: `w` holds 16 bytes of output, `h` the gate's values for them.
__device__ __forceinline__ uint4 gate_unit(uint4 w, uint4 h, bool f32, bool bf16) {
    uint32_t v[4] = {w.x, w.y, w.z, w.w};
    const uint32_t g[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (f32) {
            if (!positive16((g[e >> 1] >> ((e & 1) * 16)) & 0xffffu, bf16)) v[e] = 0u;
        } else {
            if (!positive16(g[e] & 0xffffu, bf16)) v[e] &= 0xffff0000u;
            if (!positive16(g[e] >> 16, bf16)) v[e] &= 0x0000ffffu;
        }
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// The gate's values of the units this lane will store, asked for before the tile's sums are ready.
__device__ __forceinline__ void load_gate(const RowStore& s, uint4 (&hv)[8]) {
    const int lane = threadIdx.x & 31, unit = lane & 7;
    const uint32_t from = (uint32_t)unit * 16u;
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const uint32_t row = (uint32_t)(it * 4 + (lane >> 3));
        hv[it] = make_uint4(0u, 0u, 0u, 0u);
        if (row < s.rows && from < s.bytes) {
            const unsigned char* gp = s.gate + row * s.gate_row_bytes + (s.f32 ? unit * 8 : unit * 16);
            const uint32_t have = s.bytes - from;
            if (have >= 16u) {
                if (s.f32) {
                    const uint2 t = __ldcg(reinterpret_cast<const uint2*>(gp));
                    hv[it] = make_uint4(t.x, t.y, 0u, 0u);
                } else {
                    hv[it] = __ldcg(reinterpret_cast<const uint4*>(gp));
                }
            } else {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(gp);
                const uint32_t n = s.f32 ? have / 4u : have / 2u;
                uint32_t t[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((uint32_t)e < n) t[e >> 1] |= (uint32_t)__ldcg(h + e) << ((e & 1) * 16);
                hv[it] = make_uint4(t[0], t[1], t[2], t[3]);
            }
        }
    }
}

// Staged rows -> memory; the whole warp.
template <bool GATE>
__device__ __forceinline__ void store_rows(const RowStore& s, const unsigned char* stage, const uint4 (&hv)[8]) {
    const int lane = threadIdx.x & 31, unit = lane & 7;
    const uint32_t from = (uint32_t)unit * 16u;
    uint4 v[8];
    __syncwarp();
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const uint32_t row = (uint32_t)(it * 4 + (lane >> 3));
        v[it] = *reinterpret_cast<const uint4*>(stage + row * 128 + ((unit ^ (row & 7)) << 4));
    }
    __syncwarp();
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const uint32_t row = (uint32_t)(it * 4 + (lane >> 3));
        if (row < s.rows && from < s.bytes) {
            if (GATE) v[it] = gate_unit(v[it], hv[it], s.f32, s.bf16);
            unsigned char* p = s.out + row * s.row_bytes + from;
            const uint32_t have = s.bytes - from;
            if (have >= 16u) {
                *reinterpret_cast<uint4*>(p) = v[it];
            } else {
                const uint32_t w[4] = {v[it].x, v[it].y, v[it].z, v[it].w};
                if (s.f32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((uint32_t)e * 4u < have) reinterpret_cast<uint32_t*>(p)[e] = w[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((uint32_t)e * 2u < have) reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(w[e >> 1] >> ((e & 1) * 16));
                }
            }
        }
    }
}
__device__ __forceinline__ void store_rows(const RowStore& s, const unsigned char* stage) {
    const uint4 none[8] = {};
    store_rows<false>(s, stage, none);
}

// ---- sums kept in registers, two to a 64-bit register ----

__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) { return (uint64_t)lo | (uint64_t)hi << 32; }
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
// Two fused multiply-adds, or two additions, each rounded once.
__device__ __forceinline__ void fma2(uint64_t& sum, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sum) : "l"(a), "l"(b));
}
__device__ __forceinline__ void add2(uint64_t& sum, uint64_t a) { asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum) : "l"(a)); }

// Registers of kernels whose 8 epilogue warps hold 128 sums a thread beside two pieces of 32 in flight.  A block of 384 is
// launched with 168 a thread (64512); a share of 72 for the issuing warps would use them all.  The compiler keeps to 168 for the
// whole kernel and spills 90 to 130 bytes in the 256-column kernels with such sums, 100 in the 8-bit ones, with either share.
constexpr int kRegsIssue = 64, kRegsSum = 216;
static_assert(128 * kRegsIssue + 256 * kRegsSum <= 384 * 168, "a larger share would wait for registers forever");
__device__ __forceinline__ void regs_for_issue() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kRegsIssue)); }
__device__ __forceinline__ void regs_for_sums() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kRegsSum)); }

}  // namespace tile
}  // namespace srf
