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
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// Longest wait on one barrier.  The longest wait that real work causes is the accumulation of one output tile over
// 2^26 rows, well under a second.
constexpr uint64_t kWaitNs = 4000000000ull;

// Bounded wait.  `failed` (shared memory) tells the CTA's other warps that one of them gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* failed) {
    if (mbar_test(bar, parity)) return true;
    uint64_t t0 = 0;
    for (uint32_t i = 1; i < (1u << 30); ++i) {
        if (mbar_test(bar, parity)) return true;
        if ((i & 255u) == 0) {
            if (*failed) return false;
            const uint64_t t = now_ns();
            if (!t0) t0 = t;
            else if (t - t0 > kWaitNs) break;
        }
    }
    *failed = 1;
    return false;
}

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
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

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(slot), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(base), "r"(cols) : "memory");
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
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Instruction descriptor bits common to both kinds: fp32 accumulator, M = 128.
__host__ __device__ constexpr uint32_t idesc_shape(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24); }

// ---- ragged groups ----

// Samples [begin, end) of group g.  Offsets that point behind the buffers or run backwards are cut to what is there
// (every access stays in bounds) and reported through *bad.
struct Span { uint64_t begin, end; };
__device__ __forceinline__ Span group_span(const uint64_t* __restrict__ offsets, uint32_t g, uint64_t n_rows, bool* bad) {
    Span s = {0, n_rows};
    if (offsets) {
        s.begin = __ldg((const unsigned long long*)offsets + g);
        s.end = __ldg((const unsigned long long*)offsets + g + 1);
        if (s.begin > s.end || s.end > n_rows) *bad = true;
        s.end = s.end < n_rows ? s.end : n_rows;
        s.begin = s.begin < s.end ? s.begin : s.end;
    }
    return s;
}

// Walks the groups in windows of 32, one group per lane: unit u of the concatenation of all groups' units belongs to
// the group whose running sum first exceeds u.  Units are asked for in ascending order, so a window is never revisited.
// `units(span)` gives a group's number of units.
struct GroupWalk {
    uint64_t base = 0;       // units in front of the window
    uint64_t incl = 0;       // lane: units of the window up to and with this lane's group
    uint64_t total = 0;      // units of the window
    uint32_t g0 = 0;
    Span span = {0, 0};
    bool loaded = false;

    // Warp-collective.  False when there is no unit u.
    template <class Units>
    __device__ __forceinline__ bool find(uint64_t u, const uint64_t* offsets, uint32_t n_groups, uint64_t n_rows, Units units,
                                         uint32_t* group, Span* where, uint64_t* local, bool* bad) {
        const uint32_t lane = threadIdx.x & 31;
        for (;;) {
            if (!loaded) {
                if (g0 >= n_groups) return false;
                span = {0, 0};
                incl = 0;
                if (g0 + lane < n_groups) {
                    span = group_span(offsets, g0 + lane, n_rows, bad);
                    incl = units(span);
                }
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint64_t v = __shfl_up_sync(0xffffffffu, incl, d);
                    if ((int)lane >= d) incl += v;
                }
                total = __shfl_sync(0xffffffffu, incl, 31);
                loaded = true;
            }
            if (u < base + total) break;
            base += total;
            g0 += 32;
            loaded = false;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, base + incl > u);
        const int src = __ffs((int)hit) - 1;
        const uint64_t before = __shfl_sync(0xffffffffu, incl, src) - __shfl_sync(0xffffffffu, units(span), src);
        where->begin = __shfl_sync(0xffffffffu, span.begin, src);
        where->end = __shfl_sync(0xffffffffu, span.end, src);
        *group = g0 + (uint32_t)src;
        *local = u - base - before;
        return true;
    }
};

// Output tile `local` of a group of mt x nt tiles -> (m, n).  Tiles run down bands of 16 row tiles, so that the tiles
// in flight at one time share both operands in L2.
__device__ __forceinline__ void tile_place(uint64_t local, uint64_t mt, uint32_t nt, uint64_t* m, uint32_t* n) {
    const uint64_t band = local / (16ull * nt);
    const uint64_t m0 = band * 16;
    const uint32_t height = (uint32_t)(mt - m0 < 16 ? mt - m0 : 16);
    const uint32_t r = (uint32_t)(local - band * 16ull * nt);
    *m = m0 + r % height;
    *n = r / height;
}

// ---- storing a finished piece of a tile ----

__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
    uint32_t r;
    if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// NaN stays NaN.
__device__ __forceinline__ float relu(float v) { return v < 0.f ? 0.f : v; }

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

// Staged rows -> memory; the whole warp.
__device__ __forceinline__ void store_rows(const RowStore& s, const unsigned char* stage) {
    const int lane = threadIdx.x & 31, unit = lane & 7;
    __syncwarp();
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const uint32_t row = (uint32_t)(it * 4 + (lane >> 3));
        if (row < s.rows && (uint32_t)unit * 16u < s.bytes) {
            uint4 v = *reinterpret_cast<const uint4*>(stage + row * 128 + ((unit ^ (row & 7)) << 4));
            unsigned char* p = s.out + row * s.row_bytes + unit * 16;
            const uint32_t have = s.bytes - (uint32_t)unit * 16u;       // > 0
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            if (s.gate) {
                const unsigned char* gp = s.gate + row * s.gate_row_bytes;
                if (s.f32) {
                    const uint16_t* h = reinterpret_cast<const uint16_t*>(gp + unit * 8);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((uint32_t)e * 4u < have && !positive16(h[e], s.bf16)) w[e] = 0u;
                } else {
                    const uint16_t* h = reinterpret_cast<const uint16_t*>(gp + unit * 16);
                    uint4 hv = make_uint4(0u, 0u, 0u, 0u);
                    if (have >= 16u) hv = __ldg(reinterpret_cast<const uint4*>(h));
                    else {
                        uint32_t t[4] = {0u, 0u, 0u, 0u};
                        for (uint32_t e = 0; e * 2u < have; ++e) t[e >> 1] |= (uint32_t)h[e] << ((e & 1u) * 16);
                        hv = make_uint4(t[0], t[1], t[2], t[3]);
                    }
                    const uint32_t hw[4] = {hv.x, hv.y, hv.z, hv.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (!positive16(hw[e] & 0xffffu, s.bf16)) w[e] &= 0xffff0000u;
                        if (!positive16(hw[e] >> 16, s.bf16)) w[e] &= 0x0000ffffu;
                    }
                }
            }
            if (have >= 16u) {
                *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            } else if (s.f32) {
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
    __syncwarp();
}

}  // namespace tile
}  // namespace srf
