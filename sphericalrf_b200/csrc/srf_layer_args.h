// srf_layer_args.h -- argument checks of the layer operators (srf_grouped_matmul and its neighbours in srf_abi.h).
//
// Plain host C++ without a CUDA call, so that the refusals can be tested where there is no GPU.  Every refuse_*()
// returns the reason as text, empty when the call may go on, and resolves default strides.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <string>

#include "../../include/srf_abi.h"

namespace srf {

// One array of a call: n matrices of rows x cols, strides in elements.
struct Strided {
    const char* name;
    const void* p;
    uint64_t rows, cols, ld, size, n = 1, stride = 0;
    // bytes from the first to behind the last element; 0 when empty.  Valid strides keep it far below 2^64.
    unsigned __int128 span() const {
        if (!rows || !cols || !n) return 0;
        return ((unsigned __int128)(n - 1) * stride + (unsigned __int128)(rows - 1) * ld + cols) * size;
    }
};

inline std::string refuse_array(const Strided& a) {
    const std::string name = a.name;
    if (!a.span()) return "";
    if (!a.p) return name + " is NULL";
    if ((uintptr_t)a.p % 16) return name + " is not 16-byte aligned";
    if (a.ld < a.cols) return "row stride of " + name + " is less than its width";
    if (a.ld >= (1ull << 36) || a.stride >= (1ull << 38) || a.span() >> 40) return name + " is larger than 2^40 bytes";
    if ((a.ld * a.size) % 16 || (a.n > 1 && (a.stride * a.size) % 16)) return "strides of " + name + " are not multiples of 16 bytes (pad the rows)";
    if (a.n > 1 && (unsigned __int128)a.stride < (unsigned __int128)(a.rows - 1) * a.ld + a.cols) return "matrices of " + name + " overlap";
    return "";
}

inline std::string refuse_overlap(const Strided& out, std::initializer_list<Strided> ins) {
    const uintptr_t o0 = (uintptr_t)out.p, o1 = o0 + (uintptr_t)out.span();
    for (const Strided& a : ins) {
        const uintptr_t a0 = (uintptr_t)a.p, a1 = a0 + (uintptr_t)a.span();
        if (a.p && a.span() && out.span() && a0 < o1 && o0 < a1) return std::string(out.name) + " overlaps " + a.name;
    }
    return "";
}

inline std::string refuse_arrays(const Strided& out, std::initializer_list<Strided> ins) {
    std::string why = refuse_array(out);
    for (const Strided& a : ins)
        if (why.empty()) why = refuse_array(a);
    return why.empty() ? refuse_overlap(out, ins) : why;
}

inline uint64_t type_size(int type) { return type == SRF_TYPE_F32 ? 4 : type == SRF_TYPE_E4M3 ? 1 : 2; }

enum LayerCall { kCallMatmul, kCallGradient, kCallMatmulFp8 };

inline std::string refuse_grouped(const srf_grouped_t* in, LayerCall call, srf_grouped_t* p) {
    if (!in) return "srf_grouped_t is NULL";
    if (in->struct_size != sizeof(srf_grouped_t)) return "srf_grouped_t.struct_size does not match this library";
    *p = *in;
    if (p->reserved) return "srf_grouped_t.reserved must be 0";
    if (p->n_groups < 1 || p->n_groups > 4096) return "n_groups must be in [1, 4096]";
    if (p->n_rows >= (1ull << 31)) return "n_rows must be less than 2^31";
    if (p->n_in < 1 || p->n_in > 65536 || p->n_out < 1 || p->n_out > 65536) return "n_in and n_out must be in [1, 65536]";
    if (call == kCallMatmulFp8) {
        if (p->type != SRF_TYPE_E4M3) return "type must be SRF_TYPE_E4M3";
        if (p->out_type < SRF_TYPE_F16 || p->out_type > SRF_TYPE_F32) return "out_type must be SRF_TYPE_F16, SRF_TYPE_BF16 or SRF_TYPE_F32";
    } else {
        if (p->type != SRF_TYPE_F16 && p->type != SRF_TYPE_BF16) return "type must be SRF_TYPE_F16 or SRF_TYPE_BF16";
        if (p->out_type != p->type && p->out_type != SRF_TYPE_F32) return "out_type must be `type` or SRF_TYPE_F32";
    }
    if (call == kCallGradient && p->activation != SRF_ACT_NONE) return "a gradient takes no activation";
    if (p->activation != SRF_ACT_NONE && p->activation != SRF_ACT_RELU) return "activation must be SRF_ACT_NONE or SRF_ACT_RELU";
    if (!p->ld_x) p->ld_x = p->n_in;
    if (!p->ld_w) p->ld_w = p->n_in;
    if (!p->ld_y) p->ld_y = p->n_out;
    if (p->ld_x >= (1ull << 36) || p->ld_w >= (1ull << 36) || p->ld_y >= (1ull << 36)) return "row strides must be less than 2^36";
    if (!p->group_stride || p->n_groups == 1) p->group_stride = p->n_out * p->ld_w;
    return "";
}

inline std::string refuse_offsets(const srf_grouped_t& p, const uint64_t* d_offsets) {
    if (!d_offsets && p.n_groups != 1) return "d_offsets may be NULL for one group only";
    if ((uintptr_t)d_offsets % 8) return "d_offsets is not 8-byte aligned";
    return "";
}

inline Strided samples_in(const char* name, const void* p, const srf_grouped_t& g, int type) { return {name, p, g.n_rows, g.n_in, g.ld_x, type_size(type)}; }
inline Strided samples_out(const char* name, const void* p, const srf_grouped_t& g, int type) { return {name, p, g.n_rows, g.n_out, g.ld_y, type_size(type)}; }
inline Strided matrices(const char* name, const void* p, const srf_grouped_t& g, int type) {
    return {name, p, g.n_out, g.n_in, g.ld_w, type_size(type), g.n_groups, g.group_stride};
}
inline Strided offsets_array(const uint64_t* d, const srf_grouped_t& g) { return {"d_offsets", d, d ? 1ull : 0ull, g.n_groups + 1ull, g.n_groups + 1ull, 8}; }

inline std::string refuse_matmul(const srf_grouped_t* in, const uint64_t* d_offsets, const void* x, const void* w, const void* y, srf_grouped_t* p) {
    std::string why = refuse_grouped(in, kCallMatmul, p);
    if (why.empty()) why = refuse_offsets(*p, d_offsets);
    if (!why.empty()) return why;
    const Strided out = samples_out("d_y", y, *p, p->out_type);
    why = refuse_arrays(out, {samples_in("d_x", x, *p, p->type), matrices("d_w", w, *p, p->type)});
    return why.empty() ? refuse_overlap(out, {offsets_array(d_offsets, *p)}) : why;
}

inline std::string refuse_input_grad(const srf_grouped_t* in, const uint64_t* d_offsets, const void* dy, const void* w, const void* gate,
                                     const void* dx, srf_grouped_t* p) {
    std::string why = refuse_grouped(in, kCallGradient, p);
    if (why.empty()) why = refuse_offsets(*p, d_offsets);
    if (!why.empty()) return why;
    const Strided out = samples_in("d_dx", dx, *p, p->out_type);
    const Strided a = samples_out("d_dy", dy, *p, p->type), b = matrices("d_w", w, *p, p->type);
    why = gate ? refuse_arrays(out, {a, b, samples_in("d_gate", gate, *p, p->type)}) : refuse_arrays(out, {a, b});
    return why.empty() ? refuse_overlap(out, {offsets_array(d_offsets, *p)}) : why;
}

inline std::string refuse_weight_grad_shape(const srf_grouped_t* in, srf_grouped_t* p) {
    const std::string why = refuse_grouped(in, kCallGradient, p);
    if (!why.empty()) return why;
    if (p->n_rows > (1ull << 26)) return "n_rows must be at most 2^26 for a weight gradient";
    // the kernels count stages of 64 samples of 128 x 64 outputs (at the least), and 14 a tile, in 32 bits
    if ((p->n_rows / 64 + 15ull * p->n_groups) * ((p->n_out + 127ull) / 128) * ((p->n_in + 63ull) / 64) >= (1ull << 32)) return "n_rows x n_in x n_out is too large for one weight gradient";
    return "";
}

inline std::string refuse_weight_grad(const srf_grouped_t* in, const uint64_t* d_offsets, const void* dy, const void* x, const void* dw,
                                      const void* space, size_t space_bytes, srf_grouped_t* p) {
    std::string why = refuse_weight_grad_shape(in, p);
    if (why.empty()) why = refuse_offsets(*p, d_offsets);
    if (!why.empty()) return why;
    if (!space) return "d_workspace is NULL";
    const Strided out = matrices("d_dw", dw, *p, p->out_type);
    const Strided a = samples_out("d_dy", dy, *p, p->type), b = samples_in("d_x", x, *p, p->type), o = offsets_array(d_offsets, *p);
    const Strided s = {"d_workspace", space, 1, space_bytes, (space_bytes + 15) / 16 * 16, 1};
    why = refuse_arrays(out, {a, b, s});
    if (why.empty()) why = refuse_overlap(out, {o});
    return why.empty() ? refuse_overlap(s, {a, b, o}) : why;
}

// Scales have no padding: only their addresses and overlaps are checked.
inline std::string refuse_scales(const char* name, const void* scales, bool needed) {
    if (needed && !scales) return std::string(name) + " is NULL";
    if ((uintptr_t)scales % 4) return std::string(name) + " is not 4-byte aligned";
    return "";
}

inline std::string refuse_matmul_fp8(const srf_grouped_t* in, const uint64_t* d_offsets, const void* x, const float* x_scales, const void* w,
                                     const float* w_scales, const void* y, srf_grouped_t* p) {
    std::string why = refuse_grouped(in, kCallMatmulFp8, p);
    if (why.empty()) why = refuse_offsets(*p, d_offsets);
    if (why.empty()) why = refuse_scales("d_x_scales", x_scales, p->n_rows > 0);
    if (why.empty()) why = refuse_scales("d_w_scales", w_scales, p->n_rows > 0);
    if (!why.empty()) return why;
    const uint64_t kb = (p->n_in + 127) / 128, nb = (p->n_out + 127) / 128;
    const Strided out = samples_out("d_y", y, *p, p->out_type);
    why = refuse_arrays(out, {samples_in("d_x", x, *p, p->type), matrices("d_w", w, *p, p->type)});
    return why.empty() ? refuse_overlap(out, {{"d_x_scales", x_scales, kb, p->n_rows, p->n_rows, 4}, {"d_w_scales", w_scales, p->n_groups * nb, kb, kb, 4},
                                              offsets_array(d_offsets, *p)}) : why;
}

inline std::string refuse_quantize_rows(int type, uint64_t n_rows, const uint64_t* d_n_rows_used, uint32_t n_cols, const void* in, uint64_t* ld_in,
                                        const void* out, uint64_t* ld_out, const float* scales) {
    if (type != SRF_TYPE_F16 && type != SRF_TYPE_BF16) return "type must be SRF_TYPE_F16 or SRF_TYPE_BF16";
    if (n_rows >= (1ull << 31)) return "n_rows must be less than 2^31";
    if (n_cols < 1 || n_cols > 65536) return "n_cols must be in [1, 65536]";
    if ((uintptr_t)d_n_rows_used % 8) return "d_n_rows_used is not 8-byte aligned";
    std::string why = refuse_scales("d_scales", scales, n_rows > 0);
    if (!why.empty()) return why;
    if (!*ld_in) *ld_in = n_cols;
    if (!*ld_out) *ld_out = n_cols;
    const Strided v = {"d_in", in, n_rows, n_cols, *ld_in, 2}, q = {"d_out", out, n_rows, n_cols, *ld_out, 1};
    const Strided s = {"d_scales", scales, (n_cols + 127u) / 128u, n_rows, n_rows, 4}, c = {"d_n_rows_used", d_n_rows_used, d_n_rows_used ? 1ull : 0ull, 1, 1, 8};
    why = refuse_arrays(q, {v});
    if (why.empty()) why = refuse_overlap(q, {c});
    return why.empty() ? refuse_overlap(s, {v, q, c}) : why;
}

inline std::string refuse_quantize_weights(int type, uint32_t n_matrices, uint32_t n_rows, uint32_t n_cols, const void* in, uint64_t* ld_in,
                                           const void* out, uint64_t* ld_out, const float* scales) {
    if (type != SRF_TYPE_F16 && type != SRF_TYPE_BF16) return "type must be SRF_TYPE_F16 or SRF_TYPE_BF16";
    if (n_matrices < 1 || n_matrices > 4096) return "n_matrices must be in [1, 4096]";
    if (n_rows < 1 || n_rows > 65536 || n_cols < 1 || n_cols > 65536) return "n_rows and n_cols must be in [1, 65536]";
    std::string why = refuse_scales("d_scales", scales, true);
    if (!why.empty()) return why;
    if (!*ld_in) *ld_in = n_cols;
    if (!*ld_out) *ld_out = n_cols;
    if (*ld_in >= (1ull << 36) || *ld_out >= (1ull << 36)) return "row strides must be less than 2^36";
    const Strided v = {"d_in", in, n_rows, n_cols, *ld_in, 2, n_matrices, n_rows * *ld_in}, q = {"d_out", out, n_rows, n_cols, *ld_out, 1, n_matrices, n_rows * *ld_out};
    const uint64_t nb = (n_cols + 127u) / 128u;
    const Strided s = {"d_scales", scales, (uint64_t)n_matrices * ((n_rows + 127u) / 128u), nb, nb, 4};
    why = refuse_arrays(q, {v});
    return why.empty() ? refuse_overlap(s, {v, q}) : why;
}

}  // namespace srf
