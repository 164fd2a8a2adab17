// Thin PyTorch extension: the common GEMM calls validated, their scale factors passed through (or
// transformed) and launched from C++, so a call costs a few microseconds of host time.
//
// It covers the reference's hot entry points (csrc/apis/gemm.hpp:225-256 fp8_fp4_gemm,
// :289-324 m_grouped_fp8_fp4_gemm_contiguous, :424-453 bf16_gemm, csrc/apis/layout.hpp:37-92
// for the scale-factor pass-through and transform) for K-major, 16-byte-aligned operands with no
// bias, alpha or output epilogue.  For anything else -- and for any input these checks would
// reject -- the entry returns false and the Python layer runs its general path, which raises the
// reference's error messages.  The library is reached through function pointers the Python layer
// hands over from the loaded libdeep_gemm_amd.so, so both layers always use the same library.
#include <torch/extension.h>

#include <cstdint>
#include <cstring>
#include <stdexcept>
#include <string>

#include "../../include/deep_gemm_amd.h"

namespace {

using GemmFn = int (*)(const dg_gemm_args*, void*);
using TransformFn = int (*)(const void*, int32_t, int64_t, int64_t, int64_t, int32_t, int32_t, int32_t, int32_t,
                            int32_t, int32_t, int32_t, const int32_t*, int32_t, int32_t, int16_t*, int64_t, int32_t*,
                            void*);
using TakeFn = uint32_t (*)();
using LastErrorFn = const char* (*)();

GemmFn g_gemm = nullptr;
TransformFn g_transform = nullptr;
TakeFn g_take = nullptr;
LastErrorFn g_last_error = nullptr;
const volatile uint32_t* g_words = nullptr;

constexpr int kFP8FP8 = 0, kFP8FP4 = 1, kFP4FP4 = 2, kBF16 = 3;
constexpr int kNormal = 0, kPsum = 2, kIdx = 3, kMasked = 4;

void init(int64_t gemm, int64_t transform, int64_t take, int64_t last_error, int64_t words) {
    g_gemm = reinterpret_cast<GemmFn>(gemm);
    g_transform = reinterpret_cast<TransformFn>(transform);
    g_take = reinterpret_cast<TakeFn>(take);
    g_last_error = reinterpret_cast<LastErrorFn>(last_error);
    g_words = reinterpret_cast<const volatile uint32_t*>(words);
}

void check_rc(int rc) {
    if (rc != 0) {
        const char* msg = g_last_error != nullptr ? g_last_error() : nullptr;
        throw std::runtime_error(msg != nullptr && msg[0] ? msg : ("deep_gemm error " + std::to_string(rc)));
    }
}

// Errors that kernels of earlier calls reported through the library's sticky words (read with no
// synchronisation; the words live in host-mapped memory).
uint32_t pending_errors() {
    if (g_words == nullptr) return 0;
    uint32_t any = 0;
    for (int i = 0; i < 5; ++i) any |= g_words[i];   // (a word per DG_ERR_* bit)
    return any == 0u ? 0 : g_take();
}

// The same words as the Python layer's message (deep_gemm/_lib.py, error_message).
std::string error_message(uint32_t bits) {
    std::string msg;
    if (bits & DG_ERR_SF_INVALID)
        msg += "Invalid float32 SF: only the 8-bit exponent may be set (sign and mantissa must be 0)";
    if (bits & DG_ERR_M_INDICES) {
        if (!msg.empty()) msg += "; ";
        msg += "m_indices is not padded to the M-grouped alignment (every alignment-row block must hold one group "
               "id < num_groups followed only by -1 padding)";
    }
    const std::pair<uint32_t, const char*> others[] = {
        {DG_ERR_EXPERT_ID, "topk_idx holds an expert id >= num_groups, or a layout a group past the last adapter"},
        {DG_ERR_MOE_ROWS, "the pairs of topk_idx need more rows than num_rows"},
        {DG_ERR_TARGET, "target holds an index outside the vocabulary"},
    };
    for (const auto& [bit, text] : others)
        if (bits & bit) msg += (msg.empty() ? "" : "; ") + std::string(text);
    return msg + " [reported by a kernel of an earlier deep_gemm call]";
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t align_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

bool is_fp4(const at::Tensor& t) { return t.scalar_type() == at::kChar; }

// K-major check of the reference's get_major_type_ab (csrc/utils/layout.hpp:37-47), without its
// error (an ambiguous or MN-major operand goes to the general path).
bool k_major(const at::Tensor& t) {
    if (t.stride(-1) != 1) return false;
    return !(t.stride(-2) == 1 && t.size(-1) > 1 && t.size(-2) > 1);
}

// The kernel reads the operand in place: K rows of whole 16-byte units at 16-byte aligned
// addresses (the general path pads or transposes otherwise).
bool kernel_ready(const at::Tensor& t) {
    const int64_t elem = t.element_size();
    if ((t.size(-1) * elem) % 16 || (t.stride(-2) * elem) % 16 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15))
        return false;
    if (t.dim() == 3 && (t.stride(0) * elem) % 16) return false;
    return true;
}

// Scale factors in the kernels' layout: `sf` itself when it already is (check_sf_layout,
// csrc/apis/layout.hpp:37-65), else the output of the transform kernel
// (csrc/jit_kernels/transform_sf.hpp:15-105).  An undefined tensor: the general path decides.
// psum: the M-grouped layout of A's rows (its m_indices when rows_by_index), whose padding rows
// are skipped.
at::Tensor kernel_sf(const at::Tensor& sf, int64_t mn, int64_t k, int64_t gran_mn, int64_t gran_k, int64_t groups,
                     const at::Tensor* psum, bool rows_by_index, int64_t alignment, int64_t stream) {
    const auto dt = sf.scalar_type();
    if (dt != at::kFloat && dt != at::kShort) return {};
    const int64_t rank = groups > 0 ? 3 : 2;
    if (sf.dim() != rank || !(sf.stride(-1) == 1 || sf.stride(-2) == 1)) return {};
    if (groups > 0 && sf.size(0) != groups) return {};
    int64_t div_k = 64;
    if (dt == at::kFloat) {
        if (gran_k != 32 && gran_k != 128) return {};
        div_k = gran_k;
    } else if (gran_k != 32) {
        return {};
    }
    if (sf.size(-2) != ceil_div(mn, gran_mn) || sf.size(-1) != ceil_div(k, div_k)) return {};
    if (dt == at::kShort && gran_mn == 1 && sf.stride(-2) == 1 && sf.stride(-1) == align_up(sf.size(-2), 2)) {
        if (groups == 0 || sf.stride(0) == sf.stride(-1) * sf.size(-1)) return sf;
    }
    if (gran_mn < 1 || gran_mn > 128 || (gran_mn & (gran_mn - 1)) || !sf.is_cuda()) return {};
    if (rows_by_index && (gran_mn != 1 || groups > 0)) psum = nullptr;
    const int64_t nb = groups > 0 ? groups : 1;
    const int64_t k64 = ceil_div(k, 64), ld = align_up(mn, 2);
    at::Tensor out = at::empty({nb, k64, ld}, sf.options().dtype(at::kShort));
    const int64_t sb = groups > 0 ? sf.stride(0) : 0;
    check_rc(g_transform(sf.data_ptr(), dt == at::kFloat ? DG_SF_F32 : DG_SF_I16, sb, sf.stride(-2), sf.stride(-1),
                         (int32_t)nb, (int32_t)sf.size(-2), (int32_t)sf.size(-1), (int32_t)mn, (int32_t)k,
                         (int32_t)gran_mn, (int32_t)gran_k,
                         psum != nullptr ? psum->data_ptr<int32_t>() : nullptr,
                         psum == nullptr ? 0 : rows_by_index ? -1 : (int32_t)psum->numel(), (int32_t)alignment,
                         out.data_ptr<int16_t>(), k64 * ld, nullptr, reinterpret_cast<void*>(stream)));
    out = out.slice(2, 0, mn).transpose(-2, -1);
    return groups > 0 ? out : out.squeeze(0);
}

int operand_kind(const at::Tensor& a, const at::Tensor& b) {
    const auto ta = a.scalar_type(), tb = b.scalar_type();
    if (ta == at::kFloat8_e4m3fn && tb == at::kFloat8_e4m3fn) return kFP8FP8;
    if (ta == at::kFloat8_e4m3fn && tb == at::kChar) return kFP8FP4;
    if (ta == at::kChar && tb == at::kChar) return kFP4FP4;
    if (ta == at::kBFloat16 && tb == at::kBFloat16) return kBF16;
    return -1;
}

// GEMM over K-major operands:
//   gemm_type 0 (dense): a [M, K], b [N, K], d [M, N], c = None or d itself (accumulate);
//   gemm_type 2 / 3 (M-grouped contiguous, psum / m_indices): b [G, N, K], layout int32;
//   gemm_type 4 (masked): a [G, M, K], b [G, N, K], d [G, M, N], layout = masked_m.
// recipes: (gran_a_mn, gran_a_k, gran_b_mn, gran_b_k); num_cus 0 = the device's CUs.
bool gemm(int64_t gemm_type, const at::Tensor& a, const c10::optional<at::Tensor>& sfa_in, const at::Tensor& b,
          const c10::optional<at::Tensor>& sfb_in, const at::Tensor& d, const c10::optional<at::Tensor>& c,
          const c10::optional<at::Tensor>& layout, int64_t gran_a_mn, int64_t gran_a_k, int64_t gran_b_mn,
          int64_t gran_b_k, int64_t num_cus, int64_t alignment, int64_t stream) {
    if (g_gemm == nullptr) return false;
    if (const uint32_t bits = pending_errors()) throw std::runtime_error(error_message(bits));
    const int kind = operand_kind(a, b);
    if (kind < 0) return false;
    const bool bf16 = kind == kBF16;
    const bool grouped = gemm_type == kPsum || gemm_type == kIdx;
    const bool masked = gemm_type == kMasked;
    if (!(gemm_type == kNormal || grouped || masked)) return false;
    const int64_t ra = masked ? 3 : 2, rb = gemm_type == kNormal ? 2 : 3;
    if (a.dim() != ra || b.dim() != rb || d.dim() != ra) return false;
    if (!k_major(a) || !k_major(b) || d.stride(-1) != 1) return false;
    const auto dt = d.scalar_type();
    if (dt != at::kBFloat16 && dt != at::kFloat) return false;
    if (!a.is_cuda() || a.device() != d.device() || b.device() != d.device()) return false;
    const int64_t k = a.size(-1) * (is_fp4(a) ? 2 : 1);
    const int64_t kb = b.size(-1) * (is_fp4(b) ? 2 : 1);
    const int64_t m = a.size(-2), n = b.size(-2);
    if (k != kb || m == 0 || n == 0 || k == 0) return false;
    if (d.size(-2) != m || d.size(-1) != n) return false;
    const int64_t groups = rb == 3 ? b.size(0) : 1;
    if (masked && (a.size(0) != groups || d.size(0) != groups)) return false;
    if (!kernel_ready(a) || !kernel_ready(b)) return false;
    bool accumulate = false;
    if (c.has_value()) {
        const at::Tensor& ct = *c;
        if (gemm_type != kNormal || ct.data_ptr() != d.data_ptr() || ct.sizes() != d.sizes() ||
            ct.strides() != d.strides() || ct.scalar_type() != dt)
            return false;
        accumulate = true;
    }
    const at::Tensor* lay = nullptr;
    if (gemm_type != kNormal) {
        if (!layout.has_value()) return false;
        lay = &*layout;
        if (lay->scalar_type() != at::kInt || !lay->is_contiguous() || lay->device() != d.device()) return false;
        const int64_t want = gemm_type == kIdx ? m : groups;
        if (lay->numel() != want) return false;
    }

    dg_gemm_args args;
    std::memset(&args, 0, sizeof(args));
    at::Tensor sfa_t, sfb_t;
    if (!bf16) {
        if (!sfa_in.has_value() || !sfb_in.has_value()) return false;
        // (validate both before launching either transform)
        const at::Tensor& sfa = *sfa_in;
        const at::Tensor& sfb = *sfb_in;
        if (sfa.device() != d.device() || sfb.device() != d.device()) return false;
        const at::Tensor* rows = grouped ? lay : nullptr;
        sfa_t = kernel_sf(sfa, m, k, gran_a_mn, gran_a_k, masked ? groups : 0, rows, gemm_type == kIdx, alignment,
                          stream);
        if (!sfa_t.defined()) return false;
        sfb_t = kernel_sf(sfb, n, k, gran_b_mn, gran_b_k, rb == 3 ? groups : 0, nullptr, false, alignment, stream);
        if (!sfb_t.defined()) return false;
        args.sfa = static_cast<const int16_t*>(sfa_t.data_ptr());
        args.sfb = static_cast<const int16_t*>(sfb_t.data_ptr());
        args.sfa_ld = sfa_t.stride(-1);
        args.sfb_ld = sfb_t.stride(-1);
        if (masked) args.sfa_batch_stride = sfa_t.stride(0);
        if (rb == 3) args.sfb_batch_stride = sfb_t.stride(0);
    }
    args.kind = kind;
    args.gemm_type = (int32_t)gemm_type;
    args.a = a.data_ptr();
    args.b = b.data_ptr();
    args.d = d.data_ptr();
    args.grouped_layout = lay != nullptr ? lay->data_ptr<int32_t>() : nullptr;
    args.m = (int32_t)m;
    args.n = (int32_t)n;
    args.k = (int32_t)k;
    args.num_groups = (int32_t)groups;
    args.lda = a.stride(-2);
    args.ldb = b.stride(-2);
    args.ldd = d.stride(-2);
    if (masked) {
        args.batch_stride_a = a.stride(0);
        args.batch_stride_d = d.stride(0);
    }
    if (rb == 3) args.batch_stride_b = b.stride(0);
    args.d_dtype = dt == at::kFloat ? DG_DTYPE_F32 : DG_DTYPE_BF16;
    args.accumulate = accumulate ? 1 : 0;
    args.alpha = 1.0f;
    args.alignment = (int32_t)alignment;
    args.num_cus = (int32_t)num_cus;
    args.library_workspace = gemm_type == kNormal ? 1 : 0;
    check_rc(g_gemm(&args, reinterpret_cast<void*>(stream)));
    return true;
}

// ------------------------------------------------------------------------------------------------ operators around the GEMMs
// The same calls as deep_gemm/moe.py, mx.py and loss.py make; an empty result sends the call to their general path, which converts what
// these checks do not take or raises.
decltype(&dg_moe_sort) g_moe_sort = nullptr;
decltype(&dg_moe_sort_workspace_size) g_moe_sort_workspace_size = nullptr;
decltype(&dg_moe_dispatch) g_moe_dispatch = nullptr;
decltype(&dg_moe_combine) g_moe_combine = nullptr;
decltype(&dg_moe_combine_backward) g_moe_combine_backward = nullptr;
decltype(&dg_mx_quantize) g_mx_quantize = nullptr;
decltype(&dg_mx_dequantize) g_mx_dequantize = nullptr;
decltype(&dg_mx_gemm) g_mx_gemm = nullptr;
decltype(&dg_linear_xent_workspace_size) g_xent_workspace_size = nullptr;
decltype(&dg_linear_xent_forward) g_xent_forward = nullptr;
decltype(&dg_linear_xent_backward) g_xent_backward = nullptr;

void init_operators(int64_t sort, int64_t sort_workspace, int64_t dispatch, int64_t combine, int64_t combine_backward,
                    int64_t quantize, int64_t dequantize, int64_t mx_gemm, int64_t xent_workspace, int64_t xent_forward,
                    int64_t xent_backward) {
    g_moe_sort = reinterpret_cast<decltype(g_moe_sort)>(sort);
    g_moe_sort_workspace_size = reinterpret_cast<decltype(g_moe_sort_workspace_size)>(sort_workspace);
    g_moe_dispatch = reinterpret_cast<decltype(g_moe_dispatch)>(dispatch);
    g_moe_combine = reinterpret_cast<decltype(g_moe_combine)>(combine);
    g_moe_combine_backward = reinterpret_cast<decltype(g_moe_combine_backward)>(combine_backward);
    g_mx_quantize = reinterpret_cast<decltype(g_mx_quantize)>(quantize);
    g_mx_dequantize = reinterpret_cast<decltype(g_mx_dequantize)>(dequantize);
    g_mx_gemm = reinterpret_cast<decltype(g_mx_gemm)>(mx_gemm);
    g_xent_workspace_size = reinterpret_cast<decltype(g_xent_workspace_size)>(xent_workspace);
    g_xent_forward = reinterpret_cast<decltype(g_xent_forward)>(xent_forward);
    g_xent_backward = reinterpret_cast<decltype(g_xent_backward)>(xent_backward);
}

using Tensors = std::vector<at::Tensor>;

// (as the library: larger extents go to the general path, which refuses them)
constexpr int64_t kMaxExtent = int64_t(1) << 30;

void raise_pending() {
    if (const uint32_t bits = pending_errors()) throw std::runtime_error(error_message(bits));
}

void* stream_ptr(int64_t stream) { return reinterpret_cast<void*>(stream); }

bool int32_rows(const at::Tensor& t, int64_t dim, const at::Device& device) {
    return t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous() && t.device() == device && t.numel() <= kMaxExtent;
}

// Rows of contiguous values that do not overlap (an expanded row goes to the general path).
bool plain(const at::Tensor& t) {
    return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}

// The layout of a MoELayout's four tensors beside rows on `device`.
bool layout_of(const Tensors& l, const at::Device& device, dg_moe_layout& out) {
    if (l.size() != 4 || !int32_rows(l[0], 2, device) || !int32_rows(l[1], 1, device) || !int32_rows(l[2], 1, device) ||
        !int32_rows(l[3], 1, device) || l[3].numel() != l[1].numel())
        return false;
    out = {(int32_t)l[0].size(0), (int32_t)l[0].size(1), 0, (int32_t)l[1].numel(), 1, l[0].data_ptr<int32_t>(), l[1].data_ptr<int32_t>(),
           l[2].data_ptr<int32_t>(), l[3].data_ptr<int32_t>()};
    return true;
}

// A contiguous piece of `whole` from element `at` on, without the dispatcher and the allocator.
at::Tensor piece(const at::Tensor& whole, int64_t at, at::IntArrayRef sizes) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(whole.storage_offset() + at);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
}

// Scale factors [rows][k64] as they lie in a flat tensor: rows contiguous, `ld` apart.
at::Tensor scale_view(at::Tensor flat, int64_t rows, int64_t k64, int64_t ld) {
    flat.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef{rows, k64}, at::IntArrayRef{1, ld});
    return flat;
}

Tensors moe_sort(const at::Tensor& ids, int64_t groups, int64_t rows, int64_t alignment, int64_t num_cus, int64_t stream) {
    if (g_moe_sort == nullptr || ids.dim() != 2 || !ids.is_cuda() || !ids.is_contiguous() || groups < 1 || groups > 1024 || rows < 0 ||
        rows % alignment != 0 || rows > kMaxExtent || ids.numel() > kMaxExtent ||
        !(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong))
        return {};
    raise_pending();
    const auto options = ids.options().dtype(at::kInt);
    // One allocation for the four, which live and die together (each would cost the host 0.8 us of a latency-bound call); pieces
    // start at 128 bytes.
    const int64_t at_source = align_up(ids.numel(), 32), at_psum = at_source + align_up(rows, 32), at_indices = at_psum + align_up(groups, 32);
    const at::Tensor whole = at::empty({at_indices + rows}, options);
    Tensors l = {piece(whole, 0, ids.sizes()), piece(whole, at_source, {rows}), piece(whole, at_psum, {groups}), piece(whole, at_indices, {rows})};
    dg_moe_layout a;
    if (!layout_of(l, ids.device(), a)) return {};
    a.num_groups = (int32_t)groups;
    a.alignment = (int32_t)alignment;
    int64_t need = 0;
    check_rc(g_moe_sort_workspace_size((int32_t)ids.numel(), (int32_t)groups, &need));
    at::Tensor ws;
    if (need > 0) ws = at::empty({need}, ids.options().dtype(at::kByte));
    check_rc(g_moe_sort(ids.data_ptr(), (int32_t)ids.element_size(), &a, need > 0 ? ws.data_ptr() : nullptr, need, (int32_t)num_cus,
                        stream_ptr(stream)));
    return l;
}

Tensors moe_dispatch(const at::Tensor& x, const c10::optional<at::Tensor>& sf, const Tensors& layout, bool zero_padding, int64_t num_cus,
                     int64_t stream) {
    dg_moe_layout a;
    const int64_t e = x.element_size();
    if (g_moe_dispatch == nullptr || x.dim() != 2 || !x.is_cuda() || !(e == 1 || e == 2 || e == 4) || !layout_of(layout, x.device(), a) ||
        x.size(0) != a.tokens || !plain(x))
        return {};
    int64_t k64 = 0, sf_ld = 0;
    const int64_t out_ld = align_up(a.rows, 2);
    if (sf.has_value()) {
        if (sf->scalar_type() != at::kShort || sf->dim() != 2 || sf->size(0) != a.tokens || sf->device() != x.device() ||
            !(a.tokens <= 1 || sf->stride(0) == 1))
            return {};
        k64 = sf->size(1);
        sf_ld = k64 > 1 ? sf->stride(1) : a.tokens;
    }
    raise_pending();
    Tensors out = {at::empty({a.rows, x.size(1)}, x.options())};
    if (sf.has_value()) out.push_back(at::empty({k64 * out_ld}, sf->options()));
    check_rc(g_moe_dispatch(x.data_ptr(), x.stride(0) * e, x.size(1) * e, &a, out[0].data_ptr(), x.size(1) * e,
                            sf.has_value() ? static_cast<const int16_t*>(sf->data_ptr()) : nullptr, sf_ld, (int32_t)k64,
                            sf.has_value() ? static_cast<int16_t*>(out[1].data_ptr()) : nullptr, out_ld, zero_padding, (int32_t)num_cus,
                            stream_ptr(stream)));
    if (sf.has_value()) out[1] = scale_view(std::move(out[1]), a.rows, k64, out_ld);
    return out;
}

int rows_dtype(const at::Tensor& t) {
    return t.scalar_type() == at::kBFloat16 ? DG_DTYPE_BF16 : t.scalar_type() == at::kFloat ? DG_DTYPE_F32 : -1;
}

bool plain_rows(const at::Tensor& t, int64_t rows) {
    return t.dim() == 2 && t.is_cuda() && rows_dtype(t) >= 0 && t.size(0) == rows && plain(t);
}

bool plain_weights(const at::Tensor& w, const dg_moe_layout& a, const at::Device& device) {
    return w.scalar_type() == at::kFloat && w.dim() == 2 && w.size(0) == a.tokens && w.size(1) == a.topk && w.is_contiguous() &&
           w.device() == device;
}

Tensors moe_combine(const at::Tensor& rows, const Tensors& layout, const c10::optional<at::Tensor>& weights, int64_t num_cus,
                    int64_t stream) {
    dg_moe_layout a;
    if (g_moe_combine == nullptr || !layout_of(layout, rows.device(), a) || !plain_rows(rows, a.rows) ||
        (weights.has_value() && !plain_weights(*weights, a, rows.device())))
        return {};
    raise_pending();
    Tensors out = {at::empty({a.tokens, rows.size(1)}, rows.options())};
    check_rc(g_moe_combine(rows.data_ptr(), rows.stride(0), rows_dtype(rows), rows.size(1), &a,
                           weights.has_value() ? weights->data_ptr<float>() : nullptr, out[0].data_ptr(), rows.size(1), (int32_t)num_cus,
                           stream_ptr(stream)));
    return out;
}

Tensors moe_combine_backward(const at::Tensor& d_out, const at::Tensor& rows, const Tensors& layout, const at::Tensor& weights,
                             int64_t num_cus, int64_t stream) {
    dg_moe_layout a;
    if (g_moe_combine_backward == nullptr || !layout_of(layout, rows.device(), a) || !plain_rows(rows, a.rows) || !plain_rows(d_out, a.tokens) ||
        d_out.scalar_type() != rows.scalar_type() || d_out.size(1) != rows.size(1) || d_out.device() != rows.device() ||
        !plain_weights(weights, a, rows.device()))
        return {};
    raise_pending();
    Tensors out = {at::empty({a.rows, rows.size(1)}, rows.options()), at::empty({a.tokens, a.topk}, weights.options())};
    check_rc(g_moe_combine_backward(d_out.data_ptr(), d_out.stride(0), rows.data_ptr(), rows.stride(0), rows_dtype(rows), rows.size(1), &a,
                                    weights.data_ptr<float>(), out[0].data_ptr(), rows.size(1), out[1].data_ptr<float>(), (int32_t)num_cus,
                                    stream_ptr(stream)));
    return out;
}

// A two-dimensional x [M, K] to codes and scale factors.
Tensors mx_quantize(const at::Tensor& x, bool fp4, int64_t num_cus, int64_t stream) {
    if (g_mx_quantize == nullptr || x.dim() != 2 || !x.is_cuda() || rows_dtype(x) < 0 || x.size(1) % 32 != 0 || x.numel() == 0 ||
        !plain(x) || x.size(0) > kMaxExtent || x.size(1) > kMaxExtent)
        return {};
    raise_pending();
    const int64_t m = x.size(0), k = x.size(1), ld = align_up(m, 2), k64 = ceil_div(k, 64);
    Tensors out = {at::empty({m, fp4 ? k / 2 : k}, x.options().dtype(fp4 ? at::kChar : at::kFloat8_e4m3fn)),
                   at::empty({k64 * ld}, x.options().dtype(at::kShort))};
    dg_mx_args a = {};
    a.format = fp4 ? DG_MX_E2M1 : DG_MX_E4M3;
    a.x_dtype = rows_dtype(x);
    a.batches = 1;
    a.rows = (int32_t)m;
    a.k = (int32_t)k;
    a.x = x.data_ptr();
    a.x_ld = m > 1 ? x.stride(0) : k;
    a.codes = out[0].data_ptr();
    a.codes_ld = out[0].stride(0);
    a.sf = static_cast<int16_t*>(out[1].data_ptr());
    a.sf_ld = ld;
    a.num_cus = (int32_t)num_cus;
    check_rc(g_mx_quantize(&a, stream_ptr(stream)));
    out[1] = scale_view(std::move(out[1]), m, k64, ld);
    return out;
}

Tensors mx_dequantize(const at::Tensor& codes, const at::Tensor& sf, bool f32, int64_t num_cus, int64_t stream) {
    const bool fp4 = codes.scalar_type() == at::kChar;
    if (g_mx_dequantize == nullptr || codes.dim() != 2 || !codes.is_cuda() || !(fp4 || codes.scalar_type() == at::kFloat8_e4m3fn) ||
        codes.numel() == 0 || !plain(codes) || codes.stride(0) % 8 || (reinterpret_cast<uintptr_t>(codes.data_ptr()) & 7))
        return {};
    const int64_t m = codes.size(0), k = codes.size(1) * (fp4 ? 2 : 1), k64 = ceil_div(k, 64);
    if (k % 32 != 0 || m > kMaxExtent || k > kMaxExtent || sf.scalar_type() != at::kShort || sf.dim() != 2 ||
        sf.size(0) != m || sf.size(1) != k64 || sf.device() != codes.device() || !(m <= 1 || sf.stride(0) == 1) ||
        (reinterpret_cast<uintptr_t>(sf.data_ptr()) & 3) || (k64 > 1 && (sf.stride(1) % 2 || sf.stride(1) < m)))
        return {};
    raise_pending();
    Tensors out = {at::empty({m, k}, codes.options().dtype(f32 ? at::kFloat : at::kBFloat16))};
    dg_mx_args a = {};
    a.format = fp4 ? DG_MX_E2M1 : DG_MX_E4M3;
    a.x_dtype = f32 ? DG_DTYPE_F32 : DG_DTYPE_BF16;
    a.batches = 1;
    a.rows = (int32_t)m;
    a.k = (int32_t)k;
    a.x = out[0].data_ptr();
    a.x_ld = k;
    a.codes = codes.data_ptr();
    a.codes_ld = m > 1 ? codes.stride(0) : codes.size(1);
    a.sf = static_cast<int16_t*>(sf.data_ptr());
    a.sf_ld = k64 > 1 ? sf.stride(1) : align_up(m, 2);
    a.num_cus = (int32_t)num_cus;
    check_rc(g_mx_dequantize(&a, stream_ptr(stream)));
    return out;
}

// D (+)= quantised(x) w^T: a few rows to e2m1 in one launch, otherwise quantised first.  false: the general path.
// cus: what the GEMMs take (set_num_sms, 0 = all); num_cus: the cap, 0 = none.
bool mx_gemm(const at::Tensor& x, const at::Tensor& w, const at::Tensor& sfw, const at::Tensor& d, const c10::optional<at::Tensor>& c,
             bool fp4, int64_t cus, int64_t num_cus, int64_t alignment, int64_t stream) {
    if (g_mx_gemm == nullptr || x.dim() != 2 || w.dim() != 2 || d.dim() != 2 || sfw.dim() != 2 || !x.is_cuda() || rows_dtype(x) < 0 ||
        rows_dtype(d) < 0 || w.scalar_type() != at::kChar || sfw.scalar_type() != at::kShort || w.device() != x.device() ||
        sfw.device() != x.device() || d.device() != x.device())
        return false;
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0), k64 = ceil_div(k, 64);
    if (m > 16 || m * k > 32768 || !fp4) {   // (what dg_mx_gemm takes)
        const Tensors q = mx_quantize(x, fp4, num_cus, stream);
        return !q.empty() && gemm(kNormal, q[0], q[1], w, sfw, d, c, c10::nullopt, 1, 32, 1, 32, cus, alignment, stream);
    }
    if (m == 0 || n == 0 || k == 0 || k % 32 != 0 || k > kMaxExtent || n > kMaxExtent || w.size(1) * 2 != k ||
        sfw.size(0) != n || sfw.size(1) != k64 || d.size(0) != m || d.size(1) != n || x.stride(1) != 1 || w.stride(1) != 1 ||
        d.stride(1) != 1 || !(n <= 1 || sfw.stride(0) == 1))
        return false;
    const int64_t sf_ld = k64 > 1 ? sfw.stride(1) : align_up(n, 2), e = x.element_size();
    if (sf_ld % 2 != 0 || sf_ld < n || (reinterpret_cast<uintptr_t>(sfw.data_ptr()) & 3) || (reinterpret_cast<uintptr_t>(x.data_ptr()) & 3) ||
        (reinterpret_cast<uintptr_t>(w.data_ptr()) & 3) || (m > 1 && (x.stride(0) < k || (x.stride(0) * e) % 4 || d.stride(0) < n)) ||
        (n > 1 && (w.stride(0) < k / 2 || w.stride(0) % 4)))
        return false;
    if (c.has_value() && (c->data_ptr() != d.data_ptr() || c->sizes() != d.sizes() || c->strides() != d.strides() ||
                          c->scalar_type() != d.scalar_type()))
        return false;
    raise_pending();
    check_rc(g_mx_gemm(x.data_ptr(), rows_dtype(x), m > 1 ? x.stride(0) : k, w.data_ptr(), n > 1 ? w.stride(0) : k / 2,
                       static_cast<const int16_t*>(sfw.data_ptr()), sf_ld, d.data_ptr(), rows_dtype(d), m > 1 ? d.stride(0) : n,
                       (int32_t)m, (int32_t)n, (int32_t)k, c.has_value(), (int32_t)num_cus, stream_ptr(stream)));
    return true;
}

bool xent_rows(const at::Tensor& t, const at::Device& device) {
    return t.dim() == 2 && t.scalar_type() == at::kBFloat16 && t.is_cuda() && t.device() == device && t.stride(1) == 1 &&
           t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

bool xent_vector(const at::Tensor& t, int64_t tokens, const at::Device& device) {
    return t.dim() == 1 && t.size(0) == tokens && t.is_contiguous() && t.device() == device;
}

// Arguments of a cross entropy of x [T, H], w [V, H] and their targets; false: the general path.
bool xent_args(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target, int64_t ignore, int64_t num_cus, dg_linear_xent_args& a) {
    if (g_xent_forward == nullptr || !xent_rows(x, x.device()) || !xent_rows(w, x.device()) || x.size(1) != w.size(1) || x.size(1) == 0 ||
        x.size(1) % 8 != 0 || x.size(0) == 0 || x.size(0) > (1 << 20) || w.size(0) == 0 || w.size(0) > kMaxExtent ||
        !xent_vector(target, x.size(0), x.device()) || !(target.scalar_type() == at::kInt || target.scalar_type() == at::kLong))
        return false;
    a = {};
    a.tokens = (int32_t)x.size(0);
    a.width = (int32_t)x.size(1);
    a.vocab = (int32_t)w.size(0);
    a.x = x.data_ptr();
    a.w = w.data_ptr();
    a.x_ld = x.stride(0);
    a.w_ld = w.stride(0);
    a.target = target.data_ptr();
    a.target_bytes = (int32_t)target.element_size();
    a.ignore_index = ignore;
    a.num_cus = (int32_t)num_cus;
    return true;
}

void xent_run(decltype(g_xent_forward) fn, dg_linear_xent_args& a, int32_t backward, const at::Tensor& x, int64_t stream) {
    int64_t need = 0;
    check_rc(g_xent_workspace_size(&a, backward, &need));
    const at::Tensor ws = at::empty({need}, x.options().dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = need;
    check_rc(fn(&a, stream_ptr(stream)));
}

Tensors linear_xent(const at::Tensor& x, const at::Tensor& w, const at::Tensor& target, int64_t ignore, int64_t num_cus, int64_t stream) {
    dg_linear_xent_args a;
    if (!xent_args(x, w, target, ignore, num_cus, a)) return {};
    raise_pending();
    Tensors out = {at::empty({x.size(0)}, x.options().dtype(at::kFloat)), at::empty({x.size(0)}, x.options().dtype(at::kFloat))};
    a.loss = out[0].data_ptr<float>();
    a.lse = out[1].data_ptr<float>();
    xent_run(g_xent_forward, a, 0, x, stream);
    return out;
}

Tensors linear_xent_backward(const at::Tensor& d_loss, const at::Tensor& x, const at::Tensor& w, const at::Tensor& target,
                             const at::Tensor& lse, int64_t ignore, int64_t num_cus, int64_t stream) {
    dg_linear_xent_args a;
    if (!xent_args(x, w, target, ignore, num_cus, a) || d_loss.scalar_type() != at::kFloat || lse.scalar_type() != at::kFloat ||
        !xent_vector(d_loss, x.size(0), x.device()) || !xent_vector(lse, x.size(0), x.device()))
        return {};
    raise_pending();
    Tensors out = {at::empty(x.sizes(), x.options()), at::empty(w.sizes(), w.options())};
    a.lse = lse.data_ptr<float>();
    a.d_loss = d_loss.data_ptr<float>();
    a.d_x = out[0].data_ptr();
    a.d_w = out[1].data_ptr();
    a.d_x_ld = a.d_w_ld = a.width;
    xent_run(g_xent_backward, a, 1, x, stream);
    return out;
}

// ------------------------------------------------------------------------------------------------ what stands between the products
// The same calls as deep_gemm/moe.py (routing), norm.py, activation.py and lora.py make.
decltype(&dg_moe_route) g_route = nullptr;
decltype(&dg_moe_route_backward) g_route_backward = nullptr;
decltype(&dg_rms_norm_workspace_size) g_norm_workspace_size = nullptr;
decltype(&dg_rms_norm_forward) g_norm = nullptr;
decltype(&dg_rms_norm_backward) g_norm_backward = nullptr;
decltype(&dg_swiglu_forward) g_swiglu = nullptr;
decltype(&dg_swiglu_backward) g_swiglu_backward = nullptr;
decltype(&dg_lora_workspace_size) g_lora_workspace_size = nullptr;
decltype(&dg_lora_gemm) g_lora = nullptr;

void init_blocks(int64_t route, int64_t route_backward, int64_t norm_workspace, int64_t norm, int64_t norm_backward, int64_t swiglu,
                 int64_t swiglu_backward, int64_t lora_workspace, int64_t lora) {
    g_route = reinterpret_cast<decltype(g_route)>(route);
    g_route_backward = reinterpret_cast<decltype(g_route_backward)>(route_backward);
    g_norm_workspace_size = reinterpret_cast<decltype(g_norm_workspace_size)>(norm_workspace);
    g_norm = reinterpret_cast<decltype(g_norm)>(norm);
    g_norm_backward = reinterpret_cast<decltype(g_norm_backward)>(norm_backward);
    g_swiglu = reinterpret_cast<decltype(g_swiglu)>(swiglu);
    g_swiglu_backward = reinterpret_cast<decltype(g_swiglu_backward)>(swiglu_backward);
    g_lora_workspace_size = reinterpret_cast<decltype(g_lora_workspace_size)>(lora_workspace);
    g_lora = reinterpret_cast<decltype(g_lora)>(lora);
}

// A plain matrix of `rows` x `cols` bf16 or fp32 values on `device` (negative sizes: any).
bool matrix(const at::Tensor& t, int64_t rows, int64_t cols, const at::Device& device) {
    return t.dim() == 2 && t.is_cuda() && t.device() == device && rows_dtype(t) >= 0 && (rows < 0 || t.size(0) == rows) &&
           (cols < 0 || t.size(1) == cols) && plain(t) && t.size(0) <= kMaxExtent && t.size(1) <= kMaxExtent;
}

// A contiguous tensor of `dtype` on `device`.
bool dense(const at::Tensor& t, at::ScalarType dtype, at::IntArrayRef sizes, const at::Device& device) {
    return t.scalar_type() == dtype && t.sizes() == sizes && t.is_contiguous() && t.device() == device;
}

int64_t row_ld(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Codes of `rows` x `k` values and their scale factors, to be written.
struct Codes {
    at::Tensor codes, sf;
    int64_t ld;
};
Codes new_codes(const at::Tensor& like, bool fp4, int64_t rows, int64_t k) {
    const int64_t ld = align_up(rows, 2);
    return {at::empty({rows, fp4 ? k / 2 : k}, like.options().dtype(fp4 ? at::kChar : at::kFloat8_e4m3fn)),
            at::empty({ceil_div(k, 64) * ld}, like.options().dtype(at::kShort)), ld};
}

bool route_args(const at::Tensor& logits, int64_t topk, bool sigmoid, bool renormalize, double scale, int64_t num_cus, dg_moe_route_args& a) {
    if (g_route == nullptr || !logits.is_cuda() || !matrix(logits, -1, -1, logits.device()) || logits.numel() == 0 || logits.size(1) > 1024 || topk < 1 ||
        topk > 16 || topk > logits.size(1))
        return false;
    a = {};
    a.tokens = (int32_t)logits.size(0);
    a.experts = (int32_t)logits.size(1);
    a.topk = (int32_t)topk;
    a.scores = sigmoid ? DG_SCORES_SIGMOID : DG_SCORES_SOFTMAX;
    a.renormalize = renormalize;
    a.scale = (float)scale;
    a.dtype = rows_dtype(logits);
    a.logits = logits.data_ptr();
    a.logits_ld = row_ld(logits);
    a.num_cus = (int32_t)num_cus;
    return true;
}

Tensors moe_route(const at::Tensor& logits, int64_t topk, bool sigmoid, const c10::optional<at::Tensor>& bias, int64_t num_groups, int64_t topk_groups,
                  int64_t group_top, bool renormalize, double scale, int64_t num_cus, int64_t stream) {
    dg_moe_route_args a;
    if (!route_args(logits, topk, sigmoid, renormalize, scale, num_cus, a) || num_groups < 1 || logits.size(1) % num_groups != 0 || topk_groups < 1 ||
        topk_groups > num_groups || topk > topk_groups * (logits.size(1) / num_groups) || group_top < 1 || group_top > 2 ||
        (bias.has_value() && !dense(*bias, at::kFloat, {logits.size(1)}, logits.device())))
        return {};
    raise_pending();
    const c10::DeviceGuard guard(logits.device());
    Tensors out = {at::empty({logits.size(0), topk}, logits.options().dtype(at::kInt)), at::empty({logits.size(0), topk}, logits.options().dtype(at::kFloat))};
    a.num_groups = (int32_t)num_groups;
    a.topk_groups = (int32_t)topk_groups;
    a.group_top = (int32_t)group_top;
    a.bias = bias.has_value() ? bias->data_ptr<float>() : nullptr;
    a.ids = out[0].data_ptr<int32_t>();
    a.weights = out[1].data_ptr<float>();
    check_rc(g_route(&a, stream_ptr(stream)));
    return out;
}

Tensors moe_route_backward(const at::Tensor& d_weights, const at::Tensor& logits, const at::Tensor& ids, bool sigmoid, bool renormalize, double scale,
                           int64_t num_cus, int64_t stream) {
    dg_moe_route_args a;
    if (ids.dim() != 2 || !route_args(logits, ids.size(1), sigmoid, renormalize, scale, num_cus, a) ||
        !dense(ids, at::kInt, {logits.size(0), ids.size(1)}, logits.device()) || !dense(d_weights, at::kFloat, ids.sizes(), logits.device()))
        return {};
    raise_pending();
    const c10::DeviceGuard guard(logits.device());
    Tensors out = {at::empty(logits.sizes(), logits.options())};
    a.ids = ids.data_ptr<int32_t>();
    a.d_weights = d_weights.data_ptr<float>();
    a.d_logits = out[0].data_ptr();
    a.d_logits_ld = logits.size(1);
    check_rc(g_route_backward(&a, stream_ptr(stream)));
    return out;
}

bool norm_args(const at::Tensor& x, const at::Tensor& weight, double eps, int64_t num_cus, dg_rms_norm_args& a) {
    if (g_norm == nullptr || !x.is_cuda() || !matrix(x, -1, -1, x.device()) || x.numel() == 0 || x.size(1) > 32768 || rows_dtype(weight) < 0 ||
        !dense(weight, weight.scalar_type(), {x.size(1)}, x.device()))
        return false;
    a = {};
    a.tokens = (int32_t)x.size(0);
    a.width = (int32_t)x.size(1);
    a.dtype = rows_dtype(x);
    a.weight_dtype = rows_dtype(weight);
    a.eps = (float)eps;
    a.format = -1;
    a.weight = weight.data_ptr();
    a.num_cus = (int32_t)num_cus;
    return true;
}

// y (or codes and scale factors), rstd and, with a residual, h.  format: -1 values, DG_MX_*.
Tensors rms_norm(const at::Tensor& x, const at::Tensor& weight, const c10::optional<at::Tensor>& residual, double eps, int64_t format, int64_t num_cus,
                 int64_t stream) {
    dg_rms_norm_args a;
    if (!norm_args(x, weight, eps, num_cus, a) || (format != -1 && x.size(1) % 32 != 0) ||
        (residual.has_value() && (!matrix(*residual, x.size(0), x.size(1), x.device()) || residual->scalar_type() != x.scalar_type())))
        return {};
    raise_pending();
    const c10::DeviceGuard guard(x.device());
    a.x = x.data_ptr();
    a.x_ld = row_ld(x);
    Tensors out;
    int64_t ld = 0;
    if (format == -1) {
        out.push_back(at::empty(x.sizes(), x.options()));
        a.y_ld = x.size(1);
    } else {
        Codes c = new_codes(x, format == DG_MX_E2M1, x.size(0), x.size(1));
        a.format = (int32_t)format;
        a.y_ld = c.codes.size(1);
        a.sf = static_cast<int16_t*>(c.sf.data_ptr());
        a.sf_ld = ld = c.ld;
        out = {std::move(c.codes), std::move(c.sf)};
    }
    a.y = out[0].data_ptr();
    out.push_back(at::empty({x.size(0)}, x.options().dtype(at::kFloat)));
    a.rstd = out.back().data_ptr<float>();
    if (residual.has_value()) {
        out.push_back(at::empty(x.sizes(), x.options()));
        a.residual = residual->data_ptr();
        a.residual_ld = row_ld(*residual);
        a.h = out.back().data_ptr();
        a.h_ld = x.size(1);
    }
    check_rc(g_norm(&a, stream_ptr(stream)));
    if (format != -1) out[1] = scale_view(std::move(out[1]), x.size(0), ceil_div(x.size(1), 64), ld);
    return out;
}

Tensors rms_norm_backward(const at::Tensor& d_y, const at::Tensor& h, const at::Tensor& weight, const at::Tensor& rstd,
                          const c10::optional<at::Tensor>& d_h, int64_t num_cus, int64_t stream) {
    dg_rms_norm_args a;
    if (!norm_args(h, weight, 0, num_cus, a) || !matrix(d_y, h.size(0), h.size(1), h.device()) || d_y.scalar_type() != h.scalar_type() ||
        !dense(rstd, at::kFloat, {h.size(0)}, h.device()) ||
        (d_h.has_value() && (!matrix(*d_h, h.size(0), h.size(1), h.device()) || d_h->scalar_type() != h.scalar_type())))
        return {};
    raise_pending();
    const c10::DeviceGuard guard(h.device());
    int64_t need = 0;
    check_rc(g_norm_workspace_size(&a, &need));
    Tensors out = {at::empty(h.sizes(), h.options()), at::empty({h.size(1)}, rstd.options())};
    const at::Tensor ws = at::empty({need}, h.options().dtype(at::kByte));
    a.h = h.data_ptr();
    a.h_ld = row_ld(h);
    a.rstd = rstd.data_ptr<float>();
    a.d_y = d_y.data_ptr();
    a.d_y_ld = row_ld(d_y);
    if (d_h.has_value()) {
        a.d_h = d_h->data_ptr();
        a.d_h_ld = row_ld(*d_h);
    }
    a.d_x = out[0].data_ptr();
    a.d_x_ld = h.size(1);
    a.d_weight = out[1].data_ptr<float>();
    a.workspace = ws.data_ptr();
    a.workspace_bytes = need;
    check_rc(g_norm_backward(&a, stream_ptr(stream)));
    return out;
}

bool gate_args(int64_t rows, int64_t width, const at::Tensor& values, const c10::optional<at::Tensor>& m_indices, bool zero_padding, int64_t num_cus,
               dg_swiglu_args& a) {
    if (g_swiglu == nullptr || rows == 0 || width == 0 || (m_indices.has_value() && !dense(*m_indices, at::kInt, {rows}, values.device()))) return false;
    a = {};
    a.rows = (int32_t)rows;
    a.width = (int32_t)width;
    a.dtype = rows_dtype(values);
    a.format = -1;
    a.m_indices = m_indices.has_value() ? m_indices->data_ptr<int32_t>() : nullptr;
    a.zero_padding = zero_padding;
    a.num_cus = (int32_t)num_cus;
    return true;
}

// act (or codes and scale factors) and, with `checkpoint`, h's codes and scale factors.
Tensors swiglu(const at::Tensor& h, int64_t format, bool checkpoint, const c10::optional<at::Tensor>& m_indices, bool zero_padding, int64_t num_cus,
               int64_t stream) {
    dg_swiglu_args a;
    if (!h.is_cuda() || !matrix(h, -1, -1, h.device()) || h.size(1) % 2 != 0) return {};
    const int64_t rows = h.size(0), f = h.size(1) / 2;
    if (!gate_args(rows, f, h, m_indices, zero_padding, num_cus, a) || ((format != -1 || checkpoint) && f % 32 != 0)) return {};
    raise_pending();
    const c10::DeviceGuard guard(h.device());
    a.h = h.data_ptr();
    a.h_ld = row_ld(h);
    Tensors out;
    if (format == -1) {
        out.push_back(at::empty({rows, f}, h.options()));
        a.act_ld = f;
    } else {
        Codes c = new_codes(h, format == DG_MX_E2M1, rows, f);
        a.format = (int32_t)format;
        a.act_ld = c.codes.size(1);
        a.act_sf = static_cast<int16_t*>(c.sf.data_ptr());
        a.act_sf_ld = c.ld;
        out = {std::move(c.codes), std::move(c.sf)};
    }
    a.act = out[0].data_ptr();
    if (checkpoint) {
        Codes c = new_codes(h, false, rows, 2 * f);
        a.saved = c.codes.data_ptr();
        a.saved_ld = 2 * f;
        a.saved_sf = static_cast<int16_t*>(c.sf.data_ptr());
        a.saved_sf_ld = c.ld;
        out.push_back(std::move(c.codes));
        out.push_back(std::move(c.sf));
    }
    check_rc(g_swiglu(&a, stream_ptr(stream)));
    const int64_t ld = align_up(rows, 2);
    if (format != -1) out[1] = scale_view(std::move(out[1]), rows, ceil_div(f, 64), ld);
    if (checkpoint) out.back() = scale_view(std::move(out.back()), rows, f / 32, ld);
    return out;
}

Tensors swiglu_backward(const at::Tensor& d_act, const at::Tensor& saved, const c10::optional<at::Tensor>& sf, bool with_act,
                        const c10::optional<at::Tensor>& m_indices, bool zero_padding, int64_t num_cus, int64_t stream) {
    dg_swiglu_args a;
    if (!d_act.is_cuda() || !matrix(d_act, -1, -1, d_act.device())) return {};
    const int64_t rows = d_act.size(0), f = d_act.size(1);
    if (!gate_args(rows, f, d_act, m_indices, zero_padding, num_cus, a)) return {};
    if (sf.has_value()) {
        if (f % 32 != 0 || saved.scalar_type() != at::kFloat8_e4m3fn || saved.dim() != 2 || saved.size(0) != rows || saved.size(1) != 2 * f ||
            saved.device() != d_act.device() || !plain(saved) || row_ld(saved) % 8 != 0 || (reinterpret_cast<uintptr_t>(saved.data_ptr()) & 7) != 0)
            return {};
        const int64_t k64 = f / 32, ld = k64 > 1 ? sf->stride(1) : align_up(rows, 2);
        if (sf->scalar_type() != at::kShort || sf->dim() != 2 || sf->size(0) != rows || sf->size(1) != k64 || sf->device() != d_act.device() ||
            !(rows <= 1 || sf->stride(0) == 1) || ld % 2 != 0 || ld < rows || (reinterpret_cast<uintptr_t>(sf->data_ptr()) & 3) != 0)
            return {};
        a.saved = saved.data_ptr();
        a.saved_ld = row_ld(saved);
        a.saved_sf = static_cast<int16_t*>(sf->data_ptr());
        a.saved_sf_ld = ld;
    } else {
        if (!matrix(saved, rows, 2 * f, d_act.device()) || saved.scalar_type() != d_act.scalar_type()) return {};
        a.h = saved.data_ptr();
        a.h_ld = row_ld(saved);
    }
    raise_pending();
    const c10::DeviceGuard guard(d_act.device());
    Tensors out = {at::empty({rows, 2 * f}, d_act.options())};
    a.d_act = d_act.data_ptr();
    a.d_act_ld = row_ld(d_act);
    a.d_h = out[0].data_ptr();
    a.d_h_ld = 2 * f;
    if (with_act) {
        out.push_back(at::empty({rows, f}, d_act.options()));
        a.act = out[1].data_ptr();
        a.act_ld = f;
    }
    check_rc(g_swiglu_backward(&a, stream_ptr(stream)));
    return out;
}

bool aligned_rows(const at::Tensor& t) {
    if (t.scalar_type() != at::kBFloat16 || t.stride(-1) != 1 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) != 0) return false;
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) % 8 != 0) return false;
    return t.size(-2) <= 1 || t.stride(-2) >= t.size(-1);
}

// false: the general path
bool lora_gemm(const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const at::Tensor& d, const Tensors& layout,
               const c10::optional<at::Tensor>& scales, const c10::optional<at::Tensor>& c, int64_t num_cus, int64_t stream) {
    dg_moe_layout l;
    if (g_lora == nullptr || !x.is_cuda() || x.dim() != 2 || a.dim() != 3 || b.dim() != 3 || x.numel() == 0 || a.numel() == 0 || b.numel() == 0 ||
        !layout_of(layout, x.device(), l) || l.tokens != x.size(0) || l.topk != 1 || l.rows % 32 != 0 || !aligned_rows(x) || !aligned_rows(a) ||
        !aligned_rows(b) || a.device() != x.device() || b.device() != x.device() || a.size(0) != b.size(0) || a.size(2) != x.size(1) ||
        b.size(2) != a.size(1) || a.size(1) % 8 != 0 || a.size(1) > 256 || x.size(1) % 8 != 0 || x.size(0) > kMaxExtent || x.size(1) > kMaxExtent ||
        a.size(0) > kMaxExtent || b.size(1) > kMaxExtent || !matrix(d, x.size(0), b.size(1), x.device()) ||
        (scales.has_value() && !dense(*scales, at::kFloat, {a.size(0)}, x.device())) ||
        (c.has_value() && (!matrix(*c, x.size(0), b.size(1), x.device()) || c->scalar_type() != d.scalar_type() ||
                           (c->data_ptr() == d.data_ptr() && row_ld(*c) != row_ld(d)))))
        return false;
    raise_pending();
    const c10::DeviceGuard guard(x.device());
    l.alignment = 32;   // (every alignment that can be set is a multiple of it)
    dg_lora_args p = {};
    p.tokens = (int32_t)x.size(0);
    p.adapters = (int32_t)a.size(0);
    p.rank = (int32_t)a.size(1);
    p.n = (int32_t)b.size(1);
    p.k = (int32_t)x.size(1);
    p.x = x.data_ptr();
    p.a = a.data_ptr();
    p.b = b.data_ptr();
    p.x_ld = row_ld(x);
    p.a_ld = a.size(1) > 1 ? a.stride(1) : p.k;
    p.a_stride = a.size(0) > 1 ? a.stride(0) : 0;
    p.b_ld = b.size(1) > 1 ? b.stride(1) : p.rank;
    p.b_stride = b.size(0) > 1 ? b.stride(0) : 0;
    p.scales = scales.has_value() ? scales->data_ptr<float>() : nullptr;
    p.c = c.has_value() ? c->data_ptr() : nullptr;
    p.c_ld = c.has_value() ? row_ld(*c) : 0;
    p.d = d.data_ptr();
    p.d_ld = row_ld(d);
    p.d_dtype = rows_dtype(d);
    p.layout = &l;
    p.num_cus = (int32_t)num_cus;
    int64_t need = 0;
    check_rc(g_lora_workspace_size(&p, &need));
    const at::Tensor ws = at::empty({need}, x.options().dtype(at::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = need;
    check_rc(g_lora(&p, stream_ptr(stream)));
    return true;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "deep_gemm C++ host path (validation, scale-factor pass-through and launch)";
    m.def("init", &init, "hand over the library's entry points");
    m.def("init_operators", &init_operators, "hand over the entry points of the operators around the GEMMs");
    m.def("moe_sort", &moe_sort, "slots, source, psum and m_indices; empty (here and below): the general path must handle the call");
    m.def("moe_dispatch", &moe_dispatch, "rows (and their scale factors) from tokens");
    m.def("moe_combine", &moe_combine, "weighted sums of the tokens' rows");
    m.def("moe_combine_backward", &moe_combine_backward, "gradients of rows and weights");
    m.def("mx_quantize", &mx_quantize, "codes and scale factors of a matrix");
    m.def("mx_dequantize", &mx_dequantize, "values of codes and scale factors");
    m.def("mx_gemm", &mx_gemm, "product of rows quantised on the way; false: the general path must handle the call");
    m.def("linear_xent", &linear_xent, "loss and log sums of a linear cross entropy");
    m.def("linear_xent_backward", &linear_xent_backward, "gradients of x and the weight");
    m.def("init_blocks", &init_blocks, "hand over the entry points of what stands between the products");
    m.def("moe_route", &moe_route, "experts and weights of the tokens");
    m.def("moe_route_backward", &moe_route_backward, "gradient of the logits");
    m.def("rms_norm", &rms_norm, "normalised rows (or codes and scale factors), rstd and the sum with the residual");
    m.def("rms_norm_backward", &rms_norm_backward, "gradients of the rows and the weight");
    m.def("swiglu", &swiglu, "gated activation (or codes and scale factors) and the input's 8-bit checkpoint");
    m.def("swiglu_backward", &swiglu_backward, "gradient of the gated activation's input, and the activation again");
    m.def("lora_gemm", &lora_gemm, "adapters of many requests; false: the general path must handle the call");
    m.def("gemm", &gemm, "validate and launch one GEMM; false: the general path must handle the call");
}
