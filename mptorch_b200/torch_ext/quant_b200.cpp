// PyTorch C++ extension `quant_b200`: the reference's `quant_cuda` pybind11 module re-expressed over the
// C ABI of libmptorch_b200.so.  Same function names, argument order and tensor checks as the
// registrations in the reference's mptorch/quant/quant_cuda/pybind_cuda.cpp (lines cited per function),
// so `quant_function.py` can use this module in place of `quant_cuda`.  The extension holds no kernels:
// it checks tensors, selects the device and the current stream, allocates outputs and a small GEMM
// workspace through the caching allocator, and forwards.
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <array>
#include <optional>
#include <vector>

#include "mptorch_b200.h"

namespace {

#define CHECK_CUDA(x) TORCH_CHECK(x.is_cuda(), #x " must be a CUDA tensor")
#define CHECK_CONTIGUOUS(x) TORCH_CHECK(x.is_contiguous(), #x " must be contiguous")
#define CHECK_INPUT(x) \
    CHECK_CUDA(x);     \
    CHECK_CONTIGUOUS(x); \
    TORCH_CHECK(x.scalar_type() == at::kFloat, #x " must be float32")

void check(int rc) { TORCH_CHECK(rc == MPT_OK, mpt_last_error()); }
void* stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int g_accum_order = MPT_ORDER_CUDA, g_reduce_order = MPT_ORDER_CUDA;

struct Geom { int64_t outer; int channel; int64_t inner; };

// reference: quant_cuda/quant.cu:678-726 (partition_tensor for one dim and for a list of trailing dims)
Geom partition(const at::Tensor& t, const std::vector<int>& dims) {
    const int nd = (int)t.dim();
    std::vector<int> real;
    for (int d : dims) real.push_back((nd + (d % nd)) % nd);
    Geom g{1, 1, 1};
    for (int d : real) g.channel *= (int)t.size(d);
    for (int i = 0; i < real.back(); ++i) g.outer *= t.size(i);
    for (int i = real.front() + 1; i < nd; ++i) g.inner *= t.size(i);
    return g;
}

at::Tensor float_quantize_nearest(at::Tensor a, int man_bits, int exp_bits, bool subnormals, bool saturate) {   // :44
    CHECK_INPUT(a);
    c10::cuda::CUDAGuard guard(a.device());
    auto o = at::empty_like(a);
    check(mpt_float_quantize_nearest(a.data_ptr<float>(), o.data_ptr<float>(), a.numel(), man_bits, exp_bits, subnormals, saturate, stream()));
    return o;
}

at::Tensor float_quantize_stochastic(at::Tensor a, int man_bits, int exp_bits, int prng_bits, bool subnormals, bool saturate) {   // :98
    CHECK_INPUT(a);
    c10::cuda::CUDAGuard guard(a.device());
    auto o = at::empty_like(a);
    auto r = at::randint_like(a, INT_MAX, a.options().dtype(at::kInt));   // the reference's draw (quant.cu:132)
    check(mpt_float_quantize_stochastic(a.data_ptr<float>(), r.data_ptr<int>(), o.data_ptr<float>(), a.numel(), man_bits, exp_bits, prng_bits,
                                        subnormals, saturate, stream()));
    return o;
}

at::Tensor float_quantize_truncate(at::Tensor a, int man_bits, int exp_bits, bool subnormals, bool saturate) {   // new
    CHECK_INPUT(a);
    c10::cuda::CUDAGuard guard(a.device());
    auto o = at::empty_like(a);
    check(mpt_float_quantize_truncate(a.data_ptr<float>(), o.data_ptr<float>(), a.numel(), man_bits, exp_bits, subnormals, saturate, stream()));
    return o;
}

at::Tensor binary8(at::Tensor a, int P, int prng_bits, bool is_signed, int policy, bool subnormals, int rounding) {
    CHECK_INPUT(a);
    c10::cuda::CUDAGuard guard(a.device());
    auto o = at::empty_like(a);
    at::Tensor r;
    const int* rp = nullptr;
    if (rounding == MPT_RND_STOCHASTIC) {
        r = at::randint_like(a, INT_MAX, a.options().dtype(at::kInt));    // quant.cu:202
        rp = r.data_ptr<int>();
    }
    check(mpt_binary8_quantize(a.data_ptr<float>(), rp, o.data_ptr<float>(), a.numel(), P, is_signed, policy, subnormals, rounding, prng_bits, stream()));
    return o;
}
at::Tensor binary8_quantize_nearest(at::Tensor a, int P, bool is_signed, int policy, bool subnormals) {   // :61
    return binary8(a, P, 0, is_signed, policy, subnormals, MPT_RND_NEAREST);
}
at::Tensor binary8_quantize_stochastic(at::Tensor a, int P, int prng_bits, bool is_signed, int policy, bool subnormals) {   // :107
    return binary8(a, P, prng_bits, is_signed, policy, subnormals, MPT_RND_STOCHASTIC);
}
at::Tensor binary8_quantize_truncate(at::Tensor a, int P, bool is_signed, int policy, bool subnormals) {   // :115
    return binary8(a, P, 0, is_signed, policy, subnormals, MPT_RND_TRUNCATE);
}

at::Tensor superfp_quantize_nearest(at::Tensor a, int man_bits, int exp_bits, int binades_l, int binades_u, bool saturate) {   // :53
    CHECK_INPUT(a);
    c10::cuda::CUDAGuard guard(a.device());
    auto o = at::empty_like(a);
    check(mpt_superfp_quantize_nearest(a.data_ptr<float>(), o.data_ptr<float>(), a.numel(), man_bits, exp_bits, binades_l, binades_u, saturate, stream()));
    return o;
}

void mm_nearest(at::Tensor a, at::Tensor b, at::Tensor c, int64_t batch, int M, int N, int K, int man_add, int exp_add, int man_mul, int exp_mul,
                bool subnormals, bool saturate, bool compensated, bool fma) {
    CHECK_INPUT(a); CHECK_INPUT(b); CHECK_INPUT(c);
    c10::cuda::CUDAGuard guard(a.device());
    auto ws = at::empty({(int64_t)mpt_mm_workspace_bytes(batch)}, a.options().dtype(at::kByte));
    if (fma)
        check(mpt_float_mm_nearest_fma(a.data_ptr<float>(), b.data_ptr<float>(), c.data_ptr<float>(), batch, M, N, K, man_add, exp_add, subnormals,
                                       saturate, compensated, g_accum_order, ws.data_ptr(), (size_t)ws.numel(), stream()));
    else
        check(mpt_float_mm_nearest(a.data_ptr<float>(), b.data_ptr<float>(), c.data_ptr<float>(), batch, M, N, K, man_add, exp_add, man_mul, exp_mul,
                                   subnormals, saturate, compensated, g_accum_order, ws.data_ptr(), (size_t)ws.numel(), stream()));
}
int64_t batch_of(const at::Tensor& a) { return a.dim() > 2 ? a.size(0) : 1; }   // quant.cu:370-379

void float_quantize_nearest_mm(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_add, int exp_add, int man_mul, int exp_mul,
                               bool subnormals, bool saturate, bool compensated) {   // :123
    mm_nearest(a, b, c, 1, M, N, K, man_add, exp_add, man_mul, exp_mul, subnormals, saturate, compensated, false);
}
void float_quantize_nearest_bmm(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_add, int exp_add, int man_mul, int exp_mul,
                                bool subnormals, bool saturate, bool compensated) {   // :140
    mm_nearest(a, b, c, batch_of(a), M, N, K, man_add, exp_add, man_mul, exp_mul, subnormals, saturate, compensated, false);
}
void float_quantize_nearest_mm_fma(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_fma, int exp_fma, bool subnormals,
                                   bool saturate, bool compensated) {   // :157
    mm_nearest(a, b, c, 1, M, N, K, man_fma, exp_fma, man_fma, exp_fma, subnormals, saturate, compensated, true);
}
void float_quantize_nearest_bmm_fma(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_fma, int exp_fma, bool subnormals,
                                    bool saturate, bool compensated) {   // :173
    mm_nearest(a, b, c, batch_of(a), M, N, K, man_fma, exp_fma, man_fma, exp_fma, subnormals, saturate, compensated, true);
}

void mm_sr(at::Tensor a, at::Tensor b, at::Tensor c, int64_t batch, int M, int N, int K, int man_add, int exp_add, int rbits_add, int man_mul,
           int exp_mul, int rbits_mul, bool subnormals, bool saturate, bool fma) {
    CHECK_INPUT(a); CHECK_INPUT(b); CHECK_INPUT(c);
    c10::cuda::CUDAGuard guard(a.device());
    const uint64_t seed = (uint64_t)at::randint(0, INT64_MAX >> 1, {1}, at::kLong).item<int64_t>();   // reproducible under torch.manual_seed
    auto ws = at::empty({(int64_t)mpt_mm_workspace_bytes(batch)}, a.options().dtype(at::kByte));
    check(mpt_float_mm_stochastic(a.data_ptr<float>(), b.data_ptr<float>(), c.data_ptr<float>(), batch, M, N, K, man_add, exp_add, rbits_add, man_mul,
                                  exp_mul, rbits_mul, subnormals, saturate, fma, seed, ws.data_ptr(), (size_t)ws.numel(), stream()));
}
void float_quantize_stochastic_mm(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_add, int exp_add, int rbits_add,
                                  int man_mul, int exp_mul, int rbits_mul, bool subnormals, bool saturate) {   // :254
    mm_sr(a, b, c, 1, M, N, K, man_add, exp_add, rbits_add, man_mul, exp_mul, rbits_mul, subnormals, saturate, false);
}
void float_quantize_stochastic_bmm(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_add, int exp_add, int rbits_add,
                                   int man_mul, int exp_mul, int rbits_mul, bool subnormals, bool saturate) {   // :270
    mm_sr(a, b, c, batch_of(a), M, N, K, man_add, exp_add, rbits_add, man_mul, exp_mul, rbits_mul, subnormals, saturate, false);
}
void float_quantize_stochastic_mm_fma(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_fma, int exp_fma, int rbits_fma,
                                      bool subnormals, bool saturate) {   // :286
    mm_sr(a, b, c, 1, M, N, K, man_fma, exp_fma, rbits_fma, man_fma, exp_fma, rbits_fma, subnormals, saturate, true);
}
void float_quantize_stochastic_bmm_fma(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_fma, int exp_fma, int rbits_fma,
                                       bool subnormals, bool saturate) {   // :300
    mm_sr(a, b, c, batch_of(a), M, N, K, man_fma, exp_fma, rbits_fma, man_fma, exp_fma, rbits_fma, subnormals, saturate, true);
}

void float_quantize_nearest_softmax_forward(at::Tensor a, at::Tensor o, int dim, int man_exp, int exp_exp, int man_off, int exp_off, int man_acc,
                                            int exp_acc, bool subnormals, bool saturate) {   // :599
    CHECK_INPUT(a); CHECK_INPUT(o);
    c10::cuda::CUDAGuard guard(a.device());
    const Geom g = partition(a, {dim});
    check(mpt_float_softmax_forward(a.data_ptr<float>(), o.data_ptr<float>(), g.outer, g.channel, g.inner, man_exp, exp_exp, man_off, exp_off,
                                    man_acc, exp_acc, subnormals, saturate, g_reduce_order, stream()));
}
void float_quantize_nearest_softmax_lse_forward(at::Tensor a, at::Tensor o, int dim, int man_off, int exp_off, int man_lse, int exp_lse,
                                                bool subnormals, bool saturate) {   // :615
    CHECK_INPUT(a); CHECK_INPUT(o);
    c10::cuda::CUDAGuard guard(a.device());
    const Geom g = partition(a, {dim});
    check(mpt_float_softmax_lse_forward(a.data_ptr<float>(), o.data_ptr<float>(), g.outer, g.channel, g.inner, man_off, exp_off, man_lse, exp_lse,
                                        subnormals, saturate, g_reduce_order, stream()));
}
void float_quantize_nearest_softmax_backward(at::Tensor a, at::Tensor grad, at::Tensor o, int dim, int man_add, int exp_add, int man_mul,
                                             int exp_mul, bool subnormals, bool saturate) {   // :629
    CHECK_INPUT(a); CHECK_INPUT(grad); CHECK_INPUT(o);
    c10::cuda::CUDAGuard guard(a.device());
    const Geom g = partition(a, {dim});
    check(mpt_float_softmax_backward(a.data_ptr<float>(), grad.data_ptr<float>(), o.data_ptr<float>(), g.outer, g.channel, g.inner, man_add,
                                     exp_add, man_mul, exp_mul, subnormals, saturate, g_reduce_order, stream()));
}

void float_quantize_layernorm_forward(at::Tensor input, at::Tensor weight, at::Tensor bias, at::Tensor output, at::Tensor mean, at::Tensor rstd,
                                      float eps, std::vector<int> dims, int man_acc, int exp_acc, int man_mul, int exp_mul, int man_div,
                                      int exp_div, int man_sqrt, int exp_sqrt, bool subnormals, bool saturate) {   // :434
    CHECK_INPUT(input); CHECK_INPUT(weight); CHECK_INPUT(bias); CHECK_INPUT(output); CHECK_INPUT(mean); CHECK_INPUT(rstd);
    c10::cuda::CUDAGuard guard(input.device());
    const Geom g = partition(input, dims);
    check(mpt_float_layernorm_forward(input.data_ptr<float>(), weight.data_ptr<float>(), bias.data_ptr<float>(), output.data_ptr<float>(),
                                      mean.data_ptr<float>(), rstd.data_ptr<float>(), eps, g.outer, g.channel, g.inner, man_acc, exp_acc, man_mul,
                                      exp_mul, man_div, exp_div, man_sqrt, exp_sqrt, subnormals, saturate, g_reduce_order, stream()));
}
void float_quantize_layernorm_backward(at::Tensor input, at::Tensor grad_output, at::Tensor weight, at::Tensor bias, at::Tensor mean,
                                       at::Tensor rstd, at::Tensor grad_input, at::Tensor grad_gamma, at::Tensor grad_beta,
                                       std::vector<int> dims, int man_acc, int exp_acc, int man_mul, int exp_mul, int man_div, int exp_div,
                                       bool subnormals, bool saturate) {   // :459
    CHECK_INPUT(input); CHECK_INPUT(grad_output); CHECK_INPUT(weight); CHECK_INPUT(mean); CHECK_INPUT(rstd);
    CHECK_INPUT(grad_input); CHECK_INPUT(grad_gamma); CHECK_INPUT(grad_beta);
    (void)bias;
    c10::cuda::CUDAGuard guard(input.device());
    const Geom g = partition(input, dims);
    check(mpt_float_layernorm_backward(input.data_ptr<float>(), grad_output.data_ptr<float>(), weight.data_ptr<float>(), mean.data_ptr<float>(),
                                       rstd.data_ptr<float>(), grad_input.data_ptr<float>(), grad_gamma.data_ptr<float>(),
                                       grad_beta.data_ptr<float>(), g.outer, g.channel, g.inner, man_acc, exp_acc, man_mul, exp_mul, man_div,
                                       exp_div, subnormals, saturate, g_reduce_order, stream()));
}


// ---- the other nearest-rounding format families (pybind_cuda.cpp:815-824, :887-924) -------------------------------
enum class OverflowPolicy { SATURATE_INFTY = MPT_SATURATE_INFTY, SATURATE_MAXFLOAT = MPT_SATURATE_MAXFLOAT, SATURATE_MAXFLOAT2 = MPT_SATURATE_MAXFLOAT2 };

mpt_format superfp(int man, int exp, int bl, int bu, bool saturate) {
    mpt_format f{};
    f.kind = MPT_FMT_SUPERFP; f.man = man; f.exp = exp; f.subnormals = 1; f.saturate = saturate; f.binades_l = bl; f.binades_u = bu;
    f.P = 1; f.is_signed = 1;
    return f;
}
mpt_format binary8(int P, int policy, bool is_signed, bool subnormals) {
    mpt_format f{};
    f.kind = MPT_FMT_BINARY8; f.subnormals = subnormals; f.binades_l = f.binades_u = 1; f.P = P; f.is_signed = is_signed; f.overflow_policy = policy;
    return f;
}

void mm_fmt(at::Tensor a, at::Tensor b, at::Tensor c, int64_t batch, int M, int N, int K, const mpt_format& fa, const mpt_format& fm, bool fma) {
    CHECK_INPUT(a); CHECK_INPUT(b); CHECK_INPUT(c);
    c10::cuda::CUDAGuard guard(a.device());
    auto ws = at::empty({(int64_t)mpt_mm_workspace_bytes(batch)}, a.options().dtype(at::kByte));
    check(mpt_mm_nearest_fmt(a.data_ptr<float>(), b.data_ptr<float>(), c.data_ptr<float>(), batch, M, N, K, &fa, &fm, fma, g_accum_order,
                             ws.data_ptr(), (size_t)ws.numel(), stream()));
}
void superfp_quantize_nearest_mm(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_add, int exp_add, int man_mul, int exp_mul,
                                 int bal, int bau, int bml, int bmu, bool saturate) {   // :815
    mm_fmt(a, b, c, 1, M, N, K, superfp(man_add, exp_add, bal, bau, saturate), superfp(man_mul, exp_mul, bml, bmu, saturate), false);
}
void superfp_quantize_nearest_bmm(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_add, int exp_add, int man_mul, int exp_mul,
                                  int bal, int bau, int bml, int bmu, bool saturate) {   // :818
    mm_fmt(a, b, c, batch_of(a), M, N, K, superfp(man_add, exp_add, bal, bau, saturate), superfp(man_mul, exp_mul, bml, bmu, saturate), false);
}
void superfp_quantize_nearest_mm_fma(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_fma, int exp_fma, int bl, int bu,
                                     bool saturate) {   // :821
    const mpt_format f = superfp(man_fma, exp_fma, bl, bu, saturate);
    mm_fmt(a, b, c, 1, M, N, K, f, f, true);
}
void superfp_quantize_nearest_bmm_fma(at::Tensor a, at::Tensor b, at::Tensor c, int M, int N, int K, int man_fma, int exp_fma, int bl, int bu,
                                      bool saturate) {   // :824
    const mpt_format f = superfp(man_fma, exp_fma, bl, bu, saturate);
    mm_fmt(a, b, c, batch_of(a), M, N, K, f, f, true);
}

void softmax_fwd_fmt(at::Tensor a, at::Tensor o, int dim, const mpt_format& fe, const mpt_format& fo, const mpt_format& fa) {
    CHECK_INPUT(a); CHECK_INPUT(o);
    c10::cuda::CUDAGuard guard(a.device());
    const Geom g = partition(a, {dim});
    check(mpt_softmax_forward_fmt(a.data_ptr<float>(), o.data_ptr<float>(), g.outer, g.channel, g.inner, &fe, &fo, &fa, g_reduce_order, stream()));
}
void softmax_lse_fmt(at::Tensor a, at::Tensor o, int dim, const mpt_format& fo, const mpt_format& fl) {
    CHECK_INPUT(a); CHECK_INPUT(o);
    c10::cuda::CUDAGuard guard(a.device());
    const Geom g = partition(a, {dim});
    check(mpt_softmax_lse_forward_fmt(a.data_ptr<float>(), o.data_ptr<float>(), g.outer, g.channel, g.inner, &fo, &fl, g_reduce_order, stream()));
}
void softmax_bwd_fmt(at::Tensor a, at::Tensor gr, at::Tensor o, int dim, const mpt_format& fa, const mpt_format& fm) {
    CHECK_INPUT(a); CHECK_INPUT(gr); CHECK_INPUT(o);
    c10::cuda::CUDAGuard guard(a.device());
    const Geom g = partition(a, {dim});
    check(mpt_softmax_backward_fmt(a.data_ptr<float>(), gr.data_ptr<float>(), o.data_ptr<float>(), g.outer, g.channel, g.inner, &fa, &fm,
                                   g_reduce_order, stream()));
}
void superfp_quantize_nearest_softmax_forward(at::Tensor a, at::Tensor o, int dim, int man_exp, int exp_exp, int bel, int beu, int man_off,
                                              int exp_off, int bol, int bou, int man_acc, int exp_acc, int bal, int bau, bool saturate) {   // :887
    softmax_fwd_fmt(a, o, dim, superfp(man_exp, exp_exp, bel, beu, saturate), superfp(man_off, exp_off, bol, bou, saturate),
                    superfp(man_acc, exp_acc, bal, bau, saturate));
}
void superfp_quantize_nearest_softmax_lse_forward(at::Tensor a, at::Tensor o, int dim, int man_off, int exp_off, int bol, int bou, int man_lse,
                                                  int exp_lse, int bll, int blu, bool saturate) {   // :890
    softmax_lse_fmt(a, o, dim, superfp(man_off, exp_off, bol, bou, saturate), superfp(man_lse, exp_lse, bll, blu, saturate));
}
void superfp_quantize_nearest_softmax_backward(at::Tensor a, at::Tensor g, at::Tensor o, int dim, int man_add, int exp_add, int bal, int bau,
                                               int man_mul, int exp_mul, int bml, int bmu, bool saturate) {   // :893
    softmax_bwd_fmt(a, g, o, dim, superfp(man_add, exp_add, bal, bau, saturate), superfp(man_mul, exp_mul, bml, bmu, saturate));
}
void binary8_quantize_nearest_softmax_forward(at::Tensor a, at::Tensor o, int dim, int P_exp, int op_exp, bool signed_exp, int P_off, int op_off,
                                              bool signed_off, int P_acc, int op_acc, bool signed_acc, bool subnormals) {   // :897
    softmax_fwd_fmt(a, o, dim, binary8(P_exp, op_exp, signed_exp, subnormals), binary8(P_off, op_off, signed_off, subnormals),
                    binary8(P_acc, op_acc, signed_acc, subnormals));
}
void binary8_quantize_nearest_softmax_lse_forward(at::Tensor a, at::Tensor o, int dim, int P_off, int op_off, bool signed_off, int P_lse,
                                                  int op_lse, bool signed_lse, bool subnormals) {   // :900
    softmax_lse_fmt(a, o, dim, binary8(P_off, op_off, signed_off, subnormals), binary8(P_lse, op_lse, signed_lse, subnormals));
}
void binary8_quantize_nearest_softmax_backward(at::Tensor a, at::Tensor g, at::Tensor o, int dim, int P_add, int op_add, bool signed_add,
                                               int P_mul, int op_mul, bool signed_mul, bool subnormals) {   // :903
    softmax_bwd_fmt(a, g, o, dim, binary8(P_add, op_add, signed_add, subnormals), binary8(P_mul, op_mul, signed_mul, subnormals));
}

void layernorm_fwd_fmt(at::Tensor input, at::Tensor weight, at::Tensor bias, at::Tensor output, at::Tensor mean, at::Tensor rstd, float eps,
                       const std::vector<int>& dims, const mpt_format& fa, const mpt_format& fm, const mpt_format& fd, const mpt_format& fs) {
    CHECK_INPUT(input); CHECK_INPUT(weight); CHECK_INPUT(bias); CHECK_INPUT(output); CHECK_INPUT(mean); CHECK_INPUT(rstd);
    c10::cuda::CUDAGuard guard(input.device());
    const Geom g = partition(input, dims);
    check(mpt_layernorm_forward_fmt(input.data_ptr<float>(), weight.data_ptr<float>(), bias.data_ptr<float>(), output.data_ptr<float>(),
                                    mean.data_ptr<float>(), rstd.data_ptr<float>(), eps, g.outer, g.channel, g.inner, &fa, &fm, &fd, &fs,
                                    g_reduce_order, stream()));
}
void layernorm_bwd_fmt(at::Tensor input, at::Tensor grad_output, at::Tensor weight, at::Tensor mean, at::Tensor rstd, at::Tensor grad_input,
                       at::Tensor grad_gamma, at::Tensor grad_beta, const std::vector<int>& dims, const mpt_format& fa, const mpt_format& fm,
                       const mpt_format& fd) {
    CHECK_INPUT(input); CHECK_INPUT(grad_output); CHECK_INPUT(weight); CHECK_INPUT(mean); CHECK_INPUT(rstd);
    CHECK_INPUT(grad_input); CHECK_INPUT(grad_gamma); CHECK_INPUT(grad_beta);
    c10::cuda::CUDAGuard guard(input.device());
    const Geom g = partition(input, dims);
    check(mpt_layernorm_backward_fmt(input.data_ptr<float>(), grad_output.data_ptr<float>(), weight.data_ptr<float>(), mean.data_ptr<float>(),
                                     rstd.data_ptr<float>(), grad_input.data_ptr<float>(), grad_gamma.data_ptr<float>(),
                                     grad_beta.data_ptr<float>(), g.outer, g.channel, g.inner, &fa, &fm, &fd, g_reduce_order, stream()));
}
void superfp_quantize_layernorm_forward(at::Tensor input, at::Tensor weight, at::Tensor bias, at::Tensor output, at::Tensor mean, at::Tensor rstd,
                                        float eps, std::vector<int> dims, int man_acc, int exp_acc, int bal, int bau, int man_mul, int exp_mul,
                                        int bml, int bmu, int man_div, int exp_div, int bdl, int bdu, int man_sqrt, int exp_sqrt, int bsl,
                                        int bsu, bool saturate) {   // :914
    layernorm_fwd_fmt(input, weight, bias, output, mean, rstd, eps, dims, superfp(man_acc, exp_acc, bal, bau, saturate),
                      superfp(man_mul, exp_mul, bml, bmu, saturate), superfp(man_div, exp_div, bdl, bdu, saturate),
                      superfp(man_sqrt, exp_sqrt, bsl, bsu, saturate));
}
void superfp_quantize_layernorm_backward(at::Tensor input, at::Tensor grad_output, at::Tensor weight, at::Tensor bias, at::Tensor mean,
                                         at::Tensor rstd, at::Tensor grad_input, at::Tensor grad_gamma, at::Tensor grad_beta,
                                         std::vector<int> dims, int man_acc, int exp_acc, int bal, int bau, int man_mul, int exp_mul, int bml,
                                         int bmu, int man_div, int exp_div, int bdl, int bdu, bool saturate) {   // :917
    (void)bias;
    layernorm_bwd_fmt(input, grad_output, weight, mean, rstd, grad_input, grad_gamma, grad_beta, dims, superfp(man_acc, exp_acc, bal, bau, saturate),
                      superfp(man_mul, exp_mul, bml, bmu, saturate), superfp(man_div, exp_div, bdl, bdu, saturate));
}
void binary8_quantize_layernorm_forward(at::Tensor input, at::Tensor weight, at::Tensor bias, at::Tensor output, at::Tensor mean, at::Tensor rstd,
                                        float eps, std::vector<int> dims, int P_acc, int op_acc, bool signed_acc, int P_mul, int op_mul,
                                        bool signed_mul, int P_div, int op_div, bool signed_div, int P_sqrt, int op_sqrt, bool signed_sqrt,
                                        bool subnormals) {   // :921
    layernorm_fwd_fmt(input, weight, bias, output, mean, rstd, eps, dims, binary8(P_acc, op_acc, signed_acc, subnormals),
                      binary8(P_mul, op_mul, signed_mul, subnormals), binary8(P_div, op_div, signed_div, subnormals),
                      binary8(P_sqrt, op_sqrt, signed_sqrt, subnormals));
}
void binary8_quantize_layernorm_backward(at::Tensor input, at::Tensor grad_output, at::Tensor weight, at::Tensor bias, at::Tensor mean,
                                         at::Tensor rstd, at::Tensor grad_input, at::Tensor grad_gamma, at::Tensor grad_beta,
                                         std::vector<int> dims, int P_acc, int op_acc, bool signed_acc, int P_mul, int op_mul, bool signed_mul,
                                         int P_div, int op_div, bool signed_div, bool subnormals) {   // :924
    (void)bias;
    layernorm_bwd_fmt(input, grad_output, weight, mean, rstd, grad_input, grad_gamma, grad_beta, dims, binary8(P_acc, op_acc, signed_acc, subnormals),
                      binary8(P_mul, op_mul, signed_mul, subnormals), binary8(P_div, op_div, signed_div, subnormals));
}

// ---- entry points without a quant_cuda counterpart ----------------------------------------------------------------
at::Tensor qsum_rows(at::Tensor a, int man_bits, int exp_bits, bool subnormals, bool saturate) {
    CHECK_INPUT(a);
    TORCH_CHECK(a.dim() == 2, "qsum_rows expects a 2-D tensor");
    c10::cuda::CUDAGuard guard(a.device());
    auto o = at::empty({a.size(1)}, a.options());
    check(mpt_qsum_rows(a.data_ptr<float>(), o.data_ptr<float>(), a.size(0), a.size(1), man_bits, exp_bits, subnormals, saturate, stream()));
    return o;
}
void float_conv2d_nearest(at::Tensor x, at::Tensor wt, at::Tensor y, int groups, std::vector<int> kernel, std::vector<int> stride,
                          std::vector<int> padding, std::vector<int> dilation, int man_add, int exp_add, int man_mul, int exp_mul,
                          bool subnormals, bool saturate, bool fma) {
    CHECK_INPUT(x); CHECK_INPUT(wt); CHECK_INPUT(y);
    TORCH_CHECK(x.dim() == 4 && y.dim() == 4 && kernel.size() == 2 && stride.size() == 2 && padding.size() == 2 && dilation.size() == 2,
                "float_conv2d_nearest: NCHW tensors and 2-element geometry lists expected");
    c10::cuda::CUDAGuard guard(x.device());
    auto ws = at::empty({(int64_t)mpt_mm_workspace_bytes(1)}, x.options().dtype(at::kByte));
    check(mpt_float_conv2d_nearest(x.data_ptr<float>(), wt.data_ptr<float>(), y.data_ptr<float>(), (int)x.size(0), (int)x.size(1), (int)x.size(2),
                                   (int)x.size(3), (int)y.size(1), groups, kernel[0], kernel[1], stride[0], stride[1], padding[0], padding[1],
                                   dilation[0], dilation[1], man_add, exp_add, man_mul, exp_mul, subnormals, saturate, fma, g_accum_order,
                                   ws.data_ptr(), (size_t)ws.numel(), stream()));
}
std::vector<at::Tensor> mx_quantize(at::Tensor a, const std::string& elem, int block, bool return_scales, bool return_codes) {
    CHECK_INPUT(a);
    TORCH_CHECK(elem == "e4m3" || elem == "e2m1", "elem_format must be 'e4m3' or 'e2m1'");
    TORCH_CHECK(a.dim() >= 1 && block >= 1, "mx_quantize: at least one dimension and a positive block size");
    c10::cuda::CUDAGuard guard(a.device());
    const int64_t cols = a.size(-1), rows = cols ? a.numel() / cols : 0;
    auto o = at::empty_like(a);
    auto shape = a.sizes().vec();
    at::Tensor sc, codes;
    if (return_scales) { shape.back() = (cols + block - 1) / block; sc = at::empty(shape, a.options().dtype(at::kByte)); }
    if (return_codes) { shape.back() = elem == "e4m3" ? cols : (cols + 1) / 2; codes = at::zeros(shape, a.options().dtype(at::kByte)); }
    check(mpt_mx_quantize(a.data_ptr<float>(), o.data_ptr<float>(), return_scales ? sc.data_ptr<uint8_t>() : nullptr,
                          return_codes ? codes.data_ptr<uint8_t>() : nullptr, rows, cols, block, elem == "e4m3" ? MPT_ELEM_E4M3 : MPT_ELEM_E2M1,
                          stream()));
    std::vector<at::Tensor> out{o};
    if (return_scales) out.push_back(sc);
    if (return_codes) out.push_back(codes);
    return out;
}
std::vector<at::Tensor> nvfp4_quantize(at::Tensor a, double global_scale, bool return_scales, bool return_codes) {
    CHECK_INPUT(a);
    TORCH_CHECK(a.dim() >= 1, "nvfp4_quantize: at least one dimension");
    c10::cuda::CUDAGuard guard(a.device());
    const int64_t cols = a.size(-1), rows = cols ? a.numel() / cols : 0;
    auto o = at::empty_like(a);
    auto shape = a.sizes().vec();
    at::Tensor sc, gs, codes, scodes, ws;
    shape.back() = (cols + 15) / 16;
    if (return_scales) { sc = at::empty(shape, a.options()); gs = at::empty({1}, a.options()); }
    if (return_codes) {
        scodes = at::empty(shape, a.options().dtype(at::kByte));
        shape.back() = (cols + 1) / 2;
        codes = at::zeros(shape, a.options().dtype(at::kByte));
    }
    if (!(global_scale > 0.0)) ws = at::empty({1}, a.options().dtype(at::kInt));
    check(mpt_nvfp4_quantize(a.data_ptr<float>(), o.data_ptr<float>(), return_scales ? sc.data_ptr<float>() : nullptr,
                             return_codes ? codes.data_ptr<uint8_t>() : nullptr, return_codes ? scodes.data_ptr<uint8_t>() : nullptr, rows, cols,
                             global_scale > 0.0 ? (float)global_scale : 0.f, ws.defined() ? ws.data_ptr() : nullptr,
                             return_scales ? gs.data_ptr<float>() : nullptr, stream()));
    std::vector<at::Tensor> out{o};
    if (return_scales) { out.push_back(sc); out.push_back(gs); }
    if (return_codes) { out.push_back(codes); out.push_back(scodes); }
    return out;
}
// ---- serving from packed block formats (no quant_cuda counterpart).  Shapes and types are checked before devices. ----
int dense_type(const char* who, const at::Tensor& x) {
    switch (x.scalar_type()) {
        case at::kFloat: return MPT_DTYPE_F32;
        case at::kBFloat16: return MPT_DTYPE_BF16;
        case at::kHalf: return MPT_DTYPE_F16;
        default: TORCH_CHECK(false, who, ": float32, bfloat16 or float16 expected, not ", x.scalar_type());
    }
}
void no_gradient(const char* who, const at::Tensor& x) {
    TORCH_CHECK(!(x.requires_grad() && at::GradMode::is_enabled()), who, ": has no backward pass; call it under torch.no_grad()");
    TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && x._fw_grad(0).defined()), who, ": has no forward-mode derivative");
}
void bytes_tensor(const char* who, const char* what, const at::Tensor& t, int64_t dim) {
    TORCH_CHECK(t.scalar_type() == at::kByte && t.dim() == dim && t.is_contiguous(), who, ": ", what, " must be a contiguous uint8 tensor with ", dim,
                " dimensions");
}
void same_device(const char* who, const char* what, const at::Tensor& t, const at::Tensor& as) {
    TORCH_CHECK(t.is_cuda(), who, ": ", what, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == as.device(), who, ": ", what, " is on ", t.device(), ", expected ", as.device());
}
at::Tensor workspace(size_t bytes, const at::Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

at::Tensor block_linear(const std::string& who_s, const at::Tensor& x_in, const at::Tensor& codes, const at::Tensor& scales,
                        const std::optional<at::Tensor>& global_scale, const std::optional<at::Tensor>& bias, int format) {
    const char* who = who_s.c_str();
    const int dtype = dense_type(who, x_in);
    bytes_tensor(who, "codes", codes, 2);
    bytes_tensor(who, "scales", scales, 2);
    TORCH_CHECK(x_in.dim() >= 1, who, ": x needs at least one dimension");
    const int64_t n_in = x_in.size(-1), n_out = codes.size(0), group = format == MPT_BLOCK_NVFP4 ? 16 : 32;
    TORCH_CHECK(n_in % 32 == 0, who, ": the last dimension of x (", n_in, ") must be a multiple of 32");
    TORCH_CHECK(codes.size(1) * 2 == n_in, who, ": codes hold ", codes.size(1) * 2, " values a row, x has ", n_in);
    TORCH_CHECK(scales.size(0) == n_out && scales.size(1) * group == n_in, who, ": scales must be [", n_out, ", ", n_in / group, "]");
    if (bias) TORCH_CHECK(bias->scalar_type() == x_in.scalar_type() && bias->dim() == 1 && bias->size(0) == n_out, who, ": bias must be [", n_out, "] of x's type");
    if (global_scale) TORCH_CHECK(global_scale->scalar_type() == at::kFloat && global_scale->numel() == 1, who, ": global_scale must be one float32 value");
    no_gradient(who, x_in);
    if (bias) no_gradient(who, *bias);
    if (global_scale) no_gradient(who, *global_scale);
    TORCH_CHECK(x_in.is_cuda(), who, ": x must be a CUDA tensor");
    same_device(who, "codes", codes, x_in);
    same_device(who, "scales", scales, x_in);
    if (bias) same_device(who, "bias", *bias, x_in);
    if (global_scale) same_device(who, "global_scale", *global_scale, x_in);
    c10::cuda::CUDAGuard guard(x_in.device());
    const at::Tensor x = x_in.contiguous();
    const at::Tensor b = bias ? bias->contiguous() : at::Tensor();
    auto shape = x.sizes().vec();
    shape.back() = n_out;
    at::Tensor y = at::empty(shape, x.options());
    if (y.numel() == 0) return y;
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
    const size_t need = mpt_block_linear_workspace_bytes(rows, n_out, n_in, format, dtype);
    const at::Tensor ws = workspace(need, x);
    check(mpt_block_linear(x.data_ptr(), codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), global_scale ? global_scale->data_ptr<float>() : nullptr,
                           b.defined() ? b.data_ptr() : nullptr, y.data_ptr(), rows, n_out, n_in, format, dtype, need ? ws.data_ptr() : nullptr, need,
                           stream()));
    return y;
}
at::Tensor mx_linear(at::Tensor x, at::Tensor codes, at::Tensor scales, std::optional<at::Tensor> bias) {
    return block_linear("mx_linear", x, codes, scales, std::nullopt, bias, MPT_BLOCK_MXFP4);
}
at::Tensor nvfp4_linear(at::Tensor x, at::Tensor codes, at::Tensor scales, at::Tensor global_scale, std::optional<at::Tensor> bias) {
    return block_linear("nvfp4_linear", x, codes, scales, global_scale, bias, MPT_BLOCK_NVFP4);
}

struct ServingCall { mpt_mx_cache cache; mpt_mx_batch batch; };

// `rows`: new rows in all; `uniform_seqs`: the sequences they are split among without `starts`
ServingCall serving_call(const char* who, const std::vector<at::Tensor>& cache, const at::Tensor& pages, const at::Tensor& lens,
                         const std::optional<at::Tensor>& starts, int64_t rows) {
    static const char* const names[4] = {"k_codes", "k_scales", "v_codes", "v_scales"};
    TORCH_CHECK(cache.size() == 4, who, ": the cache is (k_codes, k_scales, v_codes, v_scales)");
    for (int i = 0; i < 4; ++i) bytes_tensor(who, names[i], cache[i], 4);
    const at::Tensor& kc = cache[0];
    const int64_t dim = cache[1].size(3) * 32;
    TORCH_CHECK(kc.size(3) == dim || kc.size(3) * 2 == dim, who, ": ", kc.size(3), " bytes of codes do not go with ", cache[1].size(3), " scales a row");
    for (int i = 1; i < 4; ++i)
        TORCH_CHECK(cache[i].size(0) == kc.size(0) && cache[i].size(1) == kc.size(1) && cache[i].size(2) == kc.size(2) &&
                    cache[i].size(3) == cache[i & 1].size(3), who, ": ", names[i], " does not match k_codes");
    TORCH_CHECK(pages.scalar_type() == at::kInt && pages.dim() == 2 && pages.is_contiguous(), who, ": pages must be a contiguous int32 matrix");
    const int64_t seqs = pages.size(0);
    TORCH_CHECK(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == seqs && lens.is_contiguous(), who, ": lens must be a contiguous int32 [", seqs, "]");
    if (starts)
        TORCH_CHECK(starts->scalar_type() == at::kInt && starts->dim() == 1 && starts->size(0) == seqs + 1 && starts->is_contiguous(), who,
                    ": starts must be a contiguous int32 [", seqs + 1, "]");
    TORCH_CHECK(kc.size(1) <= 65535 && dim <= 256 && kc.size(2) <= 256 && seqs <= INT_MAX && pages.size(1) <= INT_MAX, who, ": extents out of range");
    ServingCall s;
    s.cache = {cache[0].data_ptr<uint8_t>(), cache[1].data_ptr<uint8_t>(), cache[2].data_ptr<uint8_t>(), cache[3].data_ptr<uint8_t>(), kc.size(0),
               (int)kc.size(1), (int)dim, (int)kc.size(2), kc.size(3) == dim ? MPT_ELEM_E4M3 : MPT_ELEM_E2M1};
    s.batch = {pages.data_ptr<int>(), lens.data_ptr<int>(), starts ? starts->data_ptr<int>() : nullptr, rows, (int)seqs, (int)pages.size(1)};
    return s;
}
void serving_devices(const char* who, const at::Tensor& like, const std::vector<at::Tensor>& cache, const at::Tensor& pages, const at::Tensor& lens,
                     const std::optional<at::Tensor>& starts) {
    for (const auto& t : cache) same_device(who, "the cache", t, like);
    same_device(who, "pages", pages, like);
    same_device(who, "lens", lens, like);
    if (starts) same_device(who, "starts", *starts, like);
}
// [seqs, new, heads, dim], or [rows, heads, dim] with `starts`
void row_shape(const char* who, const char* what, const at::Tensor& t, bool ragged, int64_t seqs, int64_t dim) {
    TORCH_CHECK(ragged ? t.dim() == 3 : t.dim() == 4 && t.size(0) == seqs, who, ": ", what, " must be ",
                ragged ? "[rows, heads, head_dim] where starts is given" : "[sequences, new, heads, head_dim]");
    TORCH_CHECK(t.size(-1) == dim, who, ": ", what, " has rows of ", t.size(-1), " values, the cache of ", dim);
}
int64_t row_count(const at::Tensor& t) { return t.dim() == 3 ? t.size(0) : t.size(0) * t.size(1); }
std::array<int64_t, 3> row_strides(const at::Tensor& t) {
    const int64_t d = t.dim();
    return {d == 4 ? t.stride(0) : 0, t.stride(d - 3), t.stride(d - 2)};
}
// whether `t` may share memory with the contiguous tensor `out` and is not the same tensor: rows would be written before they are read
bool shares_memory(const at::Tensor& t, const at::Tensor& out) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    const char *a = static_cast<const char*>(t.data_ptr()), *b = static_cast<const char*>(out.data_ptr());
    const bool apart = a + (last + 1) * t.element_size() <= b || b + out.numel() * out.element_size() <= a;
    return !apart && !(a == b && t.is_contiguous());
}
at::Tensor dense_last(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

void mx_cache_write(at::Tensor k_in, at::Tensor v_in, std::vector<at::Tensor> cache, at::Tensor pages, at::Tensor lens, std::optional<at::Tensor> starts) {
    const char* who = "mx_cache_write";
    const int dtype = dense_type(who, k_in);
    TORCH_CHECK(k_in.dim() >= 3, who, ": k needs three or four dimensions");
    const ServingCall s = serving_call(who, cache, pages, lens, starts, row_count(k_in));
    row_shape(who, "k", k_in, starts.has_value(), s.batch.seqs, s.cache.dim);
    TORCH_CHECK(k_in.size(-2) == s.cache.heads, who, ": k has ", k_in.size(-2), " heads, the cache ", s.cache.heads);
    TORCH_CHECK(v_in.sizes() == k_in.sizes() && v_in.scalar_type() == k_in.scalar_type(), who, ": v must have the shape and type of k");
    no_gradient(who, k_in);
    no_gradient(who, v_in);
    TORCH_CHECK(k_in.is_cuda(), who, ": k must be a CUDA tensor");
    same_device(who, "v", v_in, k_in);
    serving_devices(who, k_in, cache, pages, lens, starts);
    c10::cuda::CUDAGuard guard(k_in.device());
    const at::Tensor k = dense_last(k_in), v = dense_last(v_in);
    const auto ks = row_strides(k), vs = row_strides(v);
    check(mpt_mx_cache_write(&s.cache, &s.batch, k.data_ptr(), v.data_ptr(), dtype, ks.data(), vs.data(), stream()));
}
std::vector<at::Tensor> mx_cache_read(std::vector<at::Tensor> cache, at::Tensor pages, at::Tensor lens, int64_t rows, std::optional<at::Tensor> starts,
                                      at::ScalarType type) {
    const char* who = "mx_cache_read";
    TORCH_CHECK(rows >= 0, who, ": a negative number of rows");
    const ServingCall s = serving_call(who, cache, pages, lens, starts, starts ? rows : rows * pages.size(0));
    TORCH_CHECK(cache[0].is_cuda(), who, ": the cache must be a CUDA tensor");
    serving_devices(who, cache[0], cache, pages, lens, starts);
    c10::cuda::CUDAGuard guard(cache[0].device());
    std::vector<int64_t> shape = starts ? std::vector<int64_t>{rows} : std::vector<int64_t>{s.batch.seqs, rows};
    shape.push_back(s.cache.heads);
    shape.push_back(s.cache.dim);
    at::Tensor k = at::empty(shape, cache[0].options().dtype(type)), v = at::empty_like(k);
    check(mpt_mx_cache_read(&s.cache, &s.batch, k.data_ptr(), v.data_ptr(), dense_type(who, k), stream()));
    return {k, v};
}
at::Tensor mx_attention(at::Tensor q_in, std::vector<at::Tensor> cache, at::Tensor pages, at::Tensor lens, std::optional<at::Tensor> starts, double scale,
                        int64_t window, int64_t sinks, std::optional<at::Tensor> out_in) {
    const char* who = "mx_attention";
    const int dtype = dense_type(who, q_in);
    TORCH_CHECK(q_in.dim() >= 3, who, ": q needs three or four dimensions");
    const ServingCall s = serving_call(who, cache, pages, lens, starts, row_count(q_in));
    row_shape(who, "q", q_in, starts.has_value(), s.batch.seqs, s.cache.dim);
    const int64_t heads = q_in.size(-2);
    TORCH_CHECK(s.cache.heads > 0 && heads > 0 && heads % s.cache.heads == 0, who, ": ", heads, " query heads do not divide among ", s.cache.heads, " kv heads");
    TORCH_CHECK(window >= 0 && sinks >= 0 && window <= INT_MAX && sinks <= INT_MAX, who, ": window and sinks must not be negative");
    if (out_in)
        TORCH_CHECK(out_in->sizes() == q_in.sizes() && out_in->scalar_type() == q_in.scalar_type() && out_in->is_contiguous(), who,
                    ": out must be contiguous with the shape and type of q");
    no_gradient(who, q_in);
    if (out_in) no_gradient(who, *out_in);
    TORCH_CHECK(q_in.is_cuda(), who, ": q must be a CUDA tensor");
    if (out_in) same_device(who, "out", *out_in, q_in);
    serving_devices(who, q_in, cache, pages, lens, starts);
    c10::cuda::CUDAGuard guard(q_in.device());
    at::Tensor q = dense_last(q_in);
    at::Tensor out = out_in ? *out_in : at::empty(q.sizes(), q.options());
    if (out.numel() == 0) return out;
    if (out_in && shares_memory(q, out)) q = q.clone();
    const auto qs = row_strides(q);
    const size_t need = mpt_mx_attention_workspace_bytes(&s.cache, &s.batch, (int)heads, dtype, (int)window, (int)sinks);
    const at::Tensor ws = workspace(need, q);
    check(mpt_mx_attention(&s.cache, &s.batch, q.data_ptr(), dtype, qs.data(), (int)heads, (float)scale, (int)window, (int)sinks, out.data_ptr(),
                           out_in ? 0 : 1, need ? ws.data_ptr() : nullptr, need, stream()));
    if (out_in && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();      // written in place
    return out;
}

void float_quantize_multi(std::vector<at::Tensor> ins, std::vector<at::Tensor> outs, int man_bits, int exp_bits, bool subnormals, bool saturate,
                          int rounding, int prng_bits, uint64_t seed) {
    TORCH_CHECK(ins.size() == outs.size(), "float_quantize_multi: as many outputs as inputs");
    if (ins.empty()) return;
    std::vector<const float*> pi(ins.size());
    std::vector<float*> po(ins.size());
    std::vector<int64_t> n(ins.size());
    for (size_t i = 0; i < ins.size(); ++i) {
        CHECK_INPUT(ins[i]); CHECK_INPUT(outs[i]);
        TORCH_CHECK(ins[i].device() == ins[0].device() && outs[i].device() == ins[0].device() && ins[i].numel() == outs[i].numel(),
                    "float_quantize_multi: tensors must live on one device and outputs must match inputs in size");
        pi[i] = ins[i].data_ptr<float>(); po[i] = outs[i].data_ptr<float>(); n[i] = ins[i].numel();
    }
    c10::cuda::CUDAGuard guard(ins[0].device());
    check(mpt_float_quantize_multi(pi.data(), po.data(), n.data(), (int)ins.size(), man_bits, exp_bits, subnormals, saturate, rounding, prng_bits,
                                   seed, stream()));
}
std::vector<at::Tensor> scale_quantize(at::Tensor a, double normal_max, int margin, bool quantize, int man, int exp, bool subnormals, bool saturate) {
    CHECK_INPUT(a);
    TORCH_CHECK(a.dim() >= 2, "scale_quantize expects at least two dimensions");
    c10::cuda::CUDAGuard guard(a.device());
    const int64_t per = a.size(-1) * a.size(-2), mats = per ? a.numel() / per : 0;
    auto o = at::empty_like(a);
    auto shape = a.sizes().vec();
    shape[shape.size() - 1] = 1; shape[shape.size() - 2] = 1;
    auto sc = at::empty(shape, a.options());
    auto ws = at::empty({(int64_t)mpt_scale_quantize_workspace_bytes(mats)}, a.options().dtype(at::kByte));
    check(mpt_scale_quantize(a.data_ptr<float>(), o.data_ptr<float>(), mats, per, normal_max, margin, quantize, man, exp, subnormals, saturate,
                             sc.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream()));
    return {o, sc};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "quant_cuda-compatible front end of the B200 simulated-arithmetic kernels";
    // reference: pybind_cuda.cpp:784-787; the binary8 entry points take the policy as an int, which accepts this enum
    py::enum_<OverflowPolicy>(m, "OverflowPolicy", py::arithmetic(), py::module_local())
        .value("SATURATE_INFTY", OverflowPolicy::SATURATE_INFTY)
        .value("SATURATE_MAXFLOAT", OverflowPolicy::SATURATE_MAXFLOAT)
        .value("SATURATE_MAXFLOAT2", OverflowPolicy::SATURATE_MAXFLOAT2);
    m.def("set_accum_order", [](const std::string& o) { g_accum_order = (o == "seq") ? MPT_ORDER_SEQ : MPT_ORDER_CUDA; });
    m.def("set_reduce_order", [](const std::string& o) { g_reduce_order = (o == "seq") ? MPT_ORDER_SEQ : MPT_ORDER_CUDA; });
    m.def("float_quantize_nearest", &float_quantize_nearest);
    m.def("float_quantize_stochastic", &float_quantize_stochastic);
    m.def("float_quantize_truncate", &float_quantize_truncate);
    m.def("binary8_quantize_nearest", &binary8_quantize_nearest);
    m.def("binary8_quantize_stochastic", &binary8_quantize_stochastic);
    m.def("binary8_quantize_truncate", &binary8_quantize_truncate);
    m.def("superfp_quantize_nearest", &superfp_quantize_nearest);
    m.def("float_quantize_nearest_mm", &float_quantize_nearest_mm);
    m.def("float_quantize_nearest_bmm", &float_quantize_nearest_bmm);
    m.def("float_quantize_nearest_mm_fma", &float_quantize_nearest_mm_fma);
    m.def("float_quantize_nearest_bmm_fma", &float_quantize_nearest_bmm_fma);
    m.def("float_quantize_stochastic_mm", &float_quantize_stochastic_mm);
    m.def("float_quantize_stochastic_bmm", &float_quantize_stochastic_bmm);
    m.def("float_quantize_stochastic_mm_fma", &float_quantize_stochastic_mm_fma);
    m.def("float_quantize_stochastic_bmm_fma", &float_quantize_stochastic_bmm_fma);
    m.def("float_quantize_nearest_softmax_forward", &float_quantize_nearest_softmax_forward);
    m.def("float_quantize_nearest_softmax_lse_forward", &float_quantize_nearest_softmax_lse_forward);
    m.def("float_quantize_nearest_softmax_backward", &float_quantize_nearest_softmax_backward);
    m.def("float_quantize_layernorm_forward", &float_quantize_layernorm_forward);
    m.def("float_quantize_layernorm_backward", &float_quantize_layernorm_backward);
    m.def("superfp_quantize_nearest_mm", &superfp_quantize_nearest_mm);
    m.def("superfp_quantize_nearest_bmm", &superfp_quantize_nearest_bmm);
    m.def("superfp_quantize_nearest_mm_fma", &superfp_quantize_nearest_mm_fma);
    m.def("superfp_quantize_nearest_bmm_fma", &superfp_quantize_nearest_bmm_fma);
    m.def("superfp_quantize_nearest_softmax_forward", &superfp_quantize_nearest_softmax_forward);
    m.def("superfp_quantize_nearest_softmax_lse_forward", &superfp_quantize_nearest_softmax_lse_forward);
    m.def("superfp_quantize_nearest_softmax_backward", &superfp_quantize_nearest_softmax_backward);
    m.def("binary8_quantize_nearest_softmax_forward", &binary8_quantize_nearest_softmax_forward);
    m.def("binary8_quantize_nearest_softmax_lse_forward", &binary8_quantize_nearest_softmax_lse_forward);
    m.def("binary8_quantize_nearest_softmax_backward", &binary8_quantize_nearest_softmax_backward);
    m.def("superfp_quantize_layernorm_forward", &superfp_quantize_layernorm_forward);
    m.def("superfp_quantize_layernorm_backward", &superfp_quantize_layernorm_backward);
    m.def("binary8_quantize_layernorm_forward", &binary8_quantize_layernorm_forward);
    m.def("binary8_quantize_layernorm_backward", &binary8_quantize_layernorm_backward);
    m.def("qsum_rows", &qsum_rows);
    m.def("float_conv2d_nearest", &float_conv2d_nearest, py::arg("x"), py::arg("wt"), py::arg("y"), py::arg("groups"), py::arg("kernel_size"),
          py::arg("stride"), py::arg("padding"), py::arg("dilation"), py::arg("man_add"), py::arg("exp_add"), py::arg("man_mul"), py::arg("exp_mul"),
          py::arg("subnormals"), py::arg("saturate"), py::arg("fma") = false);
    m.def("mx_quantize", &mx_quantize, py::arg("a"), py::arg("elem_format") = "e4m3", py::arg("block") = 32, py::arg("return_scales") = false,
          py::arg("return_codes") = false);
    m.def("nvfp4_quantize", &nvfp4_quantize, py::arg("a"), py::arg("global_scale") = 0.0, py::arg("return_scales") = false,
          py::arg("return_codes") = false);
    m.def("float_quantize_multi", &float_quantize_multi, py::arg("ins"), py::arg("outs"), py::arg("man_bits"), py::arg("exp_bits"),
          py::arg("subnormals"), py::arg("saturate"), py::arg("rounding") = 0, py::arg("prng_bits") = 0, py::arg("seed") = 0);
    m.def("scale_quantize", &scale_quantize);
    m.def("mx_linear", &mx_linear);
    m.def("nvfp4_linear", &nvfp4_linear);
    m.def("mx_cache_write", &mx_cache_write);
    m.def("mx_cache_read", &mx_cache_read);
    m.def("mx_attention", &mx_attention);
}
