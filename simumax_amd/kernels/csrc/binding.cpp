// PyTorch bindings for the simumax_amd gfx950 kernels.
// Compiled directly with hipcc (no hipify pass) by kernels/build.py.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include "vocab.h"

#define CHECK_IN(t)                                                     \
    TORCH_CHECK((t).is_cuda(), #t " must be on GPU");                   \
    TORCH_CHECK((t).is_contiguous(), #t " must be contiguous")

static hipStream_t cur_stream() {
    return c10::hip::getCurrentHIPStream().stream();
}

extern "C" {
void rmsnorm_fwd_launch(const void *, const void *, void *, void *, int, int,
                        float, hipStream_t);
void rmsnorm_bwd_launch(const void *, const void *, const void *, const void *,
                        void *, void *, int, int, hipStream_t);
void rope_launch(const void *, void *, const void *, const void *, int, int,
                 int, float, hipStream_t);
void swiglu_fwd_launch(const void *, void *, long, int, hipStream_t);
void swiglu_bwd_launch(const void *, const void *, void *, long, int,
                       hipStream_t);
void ce_fwd_launch(const void *, const void *, void *, void *, void *, long,
                   int, hipStream_t);
void ce_bwd_launch(const void *, const void *, const void *, const void *,
                   const void *, void *, long, int, hipStream_t);
void fp8_cast_launch(const void *, void *, void *, const void *, long, int,
                     float, hipStream_t);
void fp8_cast_t_launch(const void *, void *, void *, void *, const void *,
                       int, int, int, float, hipStream_t);
}

std::vector<torch::Tensor> rmsnorm_fwd(torch::Tensor x, torch::Tensor w,
                                       double eps) {
    CHECK_IN(x);
    CHECK_IN(w);
    TORCH_CHECK(x.scalar_type() == torch::kBFloat16, "x must be bf16");
    const int H = x.size(-1);
    const long rows = x.numel() / H;
    TORCH_CHECK(H % 8 == 0, "H must be a multiple of 8");
    auto y = torch::empty_like(x);
    auto rstd = torch::empty({rows}, x.options().dtype(torch::kFloat32));
    rmsnorm_fwd_launch(x.data_ptr(), w.data_ptr(), y.data_ptr(),
                       rstd.data_ptr(), (int)rows, H, (float)eps,
                       cur_stream());
    return {y, rstd};
}

std::vector<torch::Tensor> rmsnorm_bwd(torch::Tensor dy, torch::Tensor x,
                                       torch::Tensor w, torch::Tensor rstd) {
    CHECK_IN(dy);
    CHECK_IN(x);
    CHECK_IN(w);
    CHECK_IN(rstd);
    const int H = x.size(-1);
    const long rows = x.numel() / H;
    auto dx = torch::empty_like(x);
    auto dw = torch::zeros({H}, x.options().dtype(torch::kFloat32));
    rmsnorm_bwd_launch(dy.data_ptr(), x.data_ptr(), w.data_ptr(),
                       rstd.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                       (int)rows, H, cur_stream());
    return {dx, dw};
}

torch::Tensor rope(torch::Tensor x, torch::Tensor cs, torch::Tensor pos,
                   double sign) {
    CHECK_IN(x);
    CHECK_IN(cs);
    CHECK_IN(pos);
    TORCH_CHECK(x.dim() == 3, "x must be [tokens, heads, D]");
    const int D = x.size(2);
    const int heads = x.size(1);
    const int rows = x.size(0);
    TORCH_CHECK(D % 2 == 0);
    auto y = torch::empty_like(x);
    rope_launch(x.data_ptr(), y.data_ptr(), cs.data_ptr(), pos.data_ptr(),
                rows, heads, D, (float)sign, cur_stream());
    return y;
}

torch::Tensor swiglu_fwd(torch::Tensor x) {
    CHECK_IN(x);
    const int I2 = x.size(-1);
    TORCH_CHECK(I2 % 16 == 0, "last dim must be a multiple of 16");
    const long rows = x.numel() / I2;
    auto sizes = x.sizes().vec();
    sizes.back() = I2 / 2;
    auto y = torch::empty(sizes, x.options());
    swiglu_fwd_launch(x.data_ptr(), y.data_ptr(), rows, I2 / 2, cur_stream());
    return y;
}

torch::Tensor swiglu_bwd(torch::Tensor dy, torch::Tensor x) {
    CHECK_IN(dy);
    CHECK_IN(x);
    const int I2 = x.size(-1);
    const long rows = x.numel() / I2;
    auto dx = torch::empty_like(x);
    swiglu_bwd_launch(dy.data_ptr(), x.data_ptr(), dx.data_ptr(), rows, I2 / 2,
                      cur_stream());
    return dx;
}

std::vector<torch::Tensor> ce_fwd(torch::Tensor logits, torch::Tensor labels) {
    CHECK_IN(logits);
    CHECK_IN(labels);
    TORCH_CHECK(labels.scalar_type() == torch::kInt64);
    const int V = logits.size(-1);
    TORCH_CHECK(V % 8 == 0, "fused CE requires vocab % 8 == 0 (pad the vocab)");
    const long rows = logits.numel() / V;
    auto opts = logits.options().dtype(torch::kFloat32);
    auto loss = torch::empty({rows}, opts);
    auto row_max = torch::empty({rows}, opts);
    auto row_sum = torch::empty({rows}, opts);
    ce_fwd_launch(logits.data_ptr(), labels.data_ptr(), loss.data_ptr(),
                  row_max.data_ptr(), row_sum.data_ptr(), rows, V,
                  cur_stream());
    return {loss, row_max, row_sum};
}

torch::Tensor ce_bwd(torch::Tensor logits, torch::Tensor labels,
                     torch::Tensor dloss, torch::Tensor row_max,
                     torch::Tensor row_sum) {
    CHECK_IN(logits);
    const int V = logits.size(-1);
    const long rows = logits.numel() / V;
    auto dlogits = torch::empty_like(logits);
    ce_bwd_launch(logits.data_ptr(), labels.data_ptr(), dloss.data_ptr(),
                  row_max.data_ptr(), row_sum.data_ptr(), dlogits.data_ptr(),
                  rows, V, cur_stream());
    return dlogits;
}

extern "C" {
void mfma_probe_launch(const void *, const void *, void *, void *, int,
                       hipStream_t);
void fa_fwd_launch(const void *, const void *, const void *, void *, void *,
                   int, int, int, int, int, int, hipStream_t);
void fa_bwd_launch(const void *, const void *, const void *, const void *,
                   const void *, const void *, void *, void *, void *, int,
                   int, int, int, int, int, hipStream_t);
}

std::vector<torch::Tensor> mfma_probe(torch::Tensor A, torch::Tensor B,
                                      long mode) {
    CHECK_IN(A);
    CHECK_IN(B);
    auto f32 = A.options().dtype(torch::kFloat32);
    auto cm = torch::zeros({16, 16}, f32);
    auto cr = torch::zeros({64, 4}, f32);
    mfma_probe_launch(A.data_ptr(), B.data_ptr(), cm.data_ptr(), cr.data_ptr(),
                      (int)mode, cur_stream());
    return {cm, cr};
}

std::vector<torch::Tensor> fa_fwd(torch::Tensor q, torch::Tensor k,
                                  torch::Tensor v, bool causal) {
    CHECK_IN(q);
    CHECK_IN(k);
    CHECK_IN(v);
    TORCH_CHECK(q.dim() == 4, "q must be [B,S,Hq,Dqk]");
    const int B = q.size(0), S = q.size(1), Hq = q.size(2), Dqk = q.size(3);
    const int Hkv = k.size(2), Dv = v.size(3);
    TORCH_CHECK(Dqk == 128 || Dqk == 192, "fa kernel supports Dqk in {128,192}");
    TORCH_CHECK(Dv == 128, "fa kernel supports Dv=128");
    TORCH_CHECK(Hq % Hkv == 0);
    auto o = torch::empty({B, S, Hq, Dv}, q.options());
    auto lse = torch::empty({B, Hq, S}, q.options().dtype(torch::kFloat32));
    fa_fwd_launch(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                  lse.data_ptr(), B, S, Hq, Hkv, Dqk, causal ? 1 : 0,
                  cur_stream());
    return {o, lse};
}

std::vector<torch::Tensor> fa_bwd(torch::Tensor dout, torch::Tensor q,
                                  torch::Tensor k, torch::Tensor v,
                                  torch::Tensor o, torch::Tensor lse,
                                  bool causal) {
    CHECK_IN(dout);
    CHECK_IN(q);
    const int B = q.size(0), S = q.size(1), Hq = q.size(2), Dqk = q.size(3);
    const int Hkv = k.size(2), Dv = v.size(3);
    auto f32 = q.options().dtype(torch::kFloat32);
    auto dq = torch::empty({B, S, Hq, Dqk}, q.options());
    auto dkv = torch::zeros({B, S, Hkv, Dqk + Dv}, f32);
    auto dsum = torch::empty({B, Hq, S}, f32);
    fa_bwd_launch(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  o.data_ptr(), lse.data_ptr(), dq.data_ptr(), dkv.data_ptr(),
                  dsum.data_ptr(), B, S, Hq, Hkv, Dqk, causal ? 1 : 0,
                  cur_stream());
    auto dk = dkv.narrow(3, 0, Dqk).to(torch::kBFloat16);
    auto dv = dkv.narrow(3, Dqk, Dv).to(torch::kBFloat16);
    return {dq, dk.contiguous(), dv.contiguous()};
}

void wgrad_accum(torch::Tensor dout, torch::Tensor x, torch::Tensor main_grad);

extern "C" {
void gg_fwd(const void *, const void *, void *, int, int, int, int,
            hipStream_t);
void gg_dgrad(const void *, const void *, void *, int, int, int, int,
              hipStream_t);
void gg_wgrad(const void *, const void *, void *, int, int, int, int,
              hipStream_t);
}

// grouped expert GEMMs (see grouped_gemm.hip); weights are [E, N, K]
torch::Tensor grouped_fwd(torch::Tensor x, torch::Tensor w) {
    CHECK_IN(x);
    CHECK_IN(w);
    TORCH_CHECK(x.dim() == 3 && w.dim() == 3, "x [E,M,K], w [E,N,K]");
    const int E = x.size(0), M = x.size(1), K = x.size(2), N = w.size(1);
    TORCH_CHECK(w.size(0) == E && (int)w.size(2) == K);
    TORCH_CHECK(N % 128 == 0 && K % 128 == 0, "grouped fwd needs N%128, K%128");
    auto c = torch::empty({E, M, N}, x.options());
    gg_fwd(x.data_ptr(), w.data_ptr(), c.data_ptr(), E, M, N, K,
           cur_stream());
    return c;
}

torch::Tensor grouped_dgrad(torch::Tensor dout, torch::Tensor w) {
    CHECK_IN(dout);
    CHECK_IN(w);
    const int E = dout.size(0), M = dout.size(1), N = dout.size(2);
    const int K = w.size(2);
    TORCH_CHECK((int)w.size(1) == N);
    TORCH_CHECK(K % 128 == 0 && N % 32 == 0, "grouped dgrad needs K%128, N%32");
    auto dx = torch::empty({E, M, K}, dout.options());
    gg_dgrad(dout.data_ptr(), w.data_ptr(), dx.data_ptr(), E, M, N, K,
             cur_stream());
    return dx;
}

void grouped_wgrad(torch::Tensor dout, torch::Tensor x, torch::Tensor g) {
    CHECK_IN(dout);
    CHECK_IN(x);
    CHECK_IN(g);
    const int E = dout.size(0), M = dout.size(1), N = dout.size(2);
    const int K = x.size(2);
    TORCH_CHECK(g.scalar_type() == torch::kFloat32, "main_grad must be fp32");
    TORCH_CHECK((int)g.size(1) == N && (int)g.size(2) == K);
    TORCH_CHECK(N % 128 == 0 && K % 128 == 0, "grouped wgrad needs N%128, K%128");
    gg_wgrad(dout.data_ptr(), x.data_ptr(), g.data_ptr(), E, M, N, K,
             cur_stream());
}

// fused bf16 -> fp8 cast with delayed-scaling amax update; out must be a
// float8 tensor of x's shape, amax a zeroed fp32 [1], scale fp32 [1]
void fp8_cast(torch::Tensor x, torch::Tensor out, torch::Tensor amax,
              torch::Tensor scale, bool e5m2, double fmax) {
    CHECK_IN(x);
    TORCH_CHECK(out.is_cuda() && out.is_contiguous(), "out");
    TORCH_CHECK(x.scalar_type() == torch::kBFloat16, "x must be bf16");
    TORCH_CHECK(x.numel() % 8 == 0, "numel % 8");
    TORCH_CHECK(out.numel() == x.numel(), "out size");
    fp8_cast_launch(x.data_ptr(), out.data_ptr(), amax.data_ptr(),
                    scale.data_ptr(), (long)x.numel(), e5m2 ? 1 : 0,
                    (float)fmax, cur_stream());
}

// cast + transpose in one pass: out [M,N] fp8 + out_t [N,M] fp8
void fp8_cast_t(torch::Tensor x, torch::Tensor out, torch::Tensor out_t,
                torch::Tensor amax, torch::Tensor scale, bool e5m2,
                double fmax) {
    CHECK_IN(x);
    TORCH_CHECK(x.dim() == 2 && x.scalar_type() == torch::kBFloat16, "x");
    const int M = x.size(0), N = x.size(1);
    TORCH_CHECK(M % 64 == 0 && N % 64 == 0, "dims must be multiples of 64");
    TORCH_CHECK(out.numel() == x.numel() && out_t.numel() == x.numel(),
                "out sizes");
    fp8_cast_t_launch(x.data_ptr(), out.data_ptr(), out_t.data_ptr(),
                      amax.data_ptr(), scale.data_ptr(), M, N,
                      e5m2 ? 1 : 0, (float)fmax, cur_stream());
}

// ---- operators over the rows of logits (see vocab.hip) ----
extern "C" {
int vocab_segment(int);
int vocab_group(void);
void logprobs_fwd_launch(const VocabRows *, const VocabLogprobs *, int,
                         hipStream_t);
void distill_fwd_launch(const VocabRows *, const VocabDistill *, int,
                        hipStream_t);
void vocab_grad_launch(const VocabRows *, const VocabGrad *, int, void *, int,
                       hipStream_t);
}

static int vocab_dtype(const torch::Tensor &t) {
    switch (t.scalar_type()) {
        case torch::kBFloat16: return VOCAB_BF16;
        case torch::kFloat16: return VOCAB_FP16;
        case torch::kFloat32: return VOCAB_FP32;
        default: TORCH_CHECK(false, "logits must be bf16, fp16 or fp32");
    }
}

// the rows of [..., V] logits as at most two strided dimensions; false if
// their strides need more than that
static bool vocab_rows(const torch::Tensor &x, VocabRows *g) {
    TORCH_CHECK(x.is_cuda(), "logits must be on GPU");
    TORCH_CHECK(x.dim() >= 1, "logits must be [..., V]");
    const int64_t V = x.size(-1);
    TORCH_CHECK(V >= 1 && V < (1ll << 31), "vocabulary of ", V, " tokens");
    if (V > 1 && x.stride(-1) != 1) return false;
    int64_t rows = 1;
    std::vector<std::pair<int64_t, int64_t>> dims;  // (size, stride), merged
    for (int i = 0; i + 1 < x.dim(); ++i) {
        rows *= x.size(i);
        if (x.size(i) == 1) continue;
        if (!dims.empty() && dims.back().second == x.stride(i) * x.size(i)) {
            dims.back().first *= x.size(i);
            dims.back().second = x.stride(i);
        } else {
            dims.emplace_back(x.size(i), x.stride(i));
        }
    }
    TORCH_CHECK(rows < (1ll << 31), rows, " rows of logits");
    if (dims.size() > 2) return false;
    while (dims.size() < 2) dims.insert(dims.begin(), {1, 0});
    g->base = x.data_ptr();
    g->V = V;
    g->stride_o = dims[0].second;
    g->stride_i = dims[1].second;
    g->rows = (int)rows;
    g->inner = (int)std::max<int64_t>(dims[1].first, 1);
    const int seg = vocab_segment(vocab_dtype(x));
    const int64_t size = x.element_size();
    const bool shifted = (int64_t)x.data_ptr() % 128 ||
                         g->stride_o * size % 128 || g->stride_i * size % 128;
    // a vocabulary at the limit leaves no room for the shift
    g->line = shifted && V + 127 < VOCAB_MAX_TOP_V ? 127 : 0;
    g->nseg = (int)((V + (g->line ? 127 / size : 0) + seg - 1) / seg);
    TORCH_CHECK(rows * g->nseg < (1ll << 31), rows, " rows of ", V, " logits");
    return true;
}

static VocabRows vocab_rows_or_copy(torch::Tensor &x) {
    VocabRows g;
    if (!vocab_rows(x, &g)) {
        x = x.contiguous();
        TORCH_CHECK(vocab_rows(x, &g));
    }
    return g;
}

#define CHECK_ROWS(t, type, n)                                           \
    CHECK_IN(t);                                                         \
    TORCH_CHECK((t).device() == logits.device(),                         \
                #t " must be on the device of the logits");              \
    TORCH_CHECK((t).scalar_type() == (type), #t " has the wrong dtype"); \
    TORCH_CHECK((t).numel() == (int64_t)(n), #t " has the wrong size")

// torch::empty without the dispatcher: the smallest calls take as long as the
// host does, of which their up to seven tensors are the most (16 rows of 32000,
// 5 alternatives: 12.7 us with torch::empty, 11.3 us so).
static torch::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type,
                                const torch::Tensor &logits) {
    return at::detail::empty_cuda(sizes, type, logits.device(), c10::nullopt);
}

static std::vector<int64_t> lead_sizes(const torch::Tensor &x) {
    auto s = x.sizes().vec();
    s.pop_back();
    return s;
}

// -> logprobs, entropy, top_logprobs, top_ids, stat
std::vector<torch::Tensor> token_logprobs_fwd(
    torch::Tensor logits, c10::optional<torch::Tensor> tokens, int64_t topk,
    double temperature, int64_t ignore_index) {
    c10::OptionalDeviceGuard guard(logits.device());
    VocabRows g = vocab_rows_or_copy(logits);
    TORCH_CHECK(topk >= 0 && topk <= VOCAB_MAX_K && topk <= g.V, "topk");
    TORCH_CHECK(topk == 0 || g.V <= VOCAB_MAX_TOP_V,
                "top alternatives of a vocabulary above ", VOCAB_MAX_TOP_V);
    // what precedes a row in its first line is among its groups
    TORCH_CHECK(topk == 0 || g.V + g.line / logits.element_size() <=
                                 VOCAB_MAX_TOP_V,
                "a row's groups are more than its threads hold");
    TORCH_CHECK(temperature > 0, "temperature");
    if (tokens) {
        CHECK_ROWS(*tokens, torch::kInt64, g.rows);
    }
    const auto f32 = torch::kFloat32;
    const auto lead = lead_sizes(logits);
    auto top_shape = lead;
    top_shape.push_back(topk);
    auto logprobs = new_tensor(tokens ? lead : std::vector<int64_t>{0}, f32,
                               logits);
    auto entropy = new_tensor(lead, f32, logits);
    auto top_lp = new_tensor(top_shape, f32, logits);
    auto top_ids = new_tensor(top_shape, torch::kInt64, logits);
    auto stat = new_tensor({g.rows, 4}, f32, logits);
    if (g.rows > 0) {
        auto part = new_tensor({g.rows, g.nseg, 4}, f32, logits);
        const int dt = vocab_dtype(logits);
        torch::Tensor gmax;
        if (topk > 0)
            gmax = new_tensor({g.rows, g.nseg,
                               vocab_segment(dt) / vocab_group()},
                              logits.scalar_type(), logits);
        VocabLogprobs a;
        a.gmax = topk > 0 ? gmax.data_ptr() : nullptr;
        a.tokens = tokens ? tokens->data_ptr<int64_t>() : nullptr;
        a.ignore = ignore_index;
        a.K = (int)topk;
        a.temperature = temperature;
        a.part = part.data_ptr<float>();
        a.logprobs = logprobs.data_ptr<float>();
        a.entropy = entropy.data_ptr<float>();
        a.top_lp = top_lp.data_ptr<float>();
        a.top_ids = top_ids.data_ptr<int64_t>();
        a.stat = stat.data_ptr<float>();
        logprobs_fwd_launch(&g, &a, dt, cur_stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return {logprobs, entropy, top_lp, top_ids, stat};
}

torch::Tensor token_logprobs_bwd(
    torch::Tensor logits, c10::optional<torch::Tensor> tokens,
    torch::Tensor top_ids, torch::Tensor stat,
    c10::optional<torch::Tensor> d_logprobs,
    c10::optional<torch::Tensor> d_entropy, c10::optional<torch::Tensor> d_top,
    double temperature, int64_t ignore_index) {
    c10::OptionalDeviceGuard guard(logits.device());
    VocabRows g = vocab_rows_or_copy(logits);
    const int64_t K = top_ids.size(-1);
    TORCH_CHECK(K <= VOCAB_MAX_K, "topk");
    CHECK_ROWS(stat, torch::kFloat32, g.rows * 4ll);
    CHECK_ROWS(top_ids, torch::kInt64, g.rows * K);
    VocabGrad a = {};
    if (tokens) {
        CHECK_ROWS(*tokens, torch::kInt64, g.rows);
        a.tokens = tokens->data_ptr<int64_t>();
    }
    if (d_logprobs) {
        CHECK_ROWS(*d_logprobs, torch::kFloat32, g.rows);
        a.d_row = d_logprobs->data_ptr<float>();
    }
    if (d_entropy) {
        CHECK_ROWS(*d_entropy, torch::kFloat32, g.rows);
        a.d_entropy = d_entropy->data_ptr<float>();
    }
    if (d_top) {
        CHECK_ROWS(*d_top, torch::kFloat32, g.rows * K);
        a.d_top = d_top->data_ptr<float>();
    }
    a.stat = stat.data_ptr<float>();
    a.c = (float)(1.4426950408889634 / temperature);
    a.inv_t = (float)(1. / temperature);
    a.K = (int)K;
    a.ids = top_ids.data_ptr<int64_t>();
    a.ignore = ignore_index;
    auto out = new_tensor(logits.sizes(), logits.scalar_type(), logits);
    if (g.rows > 0) {
        vocab_grad_launch(&g, &a, 0, out.data_ptr(), vocab_dtype(logits),
                          cur_stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return out;
}

// -> loss, entry, stat
std::vector<torch::Tensor> topk_distillation_fwd(torch::Tensor logits,
                                                 torch::Tensor teacher_logprobs,
                                                 torch::Tensor teacher_ids,
                                                 double temperature,
                                                 bool bucket) {
    c10::OptionalDeviceGuard guard(logits.device());
    VocabRows g = vocab_rows_or_copy(logits);
    const int64_t K = teacher_ids.size(-1);
    TORCH_CHECK(K >= 1 && K <= VOCAB_MAX_K, "entries per row");
    TORCH_CHECK(temperature > 0, "temperature");
    CHECK_ROWS(teacher_ids, torch::kInt64, g.rows * K);
    CHECK_ROWS(teacher_logprobs, torch::kFloat32, g.rows * K);
    const auto f32 = torch::kFloat32;
    auto loss = new_tensor(lead_sizes(logits), f32, logits);
    auto entry = new_tensor({g.rows, K, 2}, torch::kInt32, logits);
    auto stat = new_tensor({g.rows, 4}, f32, logits);
    if (g.rows > 0) {
        auto part = new_tensor({g.rows, g.nseg, 4}, f32, logits);
        VocabDistill a;
        a.teacher_lp = teacher_logprobs.data_ptr<float>();
        a.ids = teacher_ids.data_ptr<int64_t>();
        a.K = (int)K;
        a.bucket = bucket ? 1 : 0;
        a.temperature = temperature;
        a.part = part.data_ptr<float>();
        a.loss = loss.data_ptr<float>();
        a.entry = entry.data_ptr<int>();
        a.stat = stat.data_ptr<float>();
        distill_fwd_launch(&g, &a, vocab_dtype(logits), cur_stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return {loss, entry, stat};
}

torch::Tensor topk_distillation_bwd(torch::Tensor dloss, torch::Tensor logits,
                                    torch::Tensor entry, torch::Tensor stat,
                                    double temperature) {
    c10::OptionalDeviceGuard guard(logits.device());
    VocabRows g = vocab_rows_or_copy(logits);
    TORCH_CHECK(entry.dim() == 3, "entry must be [rows, K, 2]");
    const int64_t K = entry.size(1);
    TORCH_CHECK(K >= 1 && K <= VOCAB_MAX_K, "entries per row");
    CHECK_ROWS(dloss, torch::kFloat32, g.rows);
    CHECK_ROWS(entry, torch::kInt32, g.rows * K * 2);
    CHECK_ROWS(stat, torch::kFloat32, g.rows * 4ll);
    VocabGrad a = {};
    a.stat = stat.data_ptr<float>();
    a.c = (float)(1.4426950408889634 / temperature);
    a.inv_t = (float)(1. / temperature);
    a.K = (int)K;
    a.d_row = dloss.data_ptr<float>();
    a.entry = entry.data_ptr<int>();
    auto out = new_tensor(logits.sizes(), logits.scalar_type(), logits);
    if (g.rows > 0) {
        vocab_grad_launch(&g, &a, 1, out.data_ptr(), vocab_dtype(logits),
                          cur_stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return out;
}

// ---- the same as differentiable operators, without Python on the way ----
// As under once_differentiable: a gradient of the gradient raises when it is
// asked for.
static torch::autograd::variable_list differentiable_once(
    torch::autograd::variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    auto tensor = grads[0];
    tensor = tensor.detach().requires_grad_(true);
    auto raises = std::make_shared<torch::autograd::DelayedError>(
        "this operator is differentiable once", 1);
    grads[0] = (*raises)({tensor})[0];
    return grads;
}

static c10::optional<torch::Tensor> defined_or_none(const torch::Tensor &t,
                                                    bool wanted = true) {
    if (!wanted || !t.defined()) return c10::nullopt;
    return t.contiguous();
}

struct TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
    static torch::autograd::variable_list forward(
        torch::autograd::AutogradContext *ctx, const torch::Tensor &logits,
        const c10::optional<torch::Tensor> &tokens, int64_t topk,
        double temperature, int64_t ignore_index) {
        auto o = token_logprobs_fwd(logits, tokens, topk, temperature,
                                    ignore_index);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward(
            {logits, tokens ? *tokens : torch::Tensor(), o[3], o[4]});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["ignore_index"] = ignore_index;
        ctx->mark_non_differentiable({o[3]});
        return {o[0], o[1], o[2], o[3]};
    }
    static torch::autograd::variable_list backward(
        torch::autograd::AutogradContext *ctx,
        torch::autograd::variable_list d) {
        const auto saved = ctx->get_saved_variables();
        const auto tokens = defined_or_none(saved[1]);
        auto grad = token_logprobs_bwd(
            saved[0], tokens, saved[2], saved[3],
            defined_or_none(d[0], tokens.has_value()), defined_or_none(d[1]),
            defined_or_none(d[2], saved[2].size(-1) > 0),
            ctx->saved_data["temperature"].toDouble(),
            ctx->saved_data["ignore_index"].toInt());
        return differentiable_once({grad, {}, {}, {}, {}});
    }
};

struct TopkDistillation : public torch::autograd::Function<TopkDistillation> {
    static torch::Tensor forward(torch::autograd::AutogradContext *ctx,
                                 const torch::Tensor &logits,
                                 const torch::Tensor &teacher_logprobs,
                                 const torch::Tensor &teacher_ids,
                                 double temperature, bool bucket) {
        auto o = topk_distillation_fwd(logits, teacher_logprobs, teacher_ids,
                                       temperature, bucket);
        ctx->save_for_backward({logits, o[1], o[2]});
        ctx->saved_data["temperature"] = temperature;
        return o[0];
    }
    static torch::autograd::variable_list backward(
        torch::autograd::AutogradContext *ctx,
        torch::autograd::variable_list d) {
        const auto saved = ctx->get_saved_variables();
        auto grad = topk_distillation_bwd(
            d[0].contiguous(), saved[0], saved[1], saved[2],
            ctx->saved_data["temperature"].toDouble());
        return differentiable_once({grad, {}, {}, {}, {}});
    }
};

std::vector<torch::Tensor> token_logprobs(torch::Tensor logits,
                                          c10::optional<torch::Tensor> tokens,
                                          int64_t topk, double temperature,
                                          int64_t ignore_index) {
    return TokenLogprobs::apply(logits, tokens, topk, temperature,
                                ignore_index);
}

torch::Tensor topk_distillation(torch::Tensor logits,
                                torch::Tensor teacher_logprobs,
                                torch::Tensor teacher_ids, double temperature,
                                bool bucket) {
    return TopkDistillation::apply(logits, teacher_logprobs, teacher_ids,
                                   temperature, bucket);
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("fp8_cast", &fp8_cast,
          "fused bf16->fp8 cast + running amax (delayed scaling)");
    m.def("fp8_cast_t", &fp8_cast_t,
          "fused bf16->fp8 cast + transpose + running amax");
    m.def("wgrad_accum", &wgrad_accum,
          "main_grad(fp32) += dout^T @ x (bf16 in, hipBLAS GemmEx)");
    m.def("mfma_probe", &mfma_probe, "16x16x32 bf16 fragment-layout probe");
    m.def("fa_fwd", &fa_fwd, "flash attention forward (gfx950 MFMA)");
    m.def("fa_bwd", &fa_bwd, "flash attention backward (gfx950 MFMA)");
    m.def("rmsnorm_fwd", &rmsnorm_fwd, "fused RMSNorm forward (gfx950)");
    m.def("rmsnorm_bwd", &rmsnorm_bwd, "fused RMSNorm backward (gfx950)");
    m.def("rope", &rope, "fused RoPE (sign=+1 fwd, -1 bwd) (gfx950)");
    m.def("swiglu_fwd", &swiglu_fwd, "fused SwiGLU forward (gfx950)");
    m.def("swiglu_bwd", &swiglu_bwd, "fused SwiGLU backward (gfx950)");
    m.def("ce_fwd", &ce_fwd, "fused cross-entropy forward (gfx950)");
    m.def("ce_bwd", &ce_bwd, "fused cross-entropy backward (gfx950)");
    m.def("grouped_fwd", &grouped_fwd,
          "grouped expert GEMM fwd: [E,M,K]x[E,N,K]^T -> [E,M,N] (MFMA)");
    m.def("grouped_dgrad", &grouped_dgrad,
          "grouped expert GEMM dgrad: [E,M,N]x[E,N,K] -> [E,M,K] (MFMA)");
    m.def("grouped_wgrad", &grouped_wgrad,
          "grouped expert wgrad: fp32 G[E,N,K] += dout^T @ x (MFMA)");
    m.def("token_logprobs", &token_logprobs,
          "token_logprobs_fwd with its gradient (gfx950)");
    m.def("topk_distillation", &topk_distillation,
          "topk_distillation_fwd with its gradient (gfx950)");
    m.def("token_logprobs_fwd", &token_logprobs_fwd,
          "log probabilities, entropy, top alternatives of logits (gfx950)");
    m.def("token_logprobs_bwd", &token_logprobs_bwd,
          "gradient of token_logprobs_fwd (gfx950)");
    m.def("topk_distillation_fwd", &topk_distillation_fwd,
          "divergence from a teacher's top log probabilities (gfx950)");
    m.def("topk_distillation_bwd", &topk_distillation_bwd,
          "gradient of topk_distillation_fwd (gfx950)");
}
