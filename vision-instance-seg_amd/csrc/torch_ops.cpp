// torch.ops.visionseg.* -- the operator surface of SURVEY §8(b) registered with
// TORCH_LIBRARY over the C ABI of libvisionseg_hip.so (include/visionseg.h).
//
// Contract (§8(b) "Operator C-ABI"): ATen tensors in, outputs allocated here through the
// caching allocator (the caller owns them), launches on the current HIP stream of the
// inputs' device, errors raised with TORCH_CHECK (-> Python RuntimeError), no host sync
// inside an op (msda_*: spatial_shapes / level_start_index are read on the host; pass CPU
// int64 tensors -- a device tensor costs one device->host copy, as the upstream extension's
// callers do with `.tolist()`), no global state.  The autograd wrappers stay in Python
// (visionseg/ops.py), as the upstream `MSDeformAttnFunction` wraps its extension, but for those of
// the 8-bit activation checkpoints (below: host time).
// There is no CPU kernel: a CPU tensor is refused (no fallback path exists).
//
// Host-only C++ (g++), linked against libvisionseg_hip.so; the kernels live in csrc/*.hip.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <vector>

#include "../../include/visionseg.h"

namespace {

void vs_ok(int rc, const char* what) {
  TORCH_CHECK(rc == VS_OK, "visionseg ", what, " failed (status ", rc, "): ", vs_last_error());
}

void* cur_stream(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int dcode(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return VS_F32;
  if (t.scalar_type() == at::kBFloat16) return VS_BF16;
  TORCH_CHECK(false, "visionseg kernels take float32 or bfloat16 activations, got ", t.scalar_type());
  return -1;
}

void on_device(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK(t->is_cuda(), "visionseg ops run only on a HIP device (no CPU fallback); got a tensor on ",
                t->device());
}

int as_int(int64_t v, const char* what) {
  TORCH_CHECK(v >= 0 && v <= INT32_MAX, what, " out of range: ", v);
  return (int)v;
}

// spatial_shapes [L, 2] / level_start_index [L] int64 -> host vectors (the C ABI reads them
// on the host: they size the launch)
std::vector<int64_t> host_i64(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kLong, what, " must be int64");
  at::Tensor h = t.device().is_cpu() ? t.contiguous() : t.to(at::kCPU).contiguous();
  return std::vector<int64_t>(h.data_ptr<int64_t>(), h.data_ptr<int64_t>() + h.numel());
}

// ---- a8: MSDeformAttn sampling (upstream MultiScaleDeformableAttention.ms_deform_attn_*)
struct MsdaDims {
  int64_t B, S, H, D, Q, L, P;
};

// one shape check for both directions: value [B, S, heads, 32], sampling_loc [B, Q, heads, L,
// P, 2] f32, attn_weight [B, Q, heads, L, P] f32, L levels of shapes / starts
MsdaDims check_msda(const at::Tensor& value, const std::vector<int64_t>& sh, const std::vector<int64_t>& st,
                    const at::Tensor& loc, const at::Tensor& aw) {
  TORCH_CHECK(value.dim() == 4, "value must be [B, S, heads, 32]");
  TORCH_CHECK(loc.dim() == 6 && loc.size(5) == 2, "sampling_loc must be [B, Q, heads, L, P, 2]");
  TORCH_CHECK(loc.scalar_type() == at::kFloat && aw.scalar_type() == at::kFloat,
              "sampling_loc / attn_weight must be float32");
  MsdaDims d{value.size(0), value.size(1), value.size(2), value.size(3), loc.size(1), loc.size(3), loc.size(4)};
  TORCH_CHECK((int64_t)sh.size() == 2 * d.L && (int64_t)st.size() == d.L,
              "spatial_shapes / level_start_index do not have ", d.L, " levels");
  TORCH_CHECK(loc.size(0) == d.B && loc.size(2) == d.H, "sampling_loc batch/heads do not match value");
  TORCH_CHECK(aw.sizes() == at::IntArrayRef({d.B, d.Q, d.H, d.L, d.P}), "attn_weight must be [B, Q, heads, L, P]");
  return d;
}

at::Tensor msda_fwd(const at::Tensor& value, const at::Tensor& spatial_shapes, const at::Tensor& level_start_index,
                    const at::Tensor& sampling_loc, const at::Tensor& attn_weight, int64_t im2col_step) {
  (void)im2col_step;  // the kernel tiles by query groups, not im2col steps
  on_device({&value, &sampling_loc, &attn_weight});
  const auto sh = host_i64(spatial_shapes, "spatial_shapes");
  const auto st = host_i64(level_start_index, "level_start_index");
  at::Tensor v = value.contiguous(), loc = sampling_loc.contiguous(), aw = attn_weight.contiguous();
  const MsdaDims d = check_msda(v, sh, st, loc, aw);
  at::Tensor out = at::empty({d.B, d.Q, d.H * d.D}, v.options());
  vs_ok(vs_msda_forward(dcode(v), v.data_ptr(), sh.data(), st.data(), loc.data_ptr<float>(), aw.data_ptr<float>(),
                        out.data_ptr(), as_int(d.B, "batch"), as_int(d.S, "S"), as_int(d.H, "heads"),
                        as_int(d.D, "channels"), as_int(d.L, "levels"), as_int(d.Q, "queries"), as_int(d.P, "points"),
                        cur_stream(v)),
        "msda_fwd");
  return out;
}

// -> (grad_value in value's dtype -- or the f32 accumulator itself with f32_grad_value --,
//     grad_sampling_loc f32, grad_attn_weight f32)
std::tuple<at::Tensor, at::Tensor, at::Tensor> msda_bwd(const at::Tensor& value, const at::Tensor& spatial_shapes,
                                                        const at::Tensor& level_start_index,
                                                        const at::Tensor& sampling_loc, const at::Tensor& attn_weight,
                                                        const at::Tensor& grad_output, int64_t im2col_step,
                                                        bool f32_grad_value) {
  (void)im2col_step;
  on_device({&value, &sampling_loc, &attn_weight, &grad_output});
  const auto sh = host_i64(spatial_shapes, "spatial_shapes");
  const auto st = host_i64(level_start_index, "level_start_index");
  at::Tensor v = value.contiguous(), loc = sampling_loc.contiguous(), aw = attn_weight.contiguous();
  const MsdaDims d = check_msda(v, sh, st, loc, aw);
  TORCH_CHECK(grad_output.numel() == d.B * d.Q * d.H * d.D && grad_output.dim() >= 2 && grad_output.size(0) == d.B &&
                  grad_output.size(1) == d.Q,
              "grad_output must be [B, Q, heads*32]");
  at::Tensor g = grad_output.to(v.scalar_type()).contiguous();
  // grad_value accumulates in f32 (float atomics), then takes value's dtype
  at::Tensor gv = at::empty({d.B, d.S, d.H, d.D}, v.options().dtype(at::kFloat));
  at::Tensor gl = at::empty_like(loc), ga = at::empty_like(aw);
  // workspace: reserved by the C ABI (0 bytes since round 6; csrc/msda.hip)
  const long long wsb = vs_msda_backward_workspace_bytes(as_int(d.B, "batch"), as_int(d.Q, "queries"),
                                                         as_int(d.H, "heads"), as_int(d.L, "levels"),
                                                         as_int(d.P, "points"));
  TORCH_CHECK(wsb >= 0, "msda_bwd: bad sizes");
  at::Tensor ws = at::empty({wsb}, v.options().dtype(at::kByte));
  vs_ok(vs_msda_backward_ex(dcode(v), v.data_ptr(), sh.data(), st.data(), loc.data_ptr<float>(),
                            aw.data_ptr<float>(), g.data_ptr(), gv.data_ptr<float>(), gl.data_ptr<float>(),
                            ga.data_ptr<float>(), ws.data_ptr(), as_int(d.B, "batch"), as_int(d.S, "S"),
                            as_int(d.H, "heads"), as_int(d.D, "channels"), as_int(d.L, "levels"),
                            as_int(d.Q, "queries"), as_int(d.P, "points"), cur_stream(v)),
        "msda_bwd");
  return {(v.scalar_type() == at::kFloat || f32_grad_value) ? gv : gv.to(v.scalar_type()), gl, ga};
}

// ---- a2: pad + roll + window partition (and its exact inverse)
int64_t padded(int64_t n, int64_t ws) { return n + (ws - n % ws) % ws; }

at::Tensor swin_window_fwd(const at::Tensor& x, int64_t window, int64_t shift) {
  on_device({&x});
  TORCH_CHECK(x.dim() == 4, "x must be [B, H, W, C]");
  TORCH_CHECK(window > 0 && shift >= 0 && shift < window, "bad window / shift");
  at::Tensor xc = x.contiguous();
  const int64_t B = xc.size(0), H = xc.size(1), W = xc.size(2), C = xc.size(3);
  const int64_t nw = (padded(H, window) / window) * (padded(W, window) / window);
  at::Tensor out = at::empty({B * nw, window * window, C}, xc.options());
  vs_ok(vs_window_partition(xc.data_ptr(), out.data_ptr(), (int)xc.element_size(), as_int(B, "batch"),
                            as_int(H, "height"), as_int(W, "width"), as_int(C, "channels"), (int)window, (int)shift,
                            cur_stream(xc)),
        "swin_window_fwd");
  return out;
}

at::Tensor swin_window_bwd(const at::Tensor& windows, int64_t batch, int64_t height, int64_t width, int64_t window,
                           int64_t shift) {
  on_device({&windows});
  TORCH_CHECK(windows.dim() == 3 && windows.size(1) == window * window, "windows must be [B*nW, window^2, C]");
  const int64_t nw = (padded(height, window) / window) * (padded(width, window) / window);
  TORCH_CHECK(windows.size(0) == batch * nw, "windows hold ", windows.size(0), " windows, expected ", batch * nw);
  at::Tensor wc = windows.contiguous();
  const int64_t C = wc.size(2);
  at::Tensor out = at::empty({batch, height, width, C}, wc.options());
  vs_ok(vs_window_reverse(wc.data_ptr(), out.data_ptr(), (int)wc.element_size(), as_int(batch, "batch"),
                          as_int(height, "height"), as_int(width, "width"), as_int(C, "channels"), (int)window,
                          (int)shift, cur_stream(wc)),
        "swin_window_bwd");
  return out;
}

// ---- a3/a4/a5: window attention core (qkv = the fused q;k;v Linear output per window)
void check_qkv(const at::Tensor& qkv, int64_t heads, int64_t window) {
  TORCH_CHECK(qkv.dim() == 3 && qkv.size(1) == window * window && qkv.size(2) == 3 * heads * 32,
              "qkv must be [B*nW, window^2, 3*heads*32]");
}

std::tuple<at::Tensor, at::Tensor> win_attn_fwd(const at::Tensor& qkv, const at::Tensor& rel_table, int64_t heads,
                                                int64_t window, int64_t shift, int64_t nwin_h, int64_t nwin_w,
                                                double scale, bool fp8) {
  on_device({&qkv, &rel_table});
  check_qkv(qkv, heads, window);
  at::Tensor q = qkv.contiguous(), table = rel_table.to(at::kFloat).contiguous();
  TORCH_CHECK(table.numel() == (2 * window - 1) * (2 * window - 1) * heads, "rel_table must be [(2ws-1)^2, heads]");
  const int64_t Bw = q.size(0), N = q.size(1);
  at::Tensor out = at::empty({Bw, N, heads * 32}, q.options());
  at::Tensor lse = at::empty({Bw, heads, N}, q.options().dtype(at::kFloat));
  if (fp8) {
    TORCH_CHECK(q.scalar_type() == at::kBFloat16 && N <= 160, "fp8 window attention needs bf16 qkv and window^2 <= 160");
    vs_ok(vs_window_attn_forward_fp8(q.data_ptr(), table.data_ptr<float>(), out.data_ptr(), lse.data_ptr<float>(),
                                     as_int(Bw, "windows"), (int)heads, (int)window, (int)shift, (int)nwin_h,
                                     (int)nwin_w, (float)scale, cur_stream(q)),
          "win_attn_fwd (fp8)");
  } else {
    vs_ok(vs_window_attn_forward(dcode(q), q.data_ptr(), table.data_ptr<float>(), out.data_ptr(),
                                 lse.data_ptr<float>(), as_int(Bw, "windows"), (int)heads, (int)window, (int)shift,
                                 (int)nwin_h, (int)nwin_w, (float)scale, cur_stream(q)),
          "win_attn_fwd");
  }
  return {out, lse};
}

// -> (grad_qkv, grad_rel_table [(2ws-1)^2, heads] f32)
std::tuple<at::Tensor, at::Tensor> win_attn_bwd(const at::Tensor& qkv, const at::Tensor& rel_table,
                                                const at::Tensor& out, const at::Tensor& lse,
                                                const at::Tensor& grad_out, int64_t heads, int64_t window,
                                                int64_t shift, int64_t nwin_h, int64_t nwin_w, double scale,
                                                bool fp8, bool table_partials) {
  on_device({&qkv, &rel_table, &out, &lse, &grad_out});
  check_qkv(qkv, heads, window);
  at::Tensor q = qkv.contiguous(), table = rel_table.to(at::kFloat).contiguous();
  at::Tensor o = out.contiguous(), l = lse.contiguous(), g = grad_out.to(q.scalar_type()).contiguous();
  const int64_t Bw = q.size(0), N = q.size(1), T2 = (2 * window - 1) * (2 * window - 1);
  TORCH_CHECK(o.sizes() == at::IntArrayRef({Bw, N, heads * 32}) && g.sizes() == o.sizes(),
              "out / grad_out must be [B*nW, window^2, heads*32]");
  TORCH_CHECK(l.scalar_type() == at::kFloat && l.sizes() == at::IntArrayRef({Bw, heads, N}),
              "lse must be float32 [B*nW, heads, window^2]");
  TORCH_CHECK(table.numel() == T2 * heads, "rel_table must be [(2ws-1)^2, heads]");
  at::Tensor gqkv = at::empty_like(q);
  at::Tensor part = at::empty({Bw, heads, T2}, q.options().dtype(at::kFloat));
  if (fp8) {
    vs_ok(vs_window_attn_backward_fp8(q.data_ptr(), table.data_ptr<float>(), o.data_ptr(), l.data_ptr<float>(),
                                      g.data_ptr(), gqkv.data_ptr(), part.data_ptr<float>(), as_int(Bw, "windows"),
                                      (int)heads, (int)window, (int)shift, (int)nwin_h, (int)nwin_w, (float)scale,
                                      cur_stream(q)),
          "win_attn_bwd (fp8)");
  } else {
    vs_ok(vs_window_attn_backward(dcode(q), q.data_ptr(), table.data_ptr<float>(), o.data_ptr(), l.data_ptr<float>(),
                                  g.data_ptr(), gqkv.data_ptr(), part.data_ptr<float>(), as_int(Bw, "windows"),
                                  (int)heads, (int)window, (int)shift, (int)nwin_h, (int)nwin_w, (float)scale,
                                  cur_stream(q)),
          "win_attn_bwd");
  }
  // per-window partial bias gradients summed in a fixed order (deterministic); or the
  // partials themselves [Bw, heads, (2ws-1)^2] (table_partials)
  if (table_partials) return {gqkv, part};
  return {gqkv, part.sum(0).t().contiguous()};
}

// image-layout window attention (the window reverse folded in): out / grad_out
// [B, height, width, heads*32]; qkv, lse, grad_qkv in the window layout
std::tuple<at::Tensor, at::Tensor> win_attn_fwd_img(const at::Tensor& qkv, const at::Tensor& rel_table, int64_t heads,
                                                    int64_t window, int64_t shift, int64_t nwin_h, int64_t nwin_w,
                                                    int64_t height, int64_t width, double scale, bool fp8) {
  on_device({&qkv, &rel_table});
  check_qkv(qkv, heads, window);
  at::Tensor q = qkv.contiguous(), table = rel_table.to(at::kFloat).contiguous();
  TORCH_CHECK(table.numel() == (2 * window - 1) * (2 * window - 1) * heads, "rel_table must be [(2ws-1)^2, heads]");
  const int64_t Bw = q.size(0), N = q.size(1), nw = nwin_h * nwin_w;
  TORCH_CHECK(nw > 0 && Bw % nw == 0, "num_windows must be a multiple of nwin_h * nwin_w");
  at::Tensor out = at::empty({Bw / nw, height, width, heads * 32}, q.options());
  at::Tensor lse = at::empty({Bw, heads, N}, q.options().dtype(at::kFloat));
  vs_ok(vs_window_attn_forward_image(dcode(q), fp8 ? 1 : 0, q.data_ptr(), table.data_ptr<float>(), out.data_ptr(),
                                     lse.data_ptr<float>(), as_int(Bw, "windows"), (int)heads, (int)window,
                                     (int)shift, (int)nwin_h, (int)nwin_w, as_int(height, "height"),
                                     as_int(width, "width"), (float)scale, cur_stream(q)),
        "win_attn_fwd_img");
  return {out, lse};
}

// -> (grad_qkv [window layout], grad_rel_table partials [Bw, heads, (2ws-1)^2] f32)
std::tuple<at::Tensor, at::Tensor> win_attn_bwd_img(const at::Tensor& qkv, const at::Tensor& rel_table,
                                                    const at::Tensor& out, const at::Tensor& lse,
                                                    const at::Tensor& grad_out, int64_t heads, int64_t window,
                                                    int64_t shift, int64_t nwin_h, int64_t nwin_w, int64_t height,
                                                    int64_t width, double scale, bool fp8) {
  on_device({&qkv, &rel_table, &out, &lse, &grad_out});
  check_qkv(qkv, heads, window);
  at::Tensor q = qkv.contiguous(), table = rel_table.to(at::kFloat).contiguous();
  at::Tensor o = out.contiguous(), l = lse.contiguous(), g = grad_out.to(q.scalar_type()).contiguous();
  const int64_t Bw = q.size(0), N = q.size(1), T2 = (2 * window - 1) * (2 * window - 1), nw = nwin_h * nwin_w;
  TORCH_CHECK(nw > 0 && Bw % nw == 0, "num_windows must be a multiple of nwin_h * nwin_w");
  TORCH_CHECK(o.sizes() == at::IntArrayRef({Bw / nw, height, width, heads * 32}) && g.sizes() == o.sizes(),
              "out / grad_out must be [B, height, width, heads*32]");
  TORCH_CHECK(l.scalar_type() == at::kFloat && l.sizes() == at::IntArrayRef({Bw, heads, N}),
              "lse must be float32 [B*nW, heads, window^2]");
  TORCH_CHECK(table.numel() == T2 * heads, "rel_table must be [(2ws-1)^2, heads]");
  at::Tensor gqkv = at::empty_like(q);
  at::Tensor part = at::empty({Bw, heads, T2}, q.options().dtype(at::kFloat));
  vs_ok(vs_window_attn_backward_image(dcode(q), fp8 ? 1 : 0, q.data_ptr(), table.data_ptr<float>(), o.data_ptr(),
                                      l.data_ptr<float>(), g.data_ptr(), gqkv.data_ptr(), part.data_ptr<float>(),
                                      as_int(Bw, "windows"), (int)heads, (int)window, (int)shift, (int)nwin_h,
                                      (int)nwin_w, as_int(height, "height"), as_int(width, "width"), (float)scale,
                                      cur_stream(q)),
        "win_attn_bwd_img");
  return {gqkv, part};
}

// ---- a11: mask head einsum('bqc,bchw->bqhw') with channels-last pixel embedding
at::Tensor mask_head_fwd(const at::Tensor& mask_embed, const at::Tensor& pixel_nhwc, int64_t height, int64_t width) {
  on_device({&mask_embed, &pixel_nhwc});
  at::Tensor E = mask_embed.contiguous(), P = pixel_nhwc.to(E.scalar_type()).contiguous();
  TORCH_CHECK(E.dim() == 3, "mask_embed must be [B, Q, C]");
  const int64_t B = E.size(0), Q = E.size(1), C = E.size(2);
  TORCH_CHECK(P.numel() == B * height * width * C, "pixel embedding must be [B, H*W, C]");
  at::Tensor out = at::empty({B, Q, height, width}, E.options().dtype(at::kFloat));
  vs_ok(vs_mask_head_forward(dcode(E), E.data_ptr(), P.data_ptr(), out.data_ptr<float>(), as_int(B, "batch"),
                             as_int(Q, "queries"), as_int(C, "channels"), as_int(height, "height"),
                             as_int(width, "width"), cur_stream(E)),
        "mask_head_fwd");
  return out;
}

// bf16, C in {128, 256}: grad_E returned; grad_pixel [B, H*W, C] written (accumulate=False)
// or added to (accumulate=True) in place -- the decoder's 10 calls share one buffer.
// Query counts above the kernel's 128 run as chunks of 128 accumulating grad_pixel.
at::Tensor mask_head_bwd(const at::Tensor& grad_logits, const at::Tensor& mask_embed, const at::Tensor& pixel_nhwc,
                         at::Tensor& grad_pixel, bool accumulate) {
  on_device({&grad_logits, &mask_embed, &pixel_nhwc, &grad_pixel});
  at::Tensor E = mask_embed.contiguous(), P = pixel_nhwc.contiguous();
  TORCH_CHECK(E.scalar_type() == at::kBFloat16 && P.scalar_type() == at::kBFloat16, "mask_head_bwd is the bf16 path");
  const int64_t B = E.size(0), Q = E.size(1), C = E.size(2), N = P.numel() / (B * C);
  TORCH_CHECK(C == 128 || C == 256, "mask_head_bwd takes 128 or 256 channels");
  TORCH_CHECK(grad_pixel.is_contiguous() && grad_pixel.sizes() == P.sizes() &&
                  grad_pixel.scalar_type() == P.scalar_type(),
              "grad_pixel must be a contiguous tensor shaped and typed like pixel_nhwc");
  at::Tensor g = grad_logits.to(at::kFloat).contiguous();
  TORCH_CHECK(g.numel() == B * Q * N, "grad_logits must be [B, Q, H, W]");
  at::Tensor gE = at::empty_like(E);
  bool acc = accumulate;
  for (int64_t q0 = 0; q0 < Q; q0 += 128) {
    const int64_t q1 = std::min(Q, q0 + 128), nq = q1 - q0;
    const bool whole = q0 == 0 && q1 == Q;
    at::Tensor gc = whole ? g : g.view({B, Q, N}).slice(1, q0, q1).contiguous();
    at::Tensor Ec = whole ? E : E.slice(1, q0, q1).contiguous();
    at::Tensor gEc = whole ? gE : at::empty_like(Ec);
    at::Tensor ws = at::empty({vs_mask_head_backward_workspace_bytes((int)B, (int)nq, (int)C)},
                              E.options().dtype(at::kByte));
    vs_ok(vs_mask_head_backward_ex(dcode(E), gc.data_ptr<float>(), Ec.data_ptr(), P.data_ptr(), gEc.data_ptr(),
                                   grad_pixel.data_ptr(), ws.data_ptr(), (int)B, (int)nq, (int)C, (int)N, 1, (int)acc,
                                   cur_stream(E)),
          "mask_head_bwd");
    if (!whole) gE.slice(1, q0, q1).copy_(gEc);
    acc = true;
  }
  return gE;
}

// next layer's blocked-key bitmask from mask logits (HF:m2f:2049-2055, row fix 1912-1914)
at::Tensor attn_bitmask(const at::Tensor& logits, int64_t target_h, int64_t target_w) {
  on_device({&logits});
  at::Tensor lg = logits.to(at::kFloat).contiguous();
  TORCH_CHECK(lg.dim() == 4, "logits must be [B, Q, H, W]");
  const int64_t B = lg.size(0), Q = lg.size(1);
  at::Tensor words = at::empty({B, Q, (target_h * target_w + 31) / 32}, lg.options().dtype(at::kInt));
  vs_ok(vs_attn_bitmask(lg.data_ptr<float>(), (uint32_t*)words.data_ptr(), as_int(B * Q, "rows"),
                        (int)lg.size(2), (int)lg.size(3), as_int(target_h, "target_h"), as_int(target_w, "target_w"),
                        cur_stream(lg)),
        "attn_bitmask");
  return words;
}

// ---- a10: masked cross-attention core
void check_xattn(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& words,
                 int64_t heads) {
  TORCH_CHECK(q.dim() == 3 && q.size(2) == heads * 32, "q must be [B, Q, heads*32]");
  TORCH_CHECK(k.sizes() == v.sizes() && k.dim() == 3 && k.size(0) == q.size(0) && k.size(2) == q.size(2),
              "k / v must be [B, S, heads*32]");
  TORCH_CHECK(words.sizes() == at::IntArrayRef({q.size(0), q.size(1), (k.size(1) + 31) / 32}),
              "bitmask does not cover the keys");
}

std::tuple<at::Tensor, at::Tensor> masked_xattn_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                    const at::Tensor& words, int64_t heads, double scale) {
  on_device({&q, &k, &v, &words});
  check_xattn(q, k, v, words, heads);
  at::Tensor qc = q.contiguous(), kc = k.to(q.scalar_type()).contiguous(), vc = v.to(q.scalar_type()).contiguous();
  at::Tensor wc = words.contiguous();
  const int B = as_int(q.size(0), "batch"), Q = as_int(q.size(1), "queries"), S = as_int(k.size(1), "keys");
  at::Tensor out = at::empty_like(qc);
  at::Tensor lse = at::empty({B, heads, Q}, qc.options().dtype(at::kFloat));
  at::Tensor ws = at::empty({vs_masked_attn_workspace_bytes(B, Q, S, (int)heads)}, qc.options().dtype(at::kByte));
  vs_ok(vs_masked_attn_forward(dcode(qc), qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), (const uint32_t*)wc.data_ptr(),
                               out.data_ptr(), lse.data_ptr<float>(), ws.data_ptr(), B, Q, S, (int)heads,
                               (float)scale, cur_stream(qc)),
        "masked_xattn_fwd");
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> masked_xattn_bwd(const at::Tensor& q, const at::Tensor& k,
                                                                const at::Tensor& v, const at::Tensor& words,
                                                                const at::Tensor& out, const at::Tensor& lse,
                                                                const at::Tensor& grad_out, int64_t heads,
                                                                double scale) {
  on_device({&q, &k, &v, &words, &out, &lse, &grad_out});
  check_xattn(q, k, v, words, heads);
  at::Tensor qc = q.contiguous(), kc = k.contiguous(), vc = v.contiguous(), wc = words.contiguous();
  at::Tensor oc = out.contiguous(), lc = lse.contiguous(), g = grad_out.to(q.scalar_type()).contiguous();
  TORCH_CHECK(kc.scalar_type() == qc.scalar_type() && vc.scalar_type() == qc.scalar_type(), "q / k / v dtypes differ");
  const int B = as_int(q.size(0), "batch"), Q = as_int(q.size(1), "queries"), S = as_int(k.size(1), "keys");
  TORCH_CHECK(oc.sizes() == qc.sizes() && g.sizes() == qc.sizes(), "out / grad_out must be shaped like q");
  TORCH_CHECK(lc.scalar_type() == at::kFloat && lc.sizes() == at::IntArrayRef({(int64_t)B, heads, (int64_t)Q}),
              "lse must be float32 [B, heads, Q]");
  at::Tensor gq = at::empty_like(qc), gk = at::empty_like(kc), gv = at::empty_like(vc);
  at::Tensor ws = at::empty({vs_masked_attn_workspace_bytes(B, Q, S, (int)heads)}, qc.options().dtype(at::kByte));
  vs_ok(vs_masked_attn_backward(dcode(qc), qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), (const uint32_t*)wc.data_ptr(),
                                oc.data_ptr(), lc.data_ptr<float>(), g.data_ptr(), gq.data_ptr(), gk.data_ptr(),
                                gv.data_ptr(), ws.data_ptr(), B, Q, S, (int)heads, (float)scale, cur_stream(qc)),
        "masked_xattn_bwd");
  return {gq, gk, gv};
}


// ---- a10: decoder self-attention core (words: an empty tensor = no mask, [Q, nw] shared by the
// batch, or [B, Q, nw])
long long self_attn_words(const at::Tensor& words, int B, int Q, int S) {
  if (words.numel() == 0) return -1;
  const int64_t nw = (S + 31) / 32;
  TORCH_CHECK(words.scalar_type() == at::kInt && words.is_contiguous(), "words must be contiguous int32");
  if (words.dim() == 2) {
    TORCH_CHECK(words.sizes() == at::IntArrayRef({(int64_t)Q, nw}), "words must be [Q, ceil(S/32)]");
    return 0;
  }
  TORCH_CHECK(words.sizes() == at::IntArrayRef({(int64_t)B, (int64_t)Q, nw}), "words must be [B, Q, ceil(S/32)]");
  return (long long)Q * nw;
}

void check_self_attn(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t heads) {
  TORCH_CHECK(q.dim() == 3 && q.size(2) == heads * 32, "q must be [B, Q, heads*32]");
  TORCH_CHECK(k.sizes() == v.sizes() && k.dim() == 3 && k.size(0) == q.size(0) && k.size(2) == q.size(2),
              "k / v must be [B, S, heads*32]");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16,
              "self_attn takes bf16 q / k / v");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> self_attn_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                 const at::Tensor& words, int64_t heads, double scale) {
  on_device({&q, &k, &v});
  check_self_attn(q, k, v, heads);
  at::Tensor qc = q.contiguous(), kc = k.contiguous(), vc = v.contiguous();
  const int B = as_int(q.size(0), "batch"), Q = as_int(q.size(1), "queries"), S = as_int(k.size(1), "keys");
  const long long wbs = self_attn_words(words, B, Q, S);
  if (wbs >= 0) on_device({&words});
  at::Tensor out = at::empty_like(qc);
  at::Tensor out32 = at::empty(qc.sizes(), qc.options().dtype(at::kFloat));
  at::Tensor lse = at::empty({B, heads, Q}, qc.options().dtype(at::kFloat));
  vs_ok(vs_self_attn_forward(VS_BF16, qc.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                             wbs >= 0 ? (const uint32_t*)words.data_ptr() : nullptr, wbs >= 0 ? wbs : 0,
                             out.data_ptr(), out32.data_ptr<float>(), lse.data_ptr<float>(), B, Q, S, (int)heads,
                             (float)scale, cur_stream(qc)),
        "self_attn_fwd");
  return {out, out32, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> self_attn_bwd(const at::Tensor& q, const at::Tensor& k,
                                                             const at::Tensor& v, const at::Tensor& words,
                                                             const at::Tensor& out, const at::Tensor& lse,
                                                             const at::Tensor& grad_out, int64_t heads, double scale) {
  on_device({&q, &k, &v, &out, &lse, &grad_out});
  check_self_attn(q, k, v, heads);
  at::Tensor qc = q.contiguous(), kc = k.contiguous(), vc = v.contiguous();
  at::Tensor oc = out.contiguous(), lc = lse.contiguous(), g = grad_out.to(at::kBFloat16).contiguous();
  const int B = as_int(q.size(0), "batch"), Q = as_int(q.size(1), "queries"), S = as_int(k.size(1), "keys");
  TORCH_CHECK(oc.sizes() == qc.sizes() && g.sizes() == qc.sizes() && oc.scalar_type() == at::kFloat,
              "out (the forward's f32 copy) / grad_out must be shaped like q");
  TORCH_CHECK(lc.scalar_type() == at::kFloat && lc.sizes() == at::IntArrayRef({(int64_t)B, heads, (int64_t)Q}),
              "lse must be float32 [B, heads, Q]");
  const long long wbs = self_attn_words(words, B, Q, S);
  if (wbs >= 0) on_device({&words});
  at::Tensor gq = at::empty_like(qc), gk = at::empty_like(kc), gv = at::empty_like(vc);
  vs_ok(vs_self_attn_backward(VS_BF16, qc.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                              wbs >= 0 ? (const uint32_t*)words.data_ptr() : nullptr, wbs >= 0 ? wbs : 0,
                              oc.data_ptr<float>(), lc.data_ptr<float>(), g.data_ptr(), gq.data_ptr(), gk.data_ptr(),
                              gv.data_ptr(), B, Q, S, (int)heads, (float)scale, cur_stream(qc)),
        "self_attn_bwd");
  return {gq, gk, gv};
}


// ---- 8-bit activation checkpoints (q int8 [..., P], scale uint8 [..., P / 32], P = the features
// rounded up to 32).  The outputs and workspaces are the caller's device's and stream's; the
// device guard makes a call on tensors of another device than the current one run there.
int64_t padded_features(int64_t C) { return (C + 31) / 32 * 32; }

void same_device(const at::Tensor& a, std::initializer_list<const at::Tensor*> ts) {
  on_device({&a});
  for (const at::Tensor* t : ts)
    TORCH_CHECK(t->device() == a.device(), "tensors on different devices: ", a.device(), " and ", t->device());
}

// No op here has a forward-mode derivative: a tangent is refused, not dropped.  (A C++ autograd
// Function refuses it by itself; a call that keeps nothing does not pass through one.)
void no_tangent(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK(!t->_fw_grad(0).defined(),
                "8-bit activation checkpoints: no forward-mode derivative (an input carries a tangent)");
}

// x as rows of its last dimension: unit feature stride, any row stride
at::Tensor as_rows(const at::Tensor& x, const char* what) {
  TORCH_CHECK(x.dim() >= 1, what, " must have at least one dimension");
  dcode(x);
  TORCH_CHECK(x.size(-1) <= (1 << 30), what, ": at most 2^30 features");
  if (x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1)) return x;
  const int64_t C = x.size(-1);
  at::Tensor r = x.contiguous().view({C ? x.numel() / C : 0, C});
  return r;
}

at::Tensor dense(const at::Tensor& x) { return x.contiguous(); }

at::Tensor new_q(const at::Tensor& x) {
  auto sz = x.sizes().vec();
  sz.back() = padded_features(sz.back());
  return at::empty(sz, x.options().dtype(at::kChar));
}
at::Tensor new_scale(const at::Tensor& x) {
  auto sz = x.sizes().vec();
  sz.back() = padded_features(sz.back()) / 32;
  return at::empty(sz, x.options().dtype(at::kByte));
}

// the checkpoint's tensors against the features it is said to have -> rows
int64_t check_checkpoint(const at::Tensor& q, const at::Tensor& scale, int64_t features) {
  same_device(q, {&scale});
  TORCH_CHECK(q.scalar_type() == at::kChar && scale.scalar_type() == at::kByte,
              "a checkpoint is q int8 and scale uint8, got ", q.scalar_type(), " and ", scale.scalar_type());
  TORCH_CHECK(features >= 0 && features <= (1 << 30), "features out of range: ", features);
  TORCH_CHECK(q.dim() >= 1 && scale.dim() == q.dim() && q.size(-1) == padded_features(features) &&
                  scale.size(-1) * 32 == q.size(-1) &&
                  q.sizes().slice(0, q.dim() - 1) == scale.sizes().slice(0, q.dim() - 1),
              "q ", q.sizes(), " and scale ", scale.sizes(), " are not a checkpoint of ", features, " features");
  return q.size(-1) ? q.numel() / q.size(-1) : 0;
}

std::tuple<at::Tensor, at::Tensor> act8_pack(const at::Tensor& x) {
  on_device({&x});
  const c10::DeviceGuard guard(x.device());
  at::Tensor r = as_rows(x, "x");
  at::Tensor q = new_q(x), scale = new_scale(x);
  vs_ok(vs_act8_pack(dcode(r), r.data_ptr(), r.stride(0), q.data_ptr(), scale.data_ptr(), r.size(0), (int)r.size(1),
                     cur_stream(r)),
        "act8_pack");
  return {q, scale};
}

at::Tensor act8_unpack(const at::Tensor& q, const at::Tensor& scale, int64_t features, at::ScalarType dtype) {
  on_device({&q});
  const int64_t rows = check_checkpoint(q, scale, features);
  const c10::DeviceGuard guard(q.device());
  auto sz = q.sizes().vec();
  sz.back() = features;
  at::Tensor qc = dense(q), sc = dense(scale), y = at::empty(sz, q.options().dtype(dtype));
  vs_ok(vs_act8_unpack(dcode(y), qc.data_ptr(), sc.data_ptr(), y.data_ptr(), rows, (int)features, cur_stream(qc)),
        "act8_unpack");
  return y;
}

// -> (gelu(x), q, scale); keep false: empty q, scale
std::tuple<at::Tensor, at::Tensor, at::Tensor> act8_gelu_fwd(const at::Tensor& x, bool keep) {
  no_tangent({&x});
  on_device({&x});
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
  const c10::DeviceGuard guard(x.device());
  at::Tensor xc = dense(x), y = at::empty_like(xc);
  at::Tensor q = keep ? new_q(xc) : at::empty({0}, xc.options().dtype(at::kChar));
  at::Tensor scale = keep ? new_scale(xc) : at::empty({0}, xc.options().dtype(at::kByte));
  const int64_t C = xc.size(-1);
  TORCH_CHECK(C <= (1 << 30), "x: at most 2^30 features");
  vs_ok(vs_act8_gelu_forward(dcode(xc), xc.data_ptr(), y.data_ptr(), keep ? q.data_ptr() : nullptr,
                             keep ? scale.data_ptr() : nullptr, C ? xc.numel() / C : 0, (int)C, cur_stream(xc)),
        "act8_gelu_fwd");
  return {y, q, scale};
}

// -> (gx, gelu(h) or an empty tensor)
std::tuple<at::Tensor, at::Tensor> act8_gelu_bwd(const at::Tensor& grad_y, const at::Tensor& q, const at::Tensor& scale,
                                                 bool recompute) {
  no_tangent({&grad_y});
  same_device(grad_y, {&q, &scale});
  TORCH_CHECK(grad_y.dim() >= 1, "grad_y must have at least one dimension");
  const int64_t C = grad_y.size(-1), rows = check_checkpoint(q, scale, C);
  TORCH_CHECK(grad_y.sizes().slice(0, grad_y.dim() - 1) == q.sizes().slice(0, q.dim() - 1),
              "grad_y ", grad_y.sizes(), " does not have the checkpoint's rows ", q.sizes());
  const c10::DeviceGuard guard(grad_y.device());
  at::Tensor g = dense(grad_y), qc = dense(q), sc = dense(scale), gx = at::empty_like(g);
  at::Tensor y = recompute ? at::empty_like(g) : at::empty({0}, g.options());
  vs_ok(vs_act8_gelu_backward(dcode(g), g.data_ptr(), qc.data_ptr(), sc.data_ptr(), gx.data_ptr(),
                              recompute ? y.data_ptr() : nullptr, rows, (int)C, cur_stream(g)),
        "act8_gelu_bwd");
  return {gx, y};
}

const int* row_map(const std::optional<at::Tensor>& rows, const at::Tensor& like, int64_t n) {
  if (!rows.has_value()) return nullptr;
  same_device(like, {&*rows});
  TORCH_CHECK(rows->scalar_type() == at::kInt && rows->is_contiguous() && rows->numel() == n,
              "rows must be contiguous int32, one for each row of x");
  return rows->data_ptr<int>();
}

// -> (s, y, q, scale, mean, rstd): s is x without a residual r; rows (int32): y [out_rows, C], row i
// of x normalised into row rows[i] of y (the others are left unwritten)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> act8_layer_norm_fwd(
    const at::Tensor& x, const std::optional<at::Tensor>& r, const at::Tensor& weight, const at::Tensor& bias,
    double eps, const std::optional<at::Tensor>& rows, int64_t out_rows, bool keep) {
  no_tangent({&x, &weight, &bias});
  if (r.has_value()) no_tangent({&*r});
  same_device(x, {&weight, &bias});
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
  const int64_t C = x.size(-1), M = C ? x.numel() / C : 0;
  TORCH_CHECK(C >= 1 && C <= 8192, "act8_layer_norm: 1 to 8192 features, got ", C);
  TORCH_CHECK(weight.scalar_type() == x.scalar_type() && bias.scalar_type() == x.scalar_type() &&
                  weight.sizes() == at::IntArrayRef({C}) && bias.sizes() == at::IntArrayRef({C}),
              "weight and bias must be [", C, "] in x's dtype");
  const c10::DeviceGuard guard(x.device());
  at::Tensor xc = dense(x), wc = dense(weight), bc = dense(bias), rc, s = xc;
  if (r.has_value()) {
    same_device(x, {&*r});
    TORCH_CHECK(r->sizes() == x.sizes() && r->scalar_type() == x.scalar_type(), "r must be shaped and typed like x");
    rc = dense(*r);
    s = at::empty_like(xc);
  }
  const int* map = row_map(rows, x, M);
  TORCH_CHECK(out_rows >= 0, "out_rows must not be negative");
  at::Tensor y = map ? at::empty({out_rows, C}, xc.options()) : at::empty_like(xc);
  at::Tensor q = keep ? new_q(xc) : at::empty({0}, xc.options().dtype(at::kChar));
  at::Tensor scale = keep ? new_scale(xc) : at::empty({0}, xc.options().dtype(at::kByte));
  at::Tensor mean = at::empty({M}, xc.options().dtype(at::kFloat)), rstd = at::empty_like(mean);
  vs_ok(vs_act8_layer_norm_forward(dcode(xc), xc.data_ptr(), r.has_value() ? rc.data_ptr() : nullptr, wc.data_ptr(),
                                   bc.data_ptr(), r.has_value() ? s.data_ptr() : nullptr, y.data_ptr(),
                                   keep ? q.data_ptr() : nullptr, keep ? scale.data_ptr() : nullptr,
                                   mean.data_ptr<float>(), rstd.data_ptr<float>(), M, (int)C, (float)eps, map, out_rows,
                                   cur_stream(xc)),
        "act8_layer_norm_fwd");
  return {s, y, q, scale, mean, rstd};
}

// -> (gx, gw, gb); grad_s: the gradient of s = x + r, added to gx
std::tuple<at::Tensor, at::Tensor, at::Tensor> act8_layer_norm_bwd(
    const at::Tensor& grad_y, const std::optional<at::Tensor>& grad_s, const at::Tensor& q, const at::Tensor& scale,
    const at::Tensor& weight, const at::Tensor& mean, const at::Tensor& rstd, const std::optional<at::Tensor>& rows) {
  no_tangent({&grad_y, &weight, &mean, &rstd});
  if (grad_s.has_value()) no_tangent({&*grad_s});
  same_device(grad_y, {&q, &scale, &weight, &mean, &rstd});
  TORCH_CHECK(weight.dim() == 1, "weight must be one-dimensional");
  const int64_t C = weight.size(0), M = check_checkpoint(q, scale, C);
  TORCH_CHECK(C >= 1 && C <= 8192, "act8_layer_norm: 1 to 8192 features, got ", C);
  TORCH_CHECK(grad_y.dim() >= 1 && grad_y.size(-1) == C && weight.scalar_type() == grad_y.scalar_type(),
              "grad_y must have weight's features and dtype");
  TORCH_CHECK(mean.scalar_type() == at::kFloat && rstd.scalar_type() == at::kFloat && mean.numel() == M &&
                  rstd.numel() == M && mean.is_contiguous() && rstd.is_contiguous(),
              "mean / rstd must be contiguous float32, one for each row of the checkpoint");
  const c10::DeviceGuard guard(grad_y.device());
  const int* map = row_map(rows, grad_y, M);
  TORCH_CHECK(map || grad_y.numel() == M * C, "grad_y ", grad_y.sizes(), " does not have the checkpoint's rows");
  auto sz = q.sizes().vec();
  sz.back() = C;
  at::Tensor g = dense(grad_y), qc = dense(q), sc = dense(scale), wc = dense(weight), ds;
  if (grad_s.has_value()) {
    same_device(grad_y, {&*grad_s});
    TORCH_CHECK(grad_s->numel() == M * C && grad_s->scalar_type() == g.scalar_type(),
                "grad_s must have the checkpoint's rows and grad_y's dtype");
    ds = dense(*grad_s);
  }
  at::Tensor gx = at::empty(sz, g.options()), gw = at::empty_like(wc), gb = at::empty_like(wc);
  at::Tensor ws = at::empty({vs_act8_layer_norm_backward_workspace_bytes(M, (int)C)}, g.options().dtype(at::kByte));
  vs_ok(vs_act8_layer_norm_backward(dcode(g), g.data_ptr(), grad_s.has_value() ? ds.data_ptr() : nullptr,
                                    qc.data_ptr(), sc.data_ptr(), wc.data_ptr(), mean.data_ptr<float>(),
                                    rstd.data_ptr<float>(), gx.data_ptr(), gw.data_ptr(), gb.data_ptr(),
                                    ws.data_ptr(), M, (int)C, map, g.numel() / C, cur_stream(g)),
        "act8_layer_norm_bwd");
  return {gx, gw, gb};
}

// -> (dw [N, features], db [N] or an empty tensor) in `dtype`
std::tuple<at::Tensor, at::Tensor> act8_wgrad(const at::Tensor& grad_y, const at::Tensor& q, const at::Tensor& scale,
                                              int64_t features, at::ScalarType dtype, bool bias) {
  no_tangent({&grad_y});
  same_device(grad_y, {&q, &scale});
  TORCH_CHECK(features >= 1, "act8_wgrad: at least one feature");
  const int64_t T = check_checkpoint(q, scale, features);
  const c10::DeviceGuard guard(grad_y.device());
  at::Tensor g = as_rows(grad_y, "grad_y"), qc = dense(q), sc = dense(scale);
  const int64_t N = grad_y.size(-1);
  if (T > 1 && g.stride(0) < N) g = g.contiguous();           // overlapping rows (an expanded tensor)
  TORCH_CHECK(N == 0 || g.size(0) == T, "grad_y has ", g.size(0), " rows, the checkpoint ", T);
  at::Tensor dw = at::empty({N, features}, g.options().dtype(dtype));
  at::Tensor db = at::empty({bias ? N : 0}, g.options().dtype(dtype));
  const int n = as_int(N, "outputs"), k = (int)features;
  const int64_t bytes = vs_act8_wgrad_workspace_bytes(dcode(g), T, n, k);
  at::Tensor ws = bytes ? at::empty({bytes}, g.options().dtype(at::kByte)) : at::Tensor();
  vs_ok(vs_act8_wgrad(dcode(g), dcode(dw), g.data_ptr(), g.stride(0), qc.data_ptr(), sc.data_ptr(), dw.data_ptr(),
                      bias ? db.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, T, n, k, cur_stream(g)),
        "act8_wgrad");
  return {dw, db};
}

// ---- their autograd forms.  C++ Functions, not Python ones as for the ops above: a call on a few
// hundred rows is all host time, and a Python forward and backward (144 us for a LayerNorm step on
// 400 rows of 256) cost several times what these do.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients that are not differentiable again: under create_graph a second backward through them
// raises (as torch.autograd.function.once_differentiable has it).
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const auto& g : grads) in.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "an op of 8-bit activation checkpoints is differentiated twice: its gradients are once differentiable",
      in.size());
  return (*error)(std::move(in));
}

bool keeps(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

struct GeluAct8 : public torch::autograd::Function<GeluAct8> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x) {
    auto [y, q, scale] = act8_gelu_fwd(x, true);
    ctx->save_for_backward({q, scale});
    ctx->saved_data["dtype"] = x.scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    at::Tensor gx;
    {
      at::NoGradGuard guard;
      gx = std::get<0>(act8_gelu_bwd(grads[0].to(ctx->saved_data["dtype"].toScalarType()), saved[0], saved[1], false));
    }
    return once({gx});
  }
};

at::Tensor gelu_act8(const at::Tensor& x) {
  return keeps({&x}) ? GeluAct8::apply(x) : std::get<0>(act8_gelu_fwd(x, false));
}

// the rows of y that no row of x goes to (the window layout's padding) are zeros
void clear_rows(at::Tensor& y, const std::optional<at::Tensor>& pad) {
  if (pad.has_value() && pad->numel()) y.index_fill_(0, *pad, 0);
}

std::optional<at::Tensor> maybe(const at::Tensor& t) {
  return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt;
}

// -> y, or with r: s and y
struct LayerNormAct8 : public torch::autograd::Function<LayerNormAct8> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& r,
                               const at::Tensor& weight, const at::Tensor& bias, double eps,
                               const std::optional<at::Tensor>& rows, const std::optional<at::Tensor>& pad,
                               int64_t out_rows) {
    ctx->set_materialize_grads(false);
    auto [s, y, q, scale, mean, rstd] = act8_layer_norm_fwd(x, r, weight, bias, eps, rows, out_rows, true);
    clear_rows(y, pad);
    ctx->save_for_backward({q, scale, weight, mean, rstd, rows.value_or(at::Tensor())});
    ctx->saved_data["residual"] = r.has_value();
    return r.has_value() ? variable_list{s, y} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const bool residual = ctx->saved_data["residual"].toBool();
    const at::Tensor gs = residual ? grads[0] : at::Tensor(), gy = residual ? grads[1] : grads[0];
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &scale = saved[1], &weight = saved[2], &mean = saved[3], &rstd = saved[4],
                     &rows = saved[5];
    at::Tensor gx, gw, gb;
    {
      at::NoGradGuard guard;
      const auto dtype = weight.scalar_type();
      if (gy.defined()) {
        std::tie(gx, gw, gb) = act8_layer_norm_bwd(gy.to(dtype), gs.defined() ? maybe(gs.to(dtype)) : std::nullopt, q,
                                                   scale, weight, mean, rstd, maybe(rows));
      } else if (gs.defined()) {                 // only s was used: its gradient passes through
        gx = gs.to(dtype);
        gw = at::zeros_like(weight);
        gb = at::zeros_like(weight);
      }
    }
    variable_list out = once({gx, gw, gb});
    return {out[0], residual ? out[0] : at::Tensor(), out[1], out[2], at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor()};
  }
};

at::Tensor layer_norm_act8(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, double eps,
                           const std::optional<at::Tensor>& rows, const std::optional<at::Tensor>& pad,
                           int64_t out_rows) {
  if (keeps({&x, &weight, &bias}))
    return LayerNormAct8::apply(x, std::optional<at::Tensor>(), weight, bias, eps, rows, pad, out_rows)[0];
  at::Tensor y = std::get<1>(act8_layer_norm_fwd(x, std::nullopt, weight, bias, eps, rows, out_rows, false));
  clear_rows(y, pad);
  return y;
}

std::tuple<at::Tensor, at::Tensor> add_layer_norm_act8(const at::Tensor& x, const at::Tensor& r,
                                                       const at::Tensor& weight, const at::Tensor& bias, double eps,
                                                       const std::optional<at::Tensor>& rows,
                                                       const std::optional<at::Tensor>& pad, int64_t out_rows) {
  if (keeps({&x, &r, &weight, &bias})) {
    auto out = LayerNormAct8::apply(x, std::optional<at::Tensor>(r), weight, bias, eps, rows, pad, out_rows);
    return {out[0], out[1]};
  }
  auto [s, y, q, scale, mean, rstd] = act8_layer_norm_fwd(x, r, weight, bias, eps, rows, out_rows, false);
  clear_rows(y, pad);
  return {s, y};
}

}  // namespace

TORCH_LIBRARY(visionseg, m) {
  m.def("msda_fwd(Tensor value, Tensor spatial_shapes, Tensor level_start_index, Tensor sampling_loc, "
        "Tensor attn_weight, int im2col_step) -> Tensor");
  m.def("msda_bwd(Tensor value, Tensor spatial_shapes, Tensor level_start_index, Tensor sampling_loc, "
        "Tensor attn_weight, Tensor grad_output, int im2col_step, bool f32_grad_value=False) -> (Tensor, Tensor, Tensor)");
  m.def("swin_window_fwd(Tensor x, int window, int shift) -> Tensor");
  m.def("swin_window_bwd(Tensor windows, int batch, int height, int width, int window, int shift) -> Tensor");
  m.def("win_attn_fwd(Tensor qkv, Tensor rel_table, int heads, int window, int shift, int nwin_h, int nwin_w, "
        "float scale, bool fp8=False) -> (Tensor, Tensor)");
  m.def("win_attn_bwd(Tensor qkv, Tensor rel_table, Tensor out, Tensor lse, Tensor grad_out, int heads, int window, "
        "int shift, int nwin_h, int nwin_w, float scale, bool fp8=False, bool table_partials=False) -> (Tensor, Tensor)");
  m.def("win_attn_fwd_img(Tensor qkv, Tensor rel_table, int heads, int window, int shift, int nwin_h, int nwin_w, "
        "int height, int width, float scale, bool fp8) -> (Tensor, Tensor)");
  m.def("win_attn_bwd_img(Tensor qkv, Tensor rel_table, Tensor out, Tensor lse, Tensor grad_out, int heads, "
        "int window, int shift, int nwin_h, int nwin_w, int height, int width, float scale, bool fp8) "
        "-> (Tensor, Tensor)");
  m.def("mask_head_fwd(Tensor mask_embed, Tensor pixel_nhwc, int height, int width) -> Tensor");
  m.def("mask_head_bwd(Tensor grad_logits, Tensor mask_embed, Tensor pixel_nhwc, Tensor(a!) grad_pixel, "
        "bool accumulate) -> Tensor");
  m.def("attn_bitmask(Tensor logits, int target_h, int target_w) -> Tensor");
  m.def("masked_xattn_fwd(Tensor q, Tensor k, Tensor v, Tensor words, int heads, float scale) -> (Tensor, Tensor)");
  m.def("masked_xattn_bwd(Tensor q, Tensor k, Tensor v, Tensor words, Tensor out, Tensor lse, Tensor grad_out, "
        "int heads, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("self_attn_fwd(Tensor q, Tensor k, Tensor v, Tensor words, int heads, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("self_attn_bwd(Tensor q, Tensor k, Tensor v, Tensor words, Tensor out, Tensor lse, Tensor grad_out, "
        "int heads, float scale) -> (Tensor, Tensor, Tensor)");
  m.def("act8_pack(Tensor x) -> (Tensor, Tensor)");
  m.def("act8_unpack(Tensor q, Tensor scale, int features, ScalarType dtype) -> Tensor");
  m.def("act8_gelu_fwd(Tensor x, bool keep=True) -> (Tensor, Tensor, Tensor)");
  m.def("act8_gelu_bwd(Tensor grad_y, Tensor q, Tensor scale, bool recompute=False) -> (Tensor, Tensor)");
  m.def("act8_layer_norm_fwd(Tensor x, Tensor? r, Tensor weight, Tensor bias, float eps, Tensor? rows=None, "
        "int out_rows=0, bool keep=True) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("act8_layer_norm_bwd(Tensor grad_y, Tensor? grad_s, Tensor q, Tensor scale, Tensor weight, Tensor mean, "
        "Tensor rstd, Tensor? rows=None) -> (Tensor, Tensor, Tensor)");
  m.def("act8_wgrad(Tensor grad_y, Tensor q, Tensor scale, int features, ScalarType dtype, bool bias=False) "
        "-> (Tensor, Tensor)");
  // with autograd (a function given here runs for every key: it takes its own gradient)
  m.def("gelu_act8(Tensor x) -> Tensor", gelu_act8);
  m.def("layer_norm_act8(Tensor x, Tensor weight, Tensor bias, float eps, Tensor? rows=None, Tensor? pad=None, "
        "int out_rows=0) -> Tensor", layer_norm_act8);
  m.def("add_layer_norm_act8(Tensor x, Tensor r, Tensor weight, Tensor bias, float eps, Tensor? rows=None, "
        "Tensor? pad=None, int out_rows=0) -> (Tensor, Tensor)", add_layer_norm_act8);
}

TORCH_LIBRARY_IMPL(visionseg, CUDA, m) {
  m.impl("msda_fwd", msda_fwd);
  m.impl("msda_bwd", msda_bwd);
  m.impl("swin_window_fwd", swin_window_fwd);
  m.impl("swin_window_bwd", swin_window_bwd);
  m.impl("win_attn_fwd", win_attn_fwd);
  m.impl("win_attn_bwd", win_attn_bwd);
  m.impl("win_attn_fwd_img", win_attn_fwd_img);
  m.impl("win_attn_bwd_img", win_attn_bwd_img);
  m.impl("mask_head_fwd", mask_head_fwd);
  m.impl("mask_head_bwd", mask_head_bwd);
  m.impl("attn_bitmask", attn_bitmask);
  m.impl("masked_xattn_fwd", masked_xattn_fwd);
  m.impl("masked_xattn_bwd", masked_xattn_bwd);
  m.impl("self_attn_fwd", self_attn_fwd);
  m.impl("self_attn_bwd", self_attn_bwd);
  m.impl("act8_pack", act8_pack);
  m.impl("act8_unpack", act8_unpack);
  m.impl("act8_gelu_fwd", act8_gelu_fwd);
  m.impl("act8_gelu_bwd", act8_gelu_bwd);
  m.impl("act8_layer_norm_fwd", act8_layer_norm_fwd);
  m.impl("act8_layer_norm_bwd", act8_layer_norm_bwd);
  m.impl("act8_wgrad", act8_wgrad);
}
