// Projections on 8-bit operands with a scale for each block of 128 (fp8_block.cu, gemm_fp8_block.cu): the part of autograd_native.cpp that
// allocates, calls and differentiates them.  Included there, inside its namespace.
//
//   y = rows(x) * tiles(w)^T      dx = rows(dy) * tiles(w)      dw = columns(dy)^T * columns(x)
//
// rows, columns, tiles: e4m3 with a scale for 128 values along the direction named.  Roundings to 8 bits pass gradients on as they are.  The
// forward pass quantises x in both forms from one read when there will be a weight gradient, and keeps the second (one byte a value).

constexpr auto E4M3 = at::kFloat8_e4m3fn;
constexpr int64_t MAX_BLOCK_SIZE = (1LL << 31) - 256;       // of a product's dimensions, which have 32 bits
int64_t blocks(int64_t n) { return (n + 127) / 128; }
enum { BY_ROWS = 1, BY_COLUMNS = 2, BY_TILES = 4 };

bool block_type(at::ScalarType t) { return t == BF16 || t == at::kHalf || t == F32; }

// Codes [R, C] whose rows begin 16 bytes apart or a multiple of it, as the product's loads want them
Tensor codes(int64_t R, int64_t C, at::Device device) {
  const int64_t ld = (C + 15) / 16 * 16;
  Tensor q = alloc({R, ld}, at::kByte, device).view(E4M3);
  return ld == C ? q : q.narrow(1, 0, C);
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 15) / 16 * 16; }
Tensor readable_codes(const Tensor& q) {
  if ((q.size(1) == 1 || q.stride(1) == 1) && row_stride(q) % 16 == 0 && row_stride(q) >= q.size(1) && on16(q)) return q;
  Tensor c = codes(q.size(0), q.size(1), q.device());
  c.view(at::kByte).copy_(q.view(at::kByte));
  return c;
}
// [.., D] -> [rows, D] with unit inner stride; any distance between rows
Tensor flat(const Tensor& x) {
  const int64_t D = x.size(-1);
  Tensor r = x.dim() == 2 ? x : x.reshape({D ? x.numel() / D : 0, D});
  return D == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

// Scales [blocks, n] as the kernels write them: rows a multiple of four apart
Tensor scale_rows(int64_t blocks, int64_t n, at::Device device) {
  const int64_t ld = (n + 3) / 4 * 4;
  Tensor s = alloc({blocks, ld}, F32, device);
  return ld == n ? s : s.narrow(1, 0, n);
}

struct Coded { Tensor q, s; };                  // codes [R, C], scales as fp8_block.cu lays them out
struct Quantized { Coded rows, cols; Tensor sums; };
Quantized quantize(const Tensor& x2, int form, bool sums = false, const Tensor& a = Tensor(), const Tensor& g = Tensor()) {
  const int64_t R = x2.size(0), C = x2.size(1);
  const at::Device dev = x2.device();
  Quantized r;
  if (form & BY_ROWS) r.rows = {codes(R, C, dev), scale_rows(blocks(C), R, dev)};
  if (form & BY_TILES) r.rows = {codes(R, C, dev), alloc({blocks(R), blocks(C)}, F32, dev)};
  if (form & BY_COLUMNS) r.cols = {codes(R, C, dev), scale_rows(blocks(R), C, dev)};
  if (sums) r.sums = alloc({blocks(R), C}, F32, dev);
  SB_CALL(sb_fp8_block_quantize, R > 0, ptr(x2), (long long)(R > 1 ? x2.stride(0) : C), (long long)R, (int)C, type_code(x2.scalar_type()), form, out(r.rows.q), f32o(r.rows.s),
          out(r.cols.q), f32o(r.cols.s), (long long)((C + 15) / 16 * 16), f32(a), ptr(g), f32o(r.sums), stream());
  return r;
}
Tensor column_sums(const Tensor& sums, at::ScalarType type) {
  Tensor o = alloc({sums.size(1)}, type, sums.device());
  SB_CALL(sb_fp8_block_column_sums, 1, f32(sums), out(o), (long long)sums.size(0), (int)sums.size(1), type_code(type), stream());
  return o;
}

// A product's operand: codes as they are stored, and where its scales lie
struct Factor {
  const Tensor& q;
  const Tensor& s;
  int64_t per_row, per_block;                   // strides of the scale
  bool transposed;                              // stored with the contraction first
};
void block_gemm(const Factor& a, const Factor& b, bool b_rows, const Tensor& o, const Tensor& bias = Tensor(), const Tensor& residual = Tensor(),
                bool accumulate = false) {
  const int M = o.size(0), N = o.size(1), K = a.transposed ? a.q.size(0) : a.q.size(1);
  const int rc = SB_RUN(sb_gemm_fp8_block, M > 0 && N > 0, ptr(a.q), f32(a.s), (long long)a.per_row, (long long)a.per_block, ptr(b.q), f32(b.s), (long long)b.per_row,
                        (long long)b.per_block, (int)b_rows, out(o), ptr(bias), ptr(residual), M, N, K, (long long)row_stride(a.q), (long long)row_stride(b.q),
                        (long long)(M > 1 ? o.stride(0) : N), (long long)(residual.defined() && M > 1 ? residual.stride(0) : N), (int)a.transposed,
                        (int)b.transposed, type_code(o.scalar_type()), (int)accumulate, status_word(o.device()), stream());
  TORCH_CHECK(rc == 0, "gemm_fp8_block failed (code ", rc, "): M=", M, " N=", N, " K=", K, " ",
              layouts({{"a", &a.q}, {"b", &b.q}, {"out", &o}, {"bias", &bias}, {"residual", &residual}}));
}
// y [T, N] = rows (xs [T, K / 128] in any strides) * tiles^T.  behind: the last launch on the stream wrote xq and xs.
Tensor block_forward(const Tensor& xq, const Tensor& xs, const Coded& w, at::ScalarType type, const Tensor& bias, const Tensor& residual, bool behind) {
  const int64_t T = xq.size(0), N = w.q.size(0);
  Tensor y = alloc({T, N}, type, xq.device());
  if (!L.sb_gemm_fp8_block_takes_few((int)T, (int)N)) {
    block_gemm({xq, xs, xs.stride(0), xs.stride(1), false}, {w.q, w.s, w.s.stride(0), w.s.stride(1), false}, false, y, bias, residual);
    return y;
  }
  SB_CALL(sb_gemm_fp8_block_few, T > 0, ptr(xq), f32(xs), (long long)xs.stride(0), (long long)xs.stride(1), ptr(w.q), f32(w.s), (long long)w.s.stride(0),
          (long long)w.s.stride(1), out(y), ptr(bias), ptr(residual), (int)T, (int)N, (int)xq.size(1), (long long)row_stride(xq), (long long)row_stride(w.q), (long long)N,
          (long long)(residual.defined() && T > 1 ? residual.stride(0) : N), type_code(type), (int)behind, status_word(xq.device()), stream());
  return y;
}
Tensor block_input_grad(const Coded& g, const Coded& w, at::ScalarType type) {
  Tensor dx = alloc({g.q.size(0), w.q.size(1)}, type, g.q.device());
  block_gemm({g.q, g.s, 1, g.s.stride(0), false}, {w.q, w.s, w.s.stride(1), w.s.stride(0), true}, false, dx);
  return dx;
}
// dw [N, K]; added by the product's epilogue straight into the parameter's gradient where that lives in a persistent flat buffer
Tensor block_weight_grad(const Coded& g, const Coded& x, at::ScalarType type, const Tensor& sink) {
  const int64_t N = g.q.size(1), K = x.q.size(1);
  const Factor a{g.q, g.s, 1, g.s.stride(0), true}, b{x.q, x.s, 1, x.s.stride(0), true};
  if (sink.defined()) {
    const Tensor& tgt = sink.grad();
    if (tgt.defined() && tgt.scalar_type() == type && tgt.is_contiguous() && tgt.dim() == 2 && tgt.size(0) == N && tgt.size(1) == K) {
      if (g.q.size(0) > 0) block_gemm(a, b, true, tgt, Tensor(), Tensor(), true);
      return Tensor();
    }
  }
  if (g.q.size(0) == 0) return zeros({N, K}, type, g.q.device());
  Tensor dw = alloc({N, K}, type, g.q.device());
  block_gemm(a, b, true, dw);
  return dw;
}

void no_second_derivative() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "projections on 8-bit operands with a scale for each block have no second derivative (create_graph)");
}
// The output gradient in the forms that the wanted gradients need, and the bias gradient
struct OutGrad { Quantized q; Tensor bias; };
OutGrad out_grad(const Tensor& g2, bool x, bool w, bool bias) {
  OutGrad r;
  const int form = (x ? BY_ROWS : 0) | (w ? BY_COLUMNS : 0);
  const bool sums = bias && w && g2.size(0) > 0;
  if (form) r.q = quantize(g2, form, sums);
  if (sums) r.bias = column_sums(r.q.sums, g2.scalar_type());
  else if (bias) r.bias = g2.to(F32).sum(0).to(g2.scalar_type());
  return r;
}

// y = x w^T (+ bias) (+ residual).  Edges: x, w where it is a tensor that training changes, bias, residual.  xs: x holds codes with these scales.
struct BlockLinear : Function<BlockLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& bias, const OptTensor& residual, const Tensor& wq,
                        const Tensor& ws, bool fuse, bool train_w, at::ScalarType type) {
    const Tensor x2 = flat(x);
    const int64_t N = wq.size(0);
    Quantized xq = quantize(x2, BY_ROWS | (train_w ? BY_COLUMNS : 0));
    Tensor y = block_forward(xq.rows.q, xq.rows.s.t(), {wq, ws}, type, opt(bias), residual.has_value() ? flat(*residual) : Tensor(), true);
    ctx->save_for_backward({train_w ? xq.cols.q : Tensor(), train_w ? xq.cols.s : Tensor(), wq, ws});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["w"] = w.has_value();
    ctx->saved_data["train_w"] = train_w;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["res"] = residual.has_value();
    ctx->saved_data["N"] = N;
    ctx->saved_data["xtype"] = (int64_t)x.scalar_type();
    if (fuse) ctx->saved_data["sink"] = *w;
    return y.view(with_last(x.sizes(), N));
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second_derivative();
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t N = ctx->saved_data["N"].toInt(), K = shape.back(), T = g[0].numel() / N;
    const bool has_w = ctx->saved_data["w"].toBool(), has_b = ctx->saved_data["bias"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1) && ctx->saved_data["train_w"].toBool(),
               need_b = has_b && ctx->needs_input_grad(1 + has_w);
    const at::Device dev = g[0].device();
    const at::ScalarType xtype = (at::ScalarType)ctx->saved_data["xtype"].toInt();
    const OutGrad go = out_grad(flat(g[0]), need_x, need_w, need_b);
    Tensor gx, gw, gr;
    if (need_x) {
      const Coded w{readable_codes(as_saved(s[2], {N, K}, E4M3, dev)), as_saved(s[3], {blocks(N), blocks(K)}, F32, dev)};
      gx = block_input_grad(go.q.rows, w, xtype).view(shape);
    }
    if (need_w) {
      const Coded x{readable_codes(as_saved(s[0], {T, K}, E4M3, dev)), as_saved(s[1], {blocks(T), K}, F32, dev)};
      gw = block_weight_grad(go.q.cols, x, g[0].scalar_type(), sink(ctx, "sink"));
    }
    if (ctx->saved_data["res"].toBool() && ctx->needs_input_grad(1 + has_w + has_b)) gr = g[0];
    return {gx, gw, go.bias, gr, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// s = x + residual, codes of norm(s) * g by rows, 1 / rms
struct BlockNorm { Tensor s, q, scale, a; };
BlockNorm block_norm(const Tensor& x, const OptTensor& residual, const Tensor& g, double eps, int64_t form, bool want_a) {
  const Tensor x2 = flat(x), r2 = residual.has_value() ? flat(*residual) : Tensor(), gc = contiguous(g);
  const int64_t T = x2.size(0), D = x2.size(1);
  const at::Device dev = x.device();
  BlockNorm n;
  n.s = residual.has_value() ? alloc({T, D}, x.scalar_type(), dev) : x2;
  n.q = codes(T, D, dev);
  n.scale = scale_rows(blocks(D), T, dev);
  if (want_a) n.a = alloc({T}, F32, dev);
  SB_CALL(sb_fp8_block_norm, T > 0, ptr(x2), (long long)(T > 1 ? x2.stride(0) : D), ptr(r2), (long long)(r2.defined() && T > 1 ? r2.stride(0) : D), ptr(gc),
          residual.has_value() ? out(n.s) : nullptr, out(n.q), (long long)((D + 15) / 16 * 16), f32o(n.scale), f32o(n.a), (long long)T, (int)D, (float)eps, (int)form,
          type_code(x.scalar_type()), stream());
  return n;
}

// (w norm(s)^T (+ bias), s), s = x + residual.  Edges: x, residual, norm weight, w, bias.
struct BlockNormLinear : Function<BlockNormLinear> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const Tensor& wn, const OptTensor& w, const OptTensor& bias,
                               const Tensor& wq, const Tensor& ws, double eps, int64_t form, bool fuse) {
    const BlockNorm n = block_norm(x, residual, wn, eps, form, true);
    Tensor y = block_forward(n.q, n.scale.t(), {wq, ws}, x.scalar_type(), opt(bias), Tensor(), true);
    Tensor s = residual.has_value() ? n.s.view(x.sizes()) : x.view_as(x);
    ctx->save_for_backward({residual.has_value() ? s : x, wn, n.a, wq, ws});
    save_norm(ctx, x, eps, form);
    ctx->saved_data["res"] = residual.has_value();
    ctx->saved_data["w"] = w.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["N"] = wq.size(0);
    if (fuse) ctx->saved_data["sink"] = *w;
    ctx->set_materialize_grads(false);
    return {y.view(with_last(x.sizes(), wq.size(0))), s};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second_derivative();
    const bool has_r = ctx->saved_data["res"].toBool(), has_w = ctx->saved_data["w"].toBool(), has_b = ctx->saved_data["bias"].toBool();
    const auto result = [&](const Tensor& dx, const Tensor& dwn, const Tensor& dw, const Tensor& db) -> variable_list {
      return {dx, has_r ? dx : Tensor(), dwn, dw, db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    };
    if (!g[0].defined()) return result(g[1], Tensor(), Tensor(), Tensor());
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t N = ctx->saved_data["N"].toInt(), D = shape.back(), T = g[0].numel() / N;
    const at::Device dev = g[0].device();
    const at::ScalarType type = g[0].scalar_type();
    const bool need_n = ctx->needs_input_grad(0) || (has_r && ctx->needs_input_grad(1)) || ctx->needs_input_grad(1 + has_r),
               need_w = has_w && ctx->needs_input_grad(2 + has_r), need_b = has_b && ctx->needs_input_grad(2 + has_r + has_w);
    const Tensor s2 = aligned(as_saved(s[0], shape, type, dev)).view({T, D}), wn = aligned(as_saved(s[1], {D}, type, dev)), a = as_saved(s[2], {T}, F32, dev);
    const OutGrad go = out_grad(flat(g[0]), need_n, need_w, need_b);
    Tensor dx, dwn, dw;
    if (need_w)
      dw = block_weight_grad(go.q.cols, quantize(s2, BY_COLUMNS, false, a, wn).cols, type, sink(ctx, "sink"));
    if (need_n) {
      if (T == 0) {
        dx = zeros(shape, type, dev);
        dwn = zeros({D}, type, dev);
      } else {
        const Coded w{readable_codes(as_saved(s[3], {N, D}, E4M3, dev)), as_saved(s[4], {blocks(N), blocks(D)}, F32, dev)};
        std::tie(dx, dwn) = norm_bwd(s2, wn, a, block_input_grad(go.q.rows, w, type), g[1].defined() ? aligned(g[1]) : g[1],
                                     ctx->saved_data["eps"].toDouble(), ctx->saved_data["form"].toInt());
        dx = dx.view(shape);
      }
    }
    return result(dx, dwn, dw, go.bias);
  }
};

// ------------------------------------------------------------------------------------ checks
void no_tangents(std::initializer_list<const Tensor*> ts) {
  no_transforms();
  for (const Tensor* t : ts)
    TORCH_CHECK(!t || !t->_fw_grad(0).defined(), "8-bit operands with a scale for each block have no forward-mode derivative");
}
void check_block_input(const char* what, const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && block_type(x.scalar_type()), what, " takes bf16, fp16 or fp32 [..., D] with D >= 1, got ", x.scalar_type(),
                    " ", x.sizes());
  TORCH_CHECK_VALUE(x.size(-1) <= MAX_BLOCK_SIZE && x.numel() / x.size(-1) <= MAX_BLOCK_SIZE, what, " takes up to ", MAX_BLOCK_SIZE, " rows of as many values, got ",
                    x.sizes());
}
// what fp8_block_quantize (rows) and fp8_block_quantize_weight (tiles) return
void check_coded(const char* what, const Tensor& q, const Tensor& s, bool tiles) {
  const bool shape = q.dim() >= 1 && q.size(-1) >= 1 && (!tiles || q.dim() == 2);
  TORCH_CHECK_VALUE(shape && q.scalar_type() == E4M3 && s.scalar_type() == F32 && s.device() == q.device() &&
                        (tiles ? s.dim() == 2 && s.size(0) == blocks(q.size(0)) && s.size(1) == blocks(q.size(1)) : s.sizes().vec() == with_last(q.sizes(), blocks(q.size(-1)))),
                    what, ": float8_e4m3fn ", tiles ? "[N, K] with fp32 scales [N / 128, K / 128]" : "[..., K] with fp32 scales [..., K / 128]", " on one device, got ",
                    q.scalar_type(), " ", q.sizes(), ", ", s.scalar_type(), " ", s.sizes());
}
// A weight as the product reads it: kept codes, or those of a tensor
Coded block_weight(const Tensor& w, const OptTensor& ws) {
  if (ws.has_value()) return {readable_codes(w), *ws};
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  return quantize(flat(w), BY_TILES).rows;
}
void check_projection(const char* what, const Tensor& x, int64_t K, const Tensor& w, const OptTensor& ws, const OptTensor& bias, const OptTensor& residual,
                      at::ScalarType type, at::IntArrayRef y) {
  if (ws.has_value()) check_coded(what, w, *ws, true);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == K && w.size(0) >= 1 && w.size(0) <= MAX_BLOCK_SIZE && w.device() == x.device() && (ws.has_value() || w.scalar_type() == type),
                    what, ": weight ", w.scalar_type(), " ", w.sizes(), " on ", w.device(), " for rows of ", K, " values of ", type, " on ", x.device());
  TORCH_CHECK_VALUE(!bias.has_value() || (bias->dim() == 1 && bias->size(0) == w.size(0) && bias->scalar_type() == type && bias->device() == x.device()), what,
                    ": bias of ", type, " [", w.size(0), "] expected");
  TORCH_CHECK_VALUE(!residual.has_value() || (residual->sizes() == y && residual->scalar_type() == type && residual->device() == x.device()), what,
                    ": residual of ", type, " ", y, " expected");
}
OptTensor contiguous(const OptTensor& t) { return t.has_value() ? OptTensor(contiguous(*t)) : t; }

// ------------------------------------------------------------------------------------ what Python calls
std::tuple<Tensor, Tensor> fp8_block_quantize(const Tensor& x, bool tiles) {
  const char* what = tiles ? "fp8_block_quantize_weight" : "fp8_block_quantize";
  no_tangents({&x});
  check_block_input(what, x);
  TORCH_CHECK_VALUE(!tiles || x.dim() == 2, what, " takes [N, K], got ", x.sizes());
  const c10::cuda::CUDAGuard device(x.device());
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  const Quantized r = quantize(flat(x), tiles ? BY_TILES : BY_ROWS);
  if (tiles) return {r.rows.q, r.rows.s};
  return {r.rows.q.view(x.sizes()), r.rows.s.t().view(with_last(x.sizes(), blocks(x.size(-1))))};
}
Tensor fp8_block_dequantize(const Tensor& q, const Tensor& s, int64_t type) {
  no_transforms();
  const bool tiles = q.dim() == 2 && s.dim() == 2 && s.size(0) != q.size(0);
  check_coded("fp8_block_dequantize", q, s, tiles);
  const c10::cuda::CUDAGuard device(q.device());
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  const int64_t C = q.size(-1), R = q.numel() / C;
  TORCH_CHECK_VALUE(C <= MAX_BLOCK_SIZE && R <= MAX_BLOCK_SIZE, "fp8_block_dequantize takes up to ", MAX_BLOCK_SIZE, " rows of as many values, got ", q.sizes());
  Tensor q2 = flat(q.view(at::kByte)), s2 = s.dim() == 2 ? s : s.reshape({tiles ? s.size(0) : R, blocks(C)});
  Tensor x = alloc(q.sizes(), type == 0 ? BF16 : type == 1 ? at::kHalf : F32, q.device());
  SB_CALL(sb_fp8_block_dequantize, R > 0, ptr(q2), (long long)(R > 1 ? q2.stride(0) : C), f32(s2), (long long)s2.stride(0), (long long)s2.stride(1), (int)tiles, out(x), (long long)R, (int)C,
          (int)type, stream());
  return x;
}
void check_norm(const char* what, const Tensor& x, const Tensor& g, const OptTensor& residual) {
  check_block_input(what, x);
  const int64_t D = x.size(-1);
  TORCH_CHECK_VALUE(g.dim() == 1 && g.size(0) == D && g.scalar_type() == x.scalar_type() && g.device() == x.device(), what, ": weight ", g.scalar_type(), " ", g.sizes(),
                    " on ", g.device(), " for ", x.scalar_type(), " rows of ", D, " values on ", x.device());
  TORCH_CHECK_VALUE(!residual.has_value() || (residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() && residual->device() == x.device()), what,
                    ": residual of x's shape, type and device expected");
}
// nothing where the kernel does not cover the width
std::optional<std::tuple<Tensor, Tensor, Tensor>> rmsnorm_fp8_block(const Tensor& x, const Tensor& g, double eps, int64_t form, const OptTensor& residual) {
  no_tangents({&x, &g, given(residual)});
  check_norm("rmsnorm_fp8_block", x, g, residual);
  if (x.size(-1) > 16384) return std::nullopt;
  const c10::cuda::CUDAGuard device(x.device());
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  const BlockNorm n = block_norm(x, residual, g, eps, form, false);
  return std::make_tuple(n.q.view(x.sizes()), n.scale.t().view(with_last(x.sizes(), blocks(x.size(-1)))), residual.has_value() ? n.s.view(x.sizes()) : x);
}
// type: of the result
Tensor linear_fp8_block(const Tensor& x, const OptTensor& xs, const py::object& weight, const OptTensor& ws, const OptTensor& bias, const OptTensor& residual,
                        int64_t type_) {
  const char* what = "linear_fp8_block";
  const at::ScalarType type = type_ == 0 ? BF16 : type_ == 1 ? at::kHalf : F32;
  const Tensor w = weight.cast<Tensor>();
  no_tangents({&x, &w, given(bias), given(residual)});
  if (xs.has_value()) check_coded(what, x, *xs, false);
  else check_block_input(what, x);
  const int64_t K = x.size(-1), T = x.numel() / K;
  TORCH_CHECK_VALUE(K <= MAX_BLOCK_SIZE && T <= MAX_BLOCK_SIZE, what, " takes up to ", MAX_BLOCK_SIZE, " rows of as many values, got ", x.sizes());
  check_projection(what, x, K, w, ws, bias, residual, type, with_last(x.sizes(), w.size(0)));
  const c10::cuda::CUDAGuard device(x.device());
  const Coded wc = block_weight(w, ws);
  const OptTensor b = contiguous(bias);
  const OptTensor wt = ws.has_value() ? OptTensor() : OptTensor(w);
  if (wants_grad({&x, given(wt), given(bias), given(residual)})) {
    TORCH_CHECK_VALUE(!xs.has_value(), what, ": inputs in 8 bits carry no gradient; call it under torch.no_grad, or with the tensor itself");
    return BlockLinear::apply(x, wt, b, residual, wc.q, wc.s, !ws.has_value() && fused(weight), wants_grad({given(wt)}), type);
  }
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  const Tensor r2 = residual.has_value() ? flat(*residual) : Tensor();
  Tensor y;
  if (xs.has_value()) {
    const Tensor q2 = readable_codes(x.dim() == 2 ? x : x.reshape({T, K}));
    y = block_forward(q2, xs->dim() == 2 ? *xs : xs->reshape({T, blocks(K)}), wc, type, opt(b), r2, false);
  } else {
    const Coded xq = quantize(flat(x), BY_ROWS).rows;
    y = block_forward(xq.q, xq.s.t(), wc, type, opt(b), r2, true);
  }
  return y.view(with_last(x.sizes(), w.size(0)));
}
// nothing where the kernels do not cover type or width
std::optional<std::tuple<Tensor, Tensor>> norm_linear_fp8_block(const Tensor& x, const Tensor& g, double eps, int64_t form, const py::object& weight, const OptTensor& ws,
                                                                const OptTensor& bias, const OptTensor& residual) {
  const char* what = "norm_linear_fp8_block";
  const Tensor w = weight.cast<Tensor>();
  no_tangents({&x, &g, &w, given(bias), given(residual)});
  check_norm(what, x, g, residual);
  const int64_t K = x.size(-1);
  check_projection(what, x, K, w, ws, bias, OptTensor(), x.scalar_type(), {});
  const OptTensor wt = ws.has_value() ? OptTensor() : OptTensor(w);
  const bool train = wants_grad({&x, &g, given(wt), given(bias), given(residual)});
  // the norm's backward kernel: bf16, rows of eights
  if (K > 16384 || (train && (x.scalar_type() != BF16 || K % 8 || K < 64))) return std::nullopt;
  const c10::cuda::CUDAGuard device(x.device());
  const Coded wc = block_weight(w, ws);
  const OptTensor b = contiguous(bias);
  if (train) {
    variable_list r = BlockNormLinear::apply(x, residual, g, wt, b, wc.q, wc.s, eps, form, !ws.has_value() && fused(weight));
    return std::make_tuple(r[0], r[1]);
  }
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  const BlockNorm n = block_norm(x, residual, g, eps, form, false);
  const Tensor y = block_forward(n.q, n.scale.t(), wc, x.scalar_type(), opt(b), Tensor(), true);
  return std::make_tuple(y.view(with_last(x.sizes(), w.size(0))), residual.has_value() ? n.s.view(x.sizes()) : x);
}
