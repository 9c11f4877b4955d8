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
int64_t up_to(int64_t n, int64_t step) { return (n + step - 1) / step * step; }
enum { BY_ROWS = 1, BY_COLUMNS = 2, BY_TILES = 4 };

bool block_type(at::ScalarType t) { return t == BF16 || t == at::kHalf || t == F32; }

// A product's operand: codes [R, C], rows `ld` bytes apart; the scale of row r (BY_COLUMNS: column) and block b at s[r * s_row + b * s_block]; for
// tiles r counts blocks of rows too.  Whose memory it is, is somebody else's business.
struct Operand {
  const void* q = nullptr;
  const float* s = nullptr;
  int64_t R = 0, C = 0, ld = 0, s_row = 0, s_block = 0;
};
// Codes and scales of one form in one buffer, as fp8_block.cu lays them out: rows of codes 16 bytes apart or a multiple of it, then the scales.
struct Packed {
  int64_t R, C, ld, codes, s_ld, bytes;
  int form;
  Packed(int64_t R_, int64_t C_, int form_) : R(R_), C(C_), ld(up_to(C_, 16)), codes(up_to(R_ * ld, 256)), form(form_) {
    s_ld = form == BY_TILES ? blocks(C) : up_to(form == BY_ROWS ? R : C, 4);
    bytes = codes + (form == BY_ROWS ? blocks(C) : blocks(R)) * s_ld * 4;
  }
  Tensor make(at::Device device) const { return alloc({bytes}, at::kByte, device); }
  Operand in(const Tensor& buf) const { return in(static_cast<const char*>(ptr(buf))); }
  Operand in(const char* p) const {
    return {p, reinterpret_cast<const float*>(p + codes), R, C, ld, form == BY_TILES ? s_ld : 1, form == BY_TILES ? 1 : s_ld};
  }
};

// Codes and scales as tensors (what fp8_block_quantize returns and linear_fp8_block takes)
struct Coded { Tensor q, s; };
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : up_to(t.size(1), 16); }
Tensor codes(int64_t R, int64_t C, at::Device device) {
  const int64_t ld = up_to(C, 16);
  Tensor q = alloc({R, ld}, E4M3, device);
  return ld == C ? q : q.narrow(1, 0, C);
}
Tensor readable_codes(const Tensor& q) {
  if ((q.size(1) == 1 || q.stride(1) == 1) && row_stride(q) % 16 == 0 && row_stride(q) >= q.size(1) && on16(q)) return q;
  Tensor c = codes(q.size(0), q.size(1), q.device());
  c.view(at::kByte).copy_(q.view(at::kByte));
  return c;
}
// Scales of x's rows, [..., D / 128], as the kernels write them: those of neighbouring rows together, blocks a multiple of four rows apart
Tensor row_scales(const Tensor& x, int64_t R, int64_t C) {
  const int64_t ld = up_to(R, 4), last = x.dim() - 1;
  std::vector<int64_t> sizes = with_last(x.sizes(), blocks(C)), strides(sizes.size(), ld);
  int64_t step = 1;
  for (int64_t i = last - 1; i >= 0; --i) { strides[i] = step; step *= sizes[i]; }
  return alloc({blocks(C) * ld}, F32, x.device()).as_strided(sizes, strides);
}
Operand operand(const Coded& c) { return {ptr(c.q), f32(c.s), c.q.size(0), c.q.size(1), row_stride(c.q), c.s.stride(0), c.s.stride(1)}; }

// [.., D] -> [rows, D] with unit inner stride; any distance between rows
Tensor flat(const Tensor& x) {
  const int64_t D = x.size(-1);
  Tensor r = x.dim() == 2 ? x : x.reshape({D ? x.numel() / D : 0, D});
  return D == 1 || r.stride(1) == 1 ? r : r.contiguous();
}
long long rows_apart(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// x2 in the forms of `form`: rows (or tiles) to `r`, columns to `c`; sums: column sums of each 128 rows; a, g: of x2 * a[row] * g[column]
void quantize(const Tensor& x2, int form, const Operand& r, const Operand& c, float* sums = nullptr, const Tensor& a = Tensor(), const Tensor& g = Tensor()) {
  const int64_t R = x2.size(0), C = x2.size(1);
  SB_CALL(sb_fp8_block_quantize, R > 0, ptr(x2), rows_apart(x2), (long long)R, (int)C, type_code(x2.scalar_type()), form, const_cast<void*>(r.q), const_cast<float*>(r.s),
          const_cast<void*>(c.q), const_cast<float*>(c.s), (long long)up_to(C, 16), f32(a), ptr(g), sums, stream());
}
Tensor column_sums(const float* sums, int64_t tiles, int64_t C, at::ScalarType type, at::Device device) {
  Tensor o = alloc({C}, type, device);
  SB_CALL(sb_fp8_block_column_sums, 1, sums, out(o), (long long)tiles, (int)C, type_code(type), stream());
  return o;
}

// o (+)= a b^T (+ bias) (+ residual); a_mn, b_mn: stored with the contraction first; b_rows: b has a scale for each of its rows
void block_gemm(const Operand& a, bool a_mn, const Operand& b, bool b_mn, bool b_rows, int64_t K, const Tensor& o, const Tensor& bias = Tensor(),
                const Tensor& residual = Tensor(), bool accumulate = false) {
  const int M = o.size(0), N = o.size(1);
  const int rc = SB_RUN(sb_gemm_fp8_block, M > 0 && N > 0, a.q, a.s, (long long)a.s_row, (long long)a.s_block, b.q, b.s, (long long)b.s_row, (long long)b.s_block, (int)b_rows,
                        out(o), ptr(bias), ptr(residual), M, N, (int)K, (long long)a.ld, (long long)b.ld, rows_apart(o), residual.defined() ? rows_apart(residual) : 0LL,
                        (int)a_mn, (int)b_mn, type_code(o.scalar_type()), (int)accumulate, status_word(o.device()), stream());
  TORCH_CHECK(rc == 0, "gemm_fp8_block failed (code ", rc, "): M=", M, " N=", N, " K=", K, " lda=", a.ld, " ldb=", b.ld, " ",
              layouts({{"out", &o}, {"bias", &bias}, {"residual", &residual}}));
}
// y [T, N] = rows * tiles^T.  behind: the last launch on the stream wrote x.
Tensor block_forward(const Operand& x, const Operand& w, at::ScalarType type, at::Device device, const Tensor& bias, const Tensor& residual, bool behind) {
  const int64_t T = x.R, N = w.R;
  Tensor y = alloc({T, N}, type, device);
  if (!L.sb_gemm_fp8_block_takes_few((int)T, (int)N)) {
    block_gemm(x, false, w, false, false, x.C, y, bias, residual);
    return y;
  }
  SB_CALL(sb_gemm_fp8_block_few, T > 0, x.q, x.s, (long long)x.s_row, (long long)x.s_block, w.q, w.s, (long long)w.s_row, (long long)w.s_block, out(y), ptr(bias), ptr(residual),
          (int)T, (int)N, (int)x.C, (long long)x.ld, (long long)w.ld, (long long)N, residual.defined() ? rows_apart(residual) : 0LL, type_code(type), (int)behind,
          status_word(device), stream());
  return y;
}
Tensor block_input_grad(const Operand& g, Operand w, at::ScalarType type, at::Device device) {
  Tensor dx = alloc({g.R, w.C}, type, device);
  std::swap(w.s_row, w.s_block);                            // the contraction goes over the weight's rows
  block_gemm(g, false, w, true, false, g.C, dx);
  return dx;
}
// dw [N, K]; added by the product's epilogue straight into the parameter's gradient where that lives in a persistent flat buffer
Tensor block_weight_grad(const Operand& g, const Operand& x, at::ScalarType type, at::Device device, const Tensor& sink) {
  const int64_t N = g.C, K = x.C, T = g.R;
  if (sink.defined()) {
    const Tensor& tgt = sink.grad();
    if (tgt.defined() && tgt.scalar_type() == type && tgt.is_contiguous() && tgt.dim() == 2 && tgt.size(0) == N && tgt.size(1) == K) {
      if (T > 0) block_gemm(g, true, x, true, true, T, tgt, Tensor(), Tensor(), true);
      return Tensor();
    }
  }
  if (T == 0) return zeros({N, K}, type, device);
  Tensor dw = alloc({N, K}, type, device);
  block_gemm(g, true, x, true, true, T, dw);
  return dw;
}

void no_second_derivative() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "projections on 8-bit operands with a scale for each block have no second derivative (create_graph)");
}
// The output gradient in the forms that the wanted gradients need, and the bias gradient
struct OutGrad {
  Tensor buf, bias;
  Operand rows, cols;
};
OutGrad out_grad(const Tensor& g2, bool x, bool w, bool bias) {
  OutGrad r;
  const int64_t T = g2.size(0), N = g2.size(1);
  const at::Device dev = g2.device();
  const bool sums = bias && w && T > 0;
  const Packed rows(T, N, BY_ROWS), cols(T, N, BY_COLUMNS);
  const int64_t at_cols = x ? up_to(rows.bytes, 256) : 0, at_sums = at_cols + (w ? up_to(cols.bytes, 256) : 0);
  float* part = nullptr;
  if (x || w) {
    r.buf = alloc({at_sums + (sums ? blocks(T) * N * 4 : 0)}, at::kByte, dev);
    char* p = static_cast<char*>(out(r.buf));
    if (x) r.rows = rows.in(p);
    if (w) r.cols = cols.in(p + at_cols);
    if (sums) part = reinterpret_cast<float*>(p + at_sums);
    quantize(g2, (x ? BY_ROWS : 0) | (w ? BY_COLUMNS : 0), r.rows, r.cols, part);
  }
  if (sums) r.bias = column_sums(part, blocks(T), N, g2.scalar_type(), dev);
  else if (bias) r.bias = g2.to(F32).sum(0).to(g2.scalar_type());
  return r;
}
// A weight that a node kept: packed codes (s absent), or the caller's pair
Operand saved_weight(const Tensor& q, const Tensor& s, int64_t N, int64_t K, at::Device dev, Coded& hold) {
  if (!s.defined()) {
    const Packed p(N, K, BY_TILES);
    hold.q = as_saved(q, {p.bytes}, at::kByte, dev);
    return p.in(hold.q);
  }
  hold = {readable_codes(as_saved(q, {N, K}, E4M3, dev)), as_saved(s, {blocks(N), blocks(K)}, F32, dev)};
  return operand(hold);
}

// y = x w^T (+ bias) (+ residual).  Edges: x, w where it is a tensor that training changes, bias, residual.
struct BlockLinear : Function<BlockLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& bias, const OptTensor& residual, const Tensor& wq,
                        const OptTensor& ws, bool fuse, bool train_w, at::ScalarType type, const Operand& wo) {
    const Tensor x2 = flat(x);
    const at::Device dev = x.device();
    const int64_t N = wo.R;
    const Packed rows(x2.size(0), x2.size(1), BY_ROWS), cols(x2.size(0), x2.size(1), BY_COLUMNS);
    const Tensor kept = train_w ? cols.make(dev) : Tensor();
    Tensor y;
    {
      const Tensor buf = rows.make(dev), r2 = residual.has_value() ? flat(*residual) : Tensor();
      quantize(x2, BY_ROWS | (train_w ? BY_COLUMNS : 0), rows.in(buf), train_w ? cols.in(kept) : Operand());
      y = block_forward(rows.in(buf), wo, type, dev, opt(bias), r2, true);
    }
    ctx->save_for_backward({kept, wq, opt(ws)});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["flags"] = int64_t(w.has_value()) | int64_t(train_w) << 1 | int64_t(bias.has_value()) << 2 | int64_t(residual.has_value()) << 3;
    ctx->saved_data["N"] = N;
    ctx->saved_data["xtype"] = (int64_t)x.scalar_type();
    if (fuse) ctx->saved_data["sink"] = *w;
    return x.dim() == 2 ? y : y.view(with_last(x.sizes(), N));
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second_derivative();
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t N = ctx->saved_data["N"].toInt(), K = shape.back(), T = g[0].numel() / N, flags = ctx->saved_data["flags"].toInt();
    const bool has_w = flags & 1, has_b = flags & 4;
    const bool need_x = ctx->needs_input_grad(0), need_w = has_w && (flags & 2) && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(1 + has_w);
    const at::Device dev = g[0].device();
    const OutGrad go = out_grad(flat(g[0]), need_x, need_w, need_b);
    Tensor gx, gw, gr;
    if (need_x) {
      Coded hold;
      const Operand w = saved_weight(s[1], s[2], N, K, dev, hold);
      gx = block_input_grad(go.rows, w, (at::ScalarType)ctx->saved_data["xtype"].toInt(), dev);
      if (shape.size() != 2) gx = gx.view(shape);
    }
    if (need_w) {
      const Packed p(T, K, BY_COLUMNS);
      const Tensor x = as_saved(s[0], {p.bytes}, at::kByte, dev);
      gw = block_weight_grad(go.cols, p.in(x), g[0].scalar_type(), dev, sink(ctx, "sink"));
    }
    if ((flags & 8) && ctx->needs_input_grad(1 + has_w + has_b)) gr = g[0];
    return {gx, gw, go.bias, gr, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// s = x + residual, codes of norm(s) * g by rows to `q`, 1 / rms
struct BlockNorm { Tensor s, a; };
BlockNorm block_norm(const Tensor& x, const OptTensor& residual, const Tensor& g, double eps, int64_t form, bool want_a, const Operand& q) {
  const Tensor x2 = flat(x), r2 = residual.has_value() ? flat(*residual) : Tensor(), gc = contiguous(g);
  const int64_t T = x2.size(0), D = x2.size(1);
  BlockNorm n;
  n.s = residual.has_value() ? alloc(x.sizes(), x.scalar_type(), x.device()) : x;
  if (want_a) n.a = alloc({T}, F32, x.device());
  SB_CALL(sb_fp8_block_norm, T > 0, ptr(x2), rows_apart(x2), ptr(r2), r2.defined() ? rows_apart(r2) : 0LL, ptr(gc), residual.has_value() ? out(n.s) : nullptr,
          const_cast<void*>(q.q), (long long)q.ld, const_cast<float*>(q.s), f32o(n.a), (long long)T, (int)D, (float)eps, (int)form, type_code(x.scalar_type()), stream());
  return n;
}

// (w norm(s)^T (+ bias), s), s = x + residual.  Edges: x, residual, norm weight, w, bias.
struct BlockNormLinear : Function<BlockNormLinear> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const Tensor& wn, const OptTensor& w, const OptTensor& bias,
                               const Tensor& wq, const OptTensor& ws, double eps, int64_t form, bool fuse, const Operand& wo) {
    const at::Device dev = x.device();
    const int64_t D = x.size(-1);
    BlockNorm n;
    Tensor y;
    {
      const Packed p(x.numel() / D, D, BY_ROWS);
      const Tensor buf = p.make(dev);
      n = block_norm(x, residual, wn, eps, form, true, p.in(buf));
      y = block_forward(p.in(buf), wo, x.scalar_type(), dev, opt(bias), Tensor(), true);
    }
    ctx->save_for_backward({n.s, wn, n.a, wq, opt(ws)});
    save_norm(ctx, x, eps, form);
    ctx->saved_data["flags"] = int64_t(residual.has_value()) | int64_t(w.has_value()) << 1 | int64_t(bias.has_value()) << 2;
    ctx->saved_data["N"] = wo.R;
    if (fuse) ctx->saved_data["sink"] = *w;
    ctx->set_materialize_grads(false);
    return {x.dim() == 2 ? y : y.view(with_last(x.sizes(), wo.R)), residual.has_value() ? n.s : x.view_as(x)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second_derivative();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const bool has_r = flags & 1, has_w = flags & 2, has_b = flags & 4;
    const auto result = [&](const Tensor& dx, const Tensor& dwn, const Tensor& dw, const Tensor& db) -> variable_list {
      return {dx, has_r ? dx : Tensor(), dwn, dw, db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
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
    if (need_w) {
      const Packed p(T, D, BY_COLUMNS);
      const Tensor x = p.make(dev);
      quantize(s2, BY_COLUMNS, Operand(), p.in(x), nullptr, a, wn);
      dw = block_weight_grad(go.cols, p.in(x), type, dev, sink(ctx, "sink"));
    }
    if (need_n) {
      if (T == 0) {
        dx = zeros(shape, type, dev);
        dwn = zeros({D}, type, dev);
      } else {
        Coded hold;
        const Operand w = saved_weight(s[3], s[4], N, D, dev, hold);
        const Tensor dn = block_input_grad(go.rows, w, F32, dev), ds = g[1].defined() ? contiguous(g[1]) : g[1];
        const int64_t parts = L.sb_fp8_block_norm_back_blocks((long long)T, (int)D);
        const Tensor dg = alloc({parts, D}, F32, dev);
        dx = alloc({T, D}, type, dev);
        SB_CALL(sb_fp8_block_norm_back, 1, ptr(s2), ptr(wn), f32(a), f32(dn), ptr(ds), out(dx), f32o(dg), (long long)T, (int)D, (float)ctx->saved_data["eps"].toDouble(),
                (int)ctx->saved_data["form"].toInt(), type_code(type), stream());
        dwn = column_sums(f32(dg), parts, D, type, dev);
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
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !s.requires_grad(), what, ": scales carry no gradient");
}
// A weight as the product reads it: the caller's codes, or packed ones of a tensor
struct BlockWeight {
  Tensor q;
  OptTensor s;
  Operand operand;
};
BlockWeight block_weight(const Tensor& w, const OptTensor& ws) {
  if (ws.has_value()) {
    const Coded c{readable_codes(w), *ws};
    return {c.q, c.s, operand(c)};
  }
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  const Packed p(w.size(0), w.size(1), BY_TILES);
  const Tensor buf = p.make(w.device());
  quantize(flat(w), BY_TILES, p.in(buf), Operand());
  return {buf, std::nullopt, p.in(buf)};
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
  const Tensor x2 = flat(x);
  const int64_t R = x2.size(0), C = x2.size(1);
  const Coded c{codes(R, C, x.device()), tiles ? alloc({blocks(R), blocks(C)}, F32, x.device()) : row_scales(x, R, C)};
  quantize(x2, tiles ? BY_TILES : BY_ROWS, {ptr(c.q), f32(c.s), R, C}, Operand());
  return {x.dim() == 2 ? c.q : c.q.view(x.sizes()), c.s};
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
  const int64_t D = x.size(-1), T = x.numel() / D;
  const Coded c{codes(T, D, x.device()), row_scales(x, T, D)};
  const BlockNorm n = block_norm(x, residual, g, eps, form, false, {ptr(c.q), f32(c.s), T, D, up_to(D, 16)});
  return std::make_tuple(x.dim() == 2 ? c.q : c.q.view(x.sizes()), c.s, n.s);
}
// type: of the result
// kept: codes and scales of a weight tensor that its owner keeps between updates (quantised here otherwise)
Tensor linear_fp8_block(const Tensor& x, const OptTensor& xs, const py::object& weight, const OptTensor& ws, const OptTensor& bias, const OptTensor& residual,
                        int64_t type_, const OptTensor& kept_q, const OptTensor& kept_s) {
  const char* what = "linear_fp8_block";
  const at::ScalarType type = type_ == 0 ? BF16 : type_ == 1 ? at::kHalf : F32;
  const Tensor w = weight.cast<Tensor>();
  no_tangents({&x, &w, given(bias), given(residual)});
  if (xs.has_value()) check_coded(what, x, *xs, false);
  else check_block_input(what, x);
  const int64_t K = x.size(-1), T = x.numel() / K;
  TORCH_CHECK_VALUE(K <= MAX_BLOCK_SIZE && T <= MAX_BLOCK_SIZE, what, " takes up to ", MAX_BLOCK_SIZE, " rows of as many values, got ", x.sizes());
  check_projection(what, x, K, w, ws, bias, residual, type, w.dim() == 2 ? with_last(x.sizes(), w.size(0)) : x.sizes().vec());
  const c10::cuda::CUDAGuard device(x.device());
  const BlockWeight wc = kept_q.has_value() ? block_weight(*kept_q, kept_s) : block_weight(w, ws);
  const OptTensor b = contiguous(bias);
  const OptTensor wt = ws.has_value() ? OptTensor() : OptTensor(w);
  if (wants_grad({&x, given(wt), given(bias), given(residual)})) {
    TORCH_CHECK_VALUE(!xs.has_value(), what, ": inputs in 8 bits carry no gradient; call it under torch.no_grad, or with the tensor itself");
    return BlockLinear::apply(x, wt, b, residual, wc.q, wc.s, !ws.has_value() && fused(weight), wants_grad({given(wt)}), type, wc.operand);
  }
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  const Tensor r2 = residual.has_value() ? flat(*residual) : Tensor();
  Tensor y;
  if (xs.has_value()) {
    const Coded c{readable_codes(x.dim() == 2 ? x : x.reshape({T, K})), xs->dim() == 2 ? *xs : xs->reshape({T, blocks(K)})};
    y = block_forward(operand(c), wc.operand, type, x.device(), opt(b), r2, false);
  } else {
    const Tensor x2 = flat(x);
    const Packed p(T, K, BY_ROWS);
    const Tensor buf = p.make(x.device());
    quantize(x2, BY_ROWS, p.in(buf), Operand());
    y = block_forward(p.in(buf), wc.operand, type, x.device(), opt(b), r2, true);
  }
  return x.dim() == 2 ? y : y.view(with_last(x.sizes(), w.size(0)));
}
// nothing where the kernels do not cover the width
std::optional<std::tuple<Tensor, Tensor>> norm_linear_fp8_block(const Tensor& x, const Tensor& g, double eps, int64_t form, const py::object& weight, const OptTensor& ws,
                                                                const OptTensor& bias, const OptTensor& residual, const OptTensor& kept_q,
                                                                const OptTensor& kept_s) {
  const char* what = "norm_linear_fp8_block";
  const Tensor w = weight.cast<Tensor>();
  no_tangents({&x, &g, &w, given(bias), given(residual)});
  check_norm(what, x, g, residual);
  const int64_t K = x.size(-1);
  check_projection(what, x, K, w, ws, bias, OptTensor(), x.scalar_type(), {});
  const OptTensor wt = ws.has_value() ? OptTensor() : OptTensor(w);
  const bool train = wants_grad({&x, &g, given(wt), given(bias), given(residual)});
  if (K > 16384) return std::nullopt;
  const c10::cuda::CUDAGuard device(x.device());
  const BlockWeight wc = kept_q.has_value() ? block_weight(*kept_q, kept_s) : block_weight(w, ws);
  const OptTensor b = contiguous(bias);
  if (train) {
    variable_list r = BlockNormLinear::apply(x, residual, g, wt, b, wc.q, wc.s, eps, form, !ws.has_value() && fused(weight), wc.operand);
    return std::make_tuple(r[0], r[1]);
  }
  const at::AutoDispatchBelowADInplaceOrView no_graph;
  const Packed p(x.numel() / K, K, BY_ROWS);
  const Tensor buf = p.make(x.device());
  const BlockNorm n = block_norm(x, residual, g, eps, form, false, p.in(buf));
  const Tensor y = block_forward(p.in(buf), wc.operand, x.scalar_type(), x.device(), opt(b), Tensor(), true);
  return std::make_tuple(x.dim() == 2 ? y : y.view(with_last(x.sizes(), w.size(0))), n.s);
}
