// Layer normalisation and attention on tensors; part of host.cpp, inside its namespace.

int feature_type(const Tensor &t, const char *what) {
  if (t.scalar_type() == at::kFloat) return MCCNN_FLOAT32;
  if (t.scalar_type() == at::kBFloat16) return MCCNN_BFLOAT16;
  throw InvalidArgument(std::string(what) + " expects float32 or bfloat16 features, got " +
                        c10::toString(t.scalar_type()));
}

void expect(bool ok, const std::string &message) {
  if (!ok) throw InvalidArgument(message);
}
std::string shape_of(const Tensor &t) {
  std::ostringstream s;
  s << t.sizes();
  return s.str();
}

// The kernels are launched on the current stream of the current device.
void expect_current_device(const Tensor &t, const char *what) {
  TORCH_CHECK_TYPE(t.is_cuda(), what, " expects GPU tensors, got one on ", t.device());
  int d = 0;
  hip_check(hipGetDevice(&d));
  expect(t.get_device() == d, std::string(what) + " expects tensors on the current device");
}
void expect_beside(const Tensor &t, const Tensor &first, const char *what) {
  expect(!t.defined() || t.device() == first.device(), std::string(what) + " got tensors on different devices");
}

// -------------------------------------------------------------------- layer norm ----

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  // `x` is contiguous already: a copy made in here would be saved without its history, and gradients
  // that are themselves differentiated would not reach the features.
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &weight_,
                        const OptTensor &bias_, double eps, bool keep) {
    const Tensor weight = opt(weight_), bias = opt(bias_);
    const int type = feature_type(x, "layer_norm");
    const int64_t cols = x.size(-1), rows = cols ? x.numel() / cols : 0;
    Tensor y = at::empty_like(x), stats;  // (means, then 1 / deviations)
    if (keep) stats = empty_f32({2, rows}, x);
    hipStream_t s = current_stream();
    {
      Region t("layer_norm", s);
      check(mccnn_layer_norm(s, type, rows, (int)cols, x.data_ptr(), f32(weight), f32(bias), (float)eps,
                             y.data_ptr(), f32(stats), keep ? f32(stats) + rows : nullptr));
    }
    if (keep) {
      ctx->save_for_backward({x, weight, bias, stats});
      ctx->saved_data["eps"] = eps;
    }
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grad_out) {
    const auto v = ctx->get_saved_variables();
    const Tensor &x = v[0], &weight = v[1], &bias = v[2];
    variable_list grads(5);
    if (recording_gradients()) {          // gradients of gradients: through torch's operations
      const Tensor z = x.to(at::kFloat), centred = z - z.mean(-1, true);
      Tensor y = centred * (centred.square().mean(-1, true) + ctx->saved_data["eps"].toDouble()).rsqrt();
      if (weight.defined()) y = y * weight;
      if (bias.defined()) y = y + bias;
      y = y.to(x.scalar_type());
      variable_list wanted;
      std::vector<size_t> slots;
      for (size_t i = 0; i < 3; ++i)
        if (v[i].defined() && v[i].requires_grad()) {
          wanted.push_back(v[i]);
          slots.push_back(i);
        }
      const auto g = torch::autograd::grad({y}, wanted, {grad_out[0]}, true, true);
      for (size_t i = 0; i < slots.size(); ++i) grads[slots[i]] = g[i];
      return grads;
    }
    const Tensor g = grad_out[0].contiguous();
    const int64_t cols = x.size(-1), rows = v[3].size(1);
    const float *stats = f32(v[3]);
    const bool sums = (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad());
    if (ctx->needs_input_grad(0)) grads[0] = at::empty_like(x);
    Tensor ws, dw, db;
    if (sums) {
      dw = empty_f32({cols}, x);
      db = empty_f32({cols}, x);
      ws = workspace(mccnn_layer_norm_grads_workspace_bytes(rows, (int)cols), x);
    }
    hipStream_t s = current_stream();
    Region t("layer_norm_grads", s);
    check(mccnn_layer_norm_grads(s, feature_type(x, "layer_norm"), rows, (int)cols, x.data_ptr(), f32(weight), stats,
                                 stats + rows, g.data_ptr(), sums ? ws.data_ptr() : nullptr, sums ? ws.numel() : 0,
                                 grads[0].defined() ? grads[0].data_ptr() : nullptr, f32(dw), f32(db)));
    if (weight.defined()) grads[1] = dw;
    if (bias.defined()) grads[2] = db;
    return grads;
  }
};

bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

Tensor layer_norm(const Tensor &features, const OptTensor &weight, const OptTensor &bias, double eps) {
  feature_type(features, "layer_norm");
  expect(features.dim() >= 1 && features.size(-1) >= 1, "layer_norm expects rows of at least one channel");
  expect(eps >= 0.0, "layer_norm expects an epsilon of at least 0");
  for (const Tensor &t : {opt(weight), opt(bias)}) {
    expect_beside(t, features, "layer_norm");
    expect(!t.defined() || (t.dim() == 1 && t.size(0) == features.size(-1)),
           "layer_norm expects a weight and a bias per channel");
  }
  expect_current_device(features, "layer_norm");
  for (const Tensor &t : {opt(weight), opt(bias)}) (void)f32(t);     // (type and layout)
  const bool keep = at::GradMode::is_enabled() &&
                    (wants_grad(features) || wants_grad(opt(weight)) || wants_grad(opt(bias)));
  return LayerNorm::apply(features.contiguous(), weight, bias, eps, keep);
}

// --------------------------------------------------------------------- attention ----

// What a call is about, in the order in which it is saved for the gradient.
enum { kQ, kK, kV, kTable, kQSplits, kKSplits, kKSizes, kKeyMask, kBuckets, kQPos, kKPos, kNumOperands };

mccnn_attention describe(const variable_list &t, bool causal, double scale) {
  mccnn_attention a{};
  const Tensor &q = t[kQ], &k = t[kK], &v = t[kV], &table = t[kTable];
  a.dtype = feature_type(q, "packed_attention");
  a.heads = (int)q.size(1);
  a.kv_heads = (int)k.size(1);
  a.dim = (int)q.size(2);
  a.clouds = t[kQSplits].defined() ? (int)t[kQSplits].size(0) - 1 : 1;
  a.causal = causal;
  a.num_q = q.size(0);
  a.num_k = k.size(0);
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.q_row = q.stride(0);
  a.q_head = q.stride(1);
  a.k_row = k.stride(0);
  a.k_head = k.stride(1);
  a.v_row = v.stride(0);
  a.v_head = v.stride(1);
  a.q_splits = i32(t[kQSplits]);
  a.k_splits = i32(t[kKSplits]);
  a.k_sizes = i32(t[kKSizes]);
  a.key_mask = static_cast<uint8_t *>(raw(t[kKeyMask], at::kBool));
  a.scale = (float)scale;
  if (table.defined()) {
    a.axes = (int)table.size(0);
    a.num_buckets = (int)table.size(1);
    a.max_offset = (int)(t[kBuckets].size(0) / 2);
    a.table = f32(table);
    a.buckets = i32(t[kBuckets]);
    a.q_pos = i32(t[kQPos]);
    a.k_pos = i32(t[kKPos]);
  }
  return a;
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                        const OptTensor &table, const variable_list &others, bool causal, double scale, bool keep) {
    variable_list t{q, k, v, opt(table)};
    for (int i = 0; i < 3; ++i)           // channels one after the other; rows and heads as they are
      if (t[i].size(2) > 1 && t[i].stride(2) != 1) t[i] = t[i].contiguous();
    t.insert(t.end(), others.begin(), others.end());
    const mccnn_attention a = describe(t, causal, scale);
    Tensor out = at::empty({a.num_q, a.heads, a.dim}, q.options().requires_grad(false));
    Tensor low, stats;                    // (maxima, then sums)
    if (keep) {
      if (a.dtype != MCCNN_FLOAT32) low = empty_f32(out.sizes(), q);
      stats = empty_f32({2, a.heads, a.num_q}, q);
    }
    const int64_t rows = (int64_t)a.heads * a.num_q;
    const size_t bytes = mccnn_attention_workspace_bytes(&a);
    Tensor ws;
    if (bytes) ws = workspace(bytes, q);
    hipStream_t s = current_stream();
    {
      Region r("packed_attention", s);
      check(mccnn_attention_forward(s, &a, bytes ? ws.data_ptr() : nullptr, bytes, out.data_ptr(),
                                    low.defined() ? f32(low) : nullptr, f32(stats),
                                    keep ? f32(stats) + rows : nullptr));
    }
    if (keep) {
      t.insert(t.end(), {out, low, stats});
      ctx->save_for_backward(t);
      ctx->saved_data["causal"] = causal;
      ctx->saved_data["scale"] = scale;
    }
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grad_out) {
    if (recording_gradients())
      throw std::runtime_error("packed_attention has no gradient of its gradient");
    const auto t = ctx->get_saved_variables();
    const mccnn_attention a = describe(t, ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
    const Tensor g = grad_out[0].contiguous();
    const Tensor &out = t[kNumOperands], &low = t[kNumOperands + 1];
    const float *top = f32(t[kNumOperands + 2]);
    variable_list grads(15);               // (undefined for what is no tensor)
    const auto like = [&](const Tensor &x) { return at::empty(x.sizes(), x.options().requires_grad(false)); };
    grads[0] = like(t[kQ]);
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
      grads[1] = like(t[kK]);
      grads[2] = like(t[kV]);
    }
    const bool table = t[kTable].defined() && ctx->needs_input_grad(3);
    if (table) grads[3] = empty_f32(t[kTable].sizes(), t[kTable]);
    const size_t bytes = mccnn_attention_grads_workspace_bytes(&a, table);
    Tensor ws = workspace(bytes, g);
    hipStream_t s = current_stream();
    Region r("packed_attention_grads", s);
    check(mccnn_attention_grads(s, &a, out.data_ptr(), low.defined() ? f32(low) : nullptr, top,
                                top + (int64_t)a.heads * a.num_q, g.data_ptr(), ws.data_ptr(), bytes, grads[0].data_ptr(),
                                grads[1].defined() ? grads[1].data_ptr() : nullptr,
                                grads[2].defined() ? grads[2].data_ptr() : nullptr, f32(grads[3])));
    return grads;
  }
};

Tensor packed_attention(const Tensor &q, const Tensor &k, const Tensor &v, const OptTensor &q_splits_,
                        const OptTensor &k_splits_, const OptTensor &k_sizes_, const OptTensor &key_mask_, bool causal,
                        std::optional<double> scale, const OptTensor &table_, const OptTensor &buckets_,
                        const OptTensor &q_pos_, const OptTensor &k_pos_) {
  const char *what = "packed_attention";
  feature_type(q, what);
  expect(q.dim() == 3 && k.dim() == 3 && v.dim() == 3,
         "packed_attention expects queries, keys and values [rows, heads, channels], got " + shape_of(q) + ", " +
             shape_of(k) + " and " + shape_of(v));
  expect(k.sizes() == v.sizes(), "packed_attention expects a value per key, got " + shape_of(v) + " for " + shape_of(k));
  expect(q.size(2) == k.size(2), "packed_attention expects queries and keys of as many channels, got " + shape_of(q) +
                                     " and " + shape_of(k));
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                   "expected queries, keys and values of one dtype, got ", q.scalar_type(), ", ", k.scalar_type(),
                   " and ", v.scalar_type());
  // (sizes that the C ABI takes as int)
  expect(q.size(1) >= 1 && q.size(1) <= 65535 && k.size(1) >= 1 && q.size(1) % k.size(1) == 0,
         "packed_attention expects the query heads to be a multiple of the key heads, got " + shape_of(q) + " and " +
             shape_of(k));
  expect(q.size(2) >= 1 && q.size(2) <= 128, "packed_attention expects 1 to 128 channels per head, got " + shape_of(q));
  const Tensor q_splits = opt(q_splits_), k_splits = opt(k_splits_), k_sizes = opt(k_sizes_), mask = opt(key_mask_),
               table = opt(table_), buckets = opt(buckets_), q_pos = opt(q_pos_), k_pos = opt(k_pos_);
  for (const Tensor &t : {k, v, q_splits, k_splits, k_sizes, mask, table, buckets, q_pos, k_pos})
    expect_beside(t, q, what);
  expect(q_splits.defined() == k_splits.defined(), "packed_attention expects row splits of both sides or of neither");
  int64_t clouds = 1;
  if (q_splits.defined()) {
    expect(q_splits.dim() == 1 && k_splits.dim() == 1 && q_splits.size(0) >= 1 && q_splits.sizes() == k_splits.sizes(),
           "packed_attention expects row splits [clouds + 1] of both sides, got " + shape_of(q_splits) + " and " +
               shape_of(k_splits));
    clouds = q_splits.size(0) - 1;
  }
  expect(clouds <= (1 << 24), "packed_attention expects at most 2^24 clouds");
  expect(!k_sizes.defined() || (k_sizes.dim() == 1 && k_sizes.size(0) == clouds),
         "packed_attention expects a key size per cloud, got " + (k_sizes.defined() ? shape_of(k_sizes) : ""));
  expect(!mask.defined() || (mask.dim() == 1 && mask.size(0) == k.size(0)),
         "packed_attention expects a mask value per key, got " + (mask.defined() ? shape_of(mask) : ""));
  expect(table.defined() == buckets.defined(), "packed_attention expects a bias table and its buckets, or neither");
  expect(q_pos.defined() == k_pos.defined() && (table.defined() || !q_pos.defined()),
         "packed_attention expects positions of both sides, with a bias table, or none");
  if (table.defined()) {
    expect(table.dim() == 3 && table.size(0) >= 1 && table.size(0) <= 3 && table.size(1) >= 1 &&
               table.size(1) <= (1 << 24) && table.size(2) == q.size(1),
           "packed_attention expects a bias table [1 to 3 axes, buckets, heads], got " + shape_of(table) + " for " +
               std::to_string(q.size(1)) + " heads");
    expect(buckets.dim() == 1 && buckets.size(0) % 2 == 1 && buckets.size(0) <= (1 << 24),
           "packed_attention expects buckets of the offsets -R to R, got " + shape_of(buckets));
    expect(table.size(0) * buckets.size(0) <= MCCNN_ATTENTION_MAX_OFFSETS,
           "packed_attention expects a bias of at most " + std::to_string(MCCNN_ATTENTION_MAX_OFFSETS) +
               " offsets over all axes, got " + std::to_string(table.size(0)) + " times " + std::to_string(buckets.size(0)));
    expect(q_pos.defined() || table.size(0) == 1,
           "packed_attention expects positions for a bias of " + std::to_string(table.size(0)) + " axes");
    for (const auto &side : {std::make_pair(q_pos, q), std::make_pair(k_pos, k)})
      expect(!side.first.defined() || (side.first.dim() == 2 && side.first.size(0) == side.second.size(0) &&
                                       side.first.size(1) == table.size(0)),
             "packed_attention expects a position per row and axis, got " +
                 (side.first.defined() ? shape_of(side.first) : ""));
  }
  const double factor = scale.has_value() ? *scale : 1.0 / std::sqrt((double)q.size(2));
  expect(factor > 0.0 && (float)factor > 0.0f && std::isfinite((float)factor),
         "packed_attention expects a finite scale above 0");
  expect_current_device(q, what);
  const variable_list others{q_splits, k_splits, k_sizes, mask, buckets, q_pos, k_pos};
  // (types and layouts, before the call is under way)
  for (const Tensor &t : {q_splits, k_splits, k_sizes, buckets, q_pos, k_pos}) (void)i32(t);
  (void)raw(mask, at::kBool);
  (void)f32(table);
  const bool keep = at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(v) || wants_grad(table));
  return PackedAttention::apply(q, k, v, table_, others, causal, factor, keep);
}
