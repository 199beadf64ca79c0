// Host path of rotate_heads (part of host.cpp, which includes it): argument checks, allocations, calls and the autograd node.

// Which pairs of a row turn, by which axis and how far for each step. The steps live on the device; a call on another stream than the one they were made on, or a
// captured one, keeps them.
struct Rotation {
  Tensor steps;   // int64 (rotated / 2): fractions of 2^64 turns
  int32_t head_dim, rotated, interleaved, axes, ends[2] = {0, 0};
  at::cuda::CUDAStream made_on;
  std::atomic<unsigned long long> held_by{0};   // the last capture whose graph has been given it to hold

  Rotation(const Tensor& steps_, int64_t head_dim_, bool interleaved_, const std::vector<int64_t>& sections)
      : steps(steps_), made_on(stream_of(steps_)) {
    KD_VALUE(steps.dim() == 1 && steps.scalar_type() == at::kLong && steps.is_contiguous(), "steps must be a contiguous int64 vector");
    head_dim = static_cast<int32_t>(head_dim_);
    rotated = static_cast<int32_t>(2 * steps.size(0));
    interleaved = interleaved_ ? 1 : 0;
    axes = static_cast<int32_t>(std::max<size_t>(sections.size(), 1));
    int64_t sum = 0;
    for (size_t i = 0; i < sections.size(); ++i) {
      sum += sections[i];
      if (i < 2) ends[i] = static_cast<int32_t>(sum);
    }
    if (sections.empty()) ends[0] = rotated / 2;
  }
  Rotation(const Rotation&) = delete;
  static at::cuda::CUDAStream stream_of(const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "rotate_heads runs on CUDA sm_100 devices only; there is no CPU path");
    return at::cuda::getCurrentCUDAStream(t.device().index());
  }
};
using RotationPtr = std::shared_ptr<Rotation>;

// What a call has besides its heads.
struct RotateArgs {
  RotationPtr rotation;
  Tensor positions, offsets;   // as the kernel takes them, or undefined
  double eps;
};

kd_rotation rotation_params(const RotateArgs& a, const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& offsets, const Tensor& q_weight, const Tensor& k_weight) {
  const Rotation& r = *a.rotation;
  kd_rotation p{};
  p.B = static_cast<int32_t>(q.size(0));
  p.Hq = static_cast<int32_t>(q.size(1));
  p.Hk = k.defined() ? static_cast<int32_t>(k.size(1)) : 0;
  p.T = static_cast<int32_t>(q.size(2));
  p.D = static_cast<int32_t>(q.size(3));
  p.R = r.rotated;
  p.dtype = p.w_dtype = dtype_code(q.scalar_type());
  for (const Tensor* w : {&q_weight, &k_weight})
    if (w->defined()) p.w_dtype = dtype_code(w->scalar_type());
  p.q_weight = q_weight.defined() ? q_weight.const_data_ptr() : nullptr;
  p.k_weight = k_weight.defined() ? k_weight.const_data_ptr() : nullptr;
  p.steps = reinterpret_cast<const uint64_t*>(r.steps.const_data_ptr<int64_t>());
  p.axes = r.axes;
  p.ends[0] = r.ends[0];
  p.ends[1] = r.ends[1];
  p.interleaved = r.interleaved;
  p.eps = static_cast<float>(a.eps);
  if (positions.defined()) {
    p.positions = positions.const_data_ptr();
    p.pos_is_64 = positions.scalar_type() == at::kLong ? 1 : 0;
    const int64_t d = positions.dim();
    p.pos_stride_a = d == 3 && positions.size(0) > 1 ? positions.stride(0) : 0;
    p.pos_stride_b = positions.size(d - 2) > 1 ? positions.stride(d - 2) : 0;
    p.pos_stride_t = positions.stride(d - 1);
  }
  if (offsets.defined()) p.offsets = offsets.const_data_ptr<int32_t>();
  return p;
}

void launch_rotation(const RotationPtr& r, const kd_rotation& p, bool grad) {
  const auto current = at::cuda::getCurrentCUDAStream();
  const cudaStream_t stream = current.stream();
  const Capture capture(stream);
  hold_for_graph(r, r->held_by, capture);
  let_go().clear();
  if (current != r->made_on) c10::cuda::CUDACachingAllocator::recordStream(r->steps.storage().data_ptr(), current);
  check(grad ? lib.rotate_grad(&p, stream) : lib.rotate(&p, stream));
}

// A tensor for what a kernel writes in the memory of `like` (or contiguous): `out`, or where rows of that are not 16-byte pieces one that is copied there at last.
struct RowsOut {
  Tensor out, rows;
  explicit RowsOut(Tensor out_) : out(std::move(out_)), rows(aligned(out) ? out : empty_on(out.sizes(), out.scalar_type(), out.device())) {}
  const Tensor& finish() {
    if (!rows.is_same(out)) out.copy_(rows);
    return out;
  }
};

// What is known of an output when its memory is gone: its gradient's, and that of the gradient of what it was made from, which has the same layout.
struct Geometry {
  std::vector<int64_t> sizes, strides;
  at::ScalarType type;
  std::optional<at::Device> device;
  void operator=(const Tensor& t) {
    sizes = t.sizes().vec();
    strides = t.strides().vec();
    type = t.scalar_type();
    device = t.device();
  }
  Tensor zeros() const { return at::zeros(sizes, at::TensorOptions().dtype(type).device(*device)); }
  Tensor empty() const {
    if (allocations_are_seen()) return at::empty_strided(sizes, strides, at::TensorOptions().dtype(type).device(*device));
    return Tensor(at::detail::empty_strided_cuda(sizes, strides, type, *device));
  }
};

struct RotateBackward : torch::autograd::Node {
  torch::autograd::SavedVariable q, k, q_weight, k_weight, positions, offsets;
  RotateArgs args;
  Geometry q_like, k_like;
  bool has_k, has_qw, has_kw;
  bool history_lost = false;   // (under mutex_)

  // Gradients have no history of their own. Where they are to have one (create_graph) and depend on what is differentiated, that is said. A loss with such gradients in it and other terms
  // comes through this node again, and would lack their part: that is refused.
  void refuse_lost_history(const torch::autograd::variable_list& grads) {
    TORCH_CHECK(!history_lost,
                "rotate_heads is differentiable once: an earlier backward pass through this call, with create_graph=True, gave gradients without a history, and what depends on them would be missing "
                "from this one. Use retain_graph=True where no second derivative is wanted");
    if (!at::GradMode::is_enabled()) return;
    for (int i = 0; i < (has_k ? 2 : 1); ++i) {
      const bool row = next_edge(i).is_valid(), weight = next_edge(i + 2).is_valid(), norm = i == 0 ? has_qw : has_kw;
      history_lost = history_lost || ((row || weight) && grads[i].defined() && grads[i].requires_grad()) || (row && norm);
    }
    if (history_lost) TORCH_WARN("rotate_heads is differentiable once: with create_graph=True its gradients have no history, and second derivatives through them will be missing");
  }

  // A gradient that is added to a leaf in a captured backward pass is added on the stream that the leaf's first graph was made on, while that lives: where that is not the capturing
  // one, torch's engine ends the process. So this is refused before it comes to that.
  void refuse_foreign_leaves() {
    const auto current = at::cuda::getCurrentCUDAStream();
    if (!Capture(current.stream()).active) return;
    const auto* asked = torch::autograd::get_current_graph_task_exec_info();
    const bool all = asked == nullptr || asked->empty();   // else only those asked for by name: torch.autograd.grad hands their gradients out, backward(inputs=...) adds them
    for (const auto& edge : next_edges())
      if (auto* leaf = dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get())) {
        if (!all) {
          const auto named = asked->find(leaf);
          if (named == asked->end() || !named->second.needed_) continue;
        }
        const auto stream = leaf->stream();
        TORCH_CHECK(!stream.has_value() || *stream == current.unwrap(),
                    "a backward pass of rotate_heads cannot be captured while an earlier graph of the same leaves lives: its gradients are added on that graph's stream. "
                    "Let go of the earlier graph, or use torch.autograd.grad");
      }
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    torch::autograd::variable_list result(4);
    Tensor tq, tk, tqw, tkw, tp, to;
    {
      std::lock_guard<std::mutex> lock(mutex_);
      refuse_lost_history(grads);
      tq = q.unpack();
      tk = k.unpack();
      tqw = q_weight.unpack();
      tkw = k_weight.unpack();
      tp = positions.unpack();
      to = offsets.unpack();
    }
    refuse_foreign_leaves();
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(*q_like.device);
    // undefined gradients count as zeros; others are brought to what the kernel reads
    auto gradient = [&](const Tensor& g, const Geometry& like) {
      if (!g.defined()) return like.zeros();
      KD_VALUE(g.sizes() == at::IntArrayRef(like.sizes) && g.device() == *like.device, "the gradient of an output of shape ", like.sizes, " on ", *like.device, " has shape ", g.sizes(),
               " on ", g.device());
      return rows16(g.scalar_type() == like.type ? g : g.to(like.type));
    };
    // (saved tensors may have been moved and brought back with other strides)
    if (tq.defined()) tq = rows16(tq);
    if (tk.defined()) tk = rows16(tk);
    if (tqw.defined()) tqw = tqw.contiguous();
    if (tkw.defined()) tkw = tkw.contiguous();
    const Tensor gq = gradient(grads[0], q_like), gk = has_k ? gradient(grads[1], k_like) : Tensor();
    RowsOut dq(q_like.empty());
    std::optional<RowsOut> dk;
    if (has_k) dk.emplace(k_like.empty());
    kd_rotation p = rotation_params(args, gq, gk, tp, to, tqw, tkw);
    p.q_out = desc(gq);
    p.dq = desc(dq.rows);
    if (tq.defined()) p.q = desc(tq);
    if (has_k) {
      p.k_out = desc(gk);
      p.dk = desc(dk->rows);
      if (tk.defined()) p.k = desc(tk);
    }
    Tensor dqw, dkw, workspace;
    const bool empty = p.B == 0 || p.T == 0;
    auto weight = [&](const Tensor& w, bool wanted, void*& slot) {
      if (!wanted) return Tensor();
      if (empty) return at::zeros_like(w);
      Tensor d = empty_on(w.sizes(), w.scalar_type(), w.device());
      slot = d.data_ptr();
      return d;
    };
    if (has_qw) dqw = weight(tqw, task_should_compute_output(2), p.dq_weight);
    if (has_kw) dkw = weight(tkw, task_should_compute_output(3), p.dk_weight);
    size_t bytes = 0;
    check(lib.rotate_grad_workspace(&p, &bytes));
    if (bytes > 0) {
      workspace = empty_on({static_cast<int64_t>(bytes)}, at::kByte, *q_like.device);
      p.workspace = workspace.data_ptr();
    }
    launch_rotation(args.rotation, p, true);
    result[0] = dq.finish();
    if (has_k) result[1] = dk->finish();
    result[2] = dqw;
    result[3] = dkw;
    return result;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* s : {&q, &k, &q_weight, &k_weight, &positions, &offsets}) s->reset_data();
  }
  std::string name() const override { return "RotateHeadsBackward"; }
};

void check_rotated(const Rotation& r, const Tensor& x, const char* name, const Tensor& q) {
  KD_VALUE(x.dim() == 4, name, " must be (batch, heads, time, head_dim)");
  TORCH_CHECK(x.is_cuda(), "rotate_heads runs on CUDA sm_100 devices only; there is no CPU path");
  const auto t = x.scalar_type();
  KD_VALUE((t == at::kHalf || t == at::kBFloat16 || t == at::kFloat) && t == q.scalar_type(), "q and k must share dtype float16, bfloat16 or float32");
  KD_VALUE(x.size(3) == r.head_dim, name, " has head_dim ", x.size(3), ", the rotation ", r.head_dim);
  KD_VALUE(x.size(0) == q.size(0) && x.size(2) == q.size(2), "q and k must have the same batch and time, got ", q.sizes(), ", ", x.sizes());
  KD_VALUE(x.size(1) >= 1 && x.size(1) <= 65535, name, " must have from 1 to 65535 heads");
  KD_VALUE(x.device() == q.device() && r.steps.device() == q.device(), "q, k and the rotation must be on the same device");
}

std::tuple<Tensor, Tensor> rotate_heads(const Tensor& q_, const OptTensor& k_, const RotationPtr& rotation, const OptTensor& positions_, const OptTensor& offsets_,
                                        const OptTensor& q_weight_, const OptTensor& k_weight_, double eps, bool like_input) {
  const Rotation& r = *rotation;
  check_rotated(r, q_, "q", q_);
  if (k_.has_value()) check_rotated(r, *k_, "k", q_);
  const int64_t B = q_.size(0), T = q_.size(2), D = q_.size(3);
  KD_VALUE(B <= INT32_MAX && T <= INT32_MAX && B * T <= INT32_MAX - 256, "too many tokens");
  KD_VALUE(eps >= 0.0 && eps < 1e30, "eps must not be negative, and finite");
  KD_VALUE(k_.has_value() || !k_weight_.has_value(), "k_weight is given, k is not");
  at::ScalarType w_type = at::kByte;
  for (const OptTensor* w : {&q_weight_, &k_weight_}) {
    if (!w->has_value()) continue;
    const auto t = (*w)->scalar_type();
    KD_VALUE((*w)->dim() == 1 && (*w)->size(0) == D, "weights must have shape (head_dim,) = (", D, ",), got ", (*w)->sizes());
    KD_VALUE((t == at::kHalf || t == at::kBFloat16 || t == at::kFloat) && (w_type == at::kByte || t == w_type), "weights must share dtype float16, bfloat16 or float32");
    KD_VALUE((*w)->device() == q_.device(), "weights must live on ", q_.device());
    w_type = t;
  }
  RotateArgs args{rotation, {}, {}, eps};
  KD_VALUE(r.axes == 1 || positions_.has_value(), "a rotation by ", r.axes, " axes needs positions");
  KD_VALUE(!(positions_.has_value() && offsets_.has_value()), "positions and offsets exclude one another");
  if (positions_.has_value()) {
    const Tensor& p = *positions_;
    const int64_t d = p.dim();
    KD_VALUE(p.scalar_type() == at::kLong || p.scalar_type() == at::kInt, "positions must be int64 or int32");
    KD_VALUE((d == 3 && p.size(0) == r.axes) || (d == 2 && r.axes == 1), "positions must have shape (axes, batch, time) with ", r.axes, " axes", r.axes == 1 ? ", or (batch, time)" : "",
             ", got ", p.sizes());
    KD_VALUE((p.size(d - 2) == B || p.size(d - 2) == 1) && p.size(d - 1) == T, "positions must be for ", B, " sequences (or 1) of ", T, " tokens, got ", p.sizes());
    KD_VALUE(p.device() == q_.device(), "positions must live on ", q_.device());
    args.positions = p;
  }
  if (offsets_.has_value()) {
    const Tensor& o = *offsets_;
    KD_VALUE(o.dim() == 1 && o.size(0) == B && o.scalar_type() == at::kInt, "offsets must be an int32 tensor of shape (batch,) = (", B, ",)");
    KD_VALUE(o.device() == q_.device(), "offsets must live on ", q_.device());
    args.offsets = o.contiguous();
  }
  const Tensor kv = k_.value_or(Tensor()), qw_ = q_weight_.value_or(Tensor()), kw_ = k_weight_.value_or(Tensor());
  bool track = false;
  for (const Tensor* t : {&q_, &kv, &qw_, &kw_}) {
    if (!t->defined()) continue;
    refuse_forward_ad("rotate_heads", *t);
    track = track || t->requires_grad();
  }
  track = track && at::GradMode::is_enabled();
  refuse_tracing("rotate_heads");
  Tensor q, k, qw, kw, q_out, k_out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::cuda::CUDAGuard guard(q_.device());
    q = rows16(q_);
    RowsOut yq(empty_out(q_, like_input));
    std::optional<RowsOut> yk;
    if (kv.defined()) {
      k = rows16(kv);
      yk.emplace(empty_out(kv, like_input));
    }
    if (qw_.defined()) qw = qw_.contiguous();
    if (kw_.defined()) kw = kw_.contiguous();
    kd_rotation p = rotation_params(args, q, k, args.positions, args.offsets, qw, kw);
    p.q = desc(q);
    p.q_out = desc(yq.rows);
    if (k.defined()) {
      p.k = desc(k);
      p.k_out = desc(yk->rows);
    }
    launch_rotation(rotation, p, false);
    q_out = yq.finish();
    if (k.defined()) k_out = yk->finish();
  }
  if (track) {
    using torch::autograd::SavedVariable;
    auto node = std::shared_ptr<RotateBackward>(new RotateBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q_, kv, qw_, kw_));
    node->has_k = k.defined();
    node->has_qw = qw.defined();
    node->has_kw = kw.defined();
    node->q_like = q_out;
    if (k.defined()) node->k_like = k_out;
    torch::autograd::set_history(q_out, node);
    if (k.defined()) torch::autograd::set_history(k_out, node);
    // (rows that have no norm are not read again)
    if (qw.defined()) node->q = SavedVariable(q, false);
    if (kw.defined()) node->k = SavedVariable(k, false);
    if (qw.defined()) node->q_weight = SavedVariable(qw, false);
    if (kw.defined()) node->k_weight = SavedVariable(kw, false);
    if (args.positions.defined()) node->positions = SavedVariable(args.positions, false);
    if (args.offsets.defined()) node->offsets = SavedVariable(args.offsets, false);
    args.positions = args.offsets = Tensor();   // (the saved ones are what the backward reads)
    node->args = std::move(args);
  }
  return {q_out, k_out};
}
