// Host path of the 8-bit key/value cache (part of host.cpp, which includes it): argument checks, allocations and calls.

// A cache is the caller's tensors; its status word is a word of pinned memory that the kernels write when a length, a page number or
// a span id does not fit, or a bounded wait gave up. The next call looks at it without a synchronisation.
struct KVCache {
  Tensor k, v, k_scale, v_scale;
  OptTensor desc;
  std::shared_ptr<StatusMirror> mirror;
  std::atomic<unsigned long long> held_by{0};   // the last capture whose graph has been given the mirror to hold
  kd_cache abi{};

  KVCache(const Tensor& k_, const Tensor& v_, const Tensor& ks, const Tensor& vs, const OptTensor& d) : k(k_), v(v_), k_scale(ks), v_scale(vs), desc(d) {
    KD_VALUE(k.dim() == 4 && k.size(2) == KD_CACHE_PAGE, "k must be (pages, heads, ", KD_CACHE_PAGE, ", head_dim), got ", k.sizes());
    KD_VALUE(v.sizes() == k.sizes(), "k and v must have the same shape, got ", k.sizes(), ", ", v.sizes());
    KD_VALUE(k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn, "k and v must be float8_e4m3fn");
    const int64_t P = k.size(0), H = k.size(1), D = k.size(3);
    KD_VALUE(D % 16 == 0 && D >= 16 && D <= 128, "head_dim ", D, " is not supported (a multiple of 16 from 16 to 128)");
    KD_VALUE(P >= 1 && P <= INT32_MAX && H >= 1 && H <= INT32_MAX, "a cache has at least one page and one head, got ", k.sizes());
    for (const Tensor* s : {&k_scale, &v_scale})
      KD_VALUE(s->dim() == 2 && s->size(0) == P && s->size(1) == H && s->scalar_type() == at::kFloat, "scales must be float32 (pages, heads) = (", P, ", ", H, ")");
    if (desc.has_value())
      KD_VALUE(desc->dim() == 3 && desc->size(0) == P && desc->size(1) == H && desc->size(2) == KD_CACHE_PAGE && desc->scalar_type() == at::kInt,
               "desc must be int32 (pages, heads, ", KD_CACHE_PAGE, ")");
    TORCH_CHECK(k.is_cuda(), "the cache lives on CUDA sm_100 devices only; there is no CPU path");
    for (const Tensor* t : {&k, &v, &k_scale, &v_scale, desc.has_value() ? &*desc : &k}) {
      KD_VALUE(t->device() == k.device(), "the tensors of a cache must be on one device");
      KD_VALUE(t->is_contiguous() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0, "the tensors of a cache must be contiguous and 16-byte aligned");
    }
    mirror = std::make_shared<StatusMirror>();
    abi.k = k.data_ptr();
    abi.v = v.data_ptr();
    abi.k_scale = k_scale.data_ptr<float>();
    abi.v_scale = v_scale.data_ptr<float>();
    abi.desc = desc.has_value() ? reinterpret_cast<uint32_t*>(desc->data_ptr<int32_t>()) : nullptr;
    abi.pages = static_cast<int32_t>(P);
    abi.H = static_cast<int32_t>(H);
    abi.D = static_cast<int32_t>(D);
    abi.status_mirror = const_cast<uint32_t*>(mirror->at);
  }
  KVCache(const KVCache&) = delete;

  // before a call's launch: what earlier ones reported, and whether the addresses still are the tensors' (storages can be resized or replaced)
  void poll() {
    KD_VALUE(k.const_data_ptr() == abi.k && v.const_data_ptr() == abi.v && k_scale.const_data_ptr() == abi.k_scale && v_scale.const_data_ptr() == abi.v_scale &&
                 (abi.desc == nullptr || desc->const_data_ptr() == abi.desc),
             "the tensors of the cache have been given other memory: make a new KVCache of them");
    const uint32_t s = *mirror->at;
    if (s == 0) return;
    *mirror->at = 0;
    if ((s & (kStatusTimeout | kStatusSpanRange)) != 0) Plan::raise_status(s);
    KD_VALUE((s & 0xFu) != 1u, "an earlier call was given a sequence length, or a number of new tokens, outside what its page table holds");
    KD_VALUE(false, "an earlier call was given a page number outside the cache");
  }
  // A captured launch writes to the status word at every replay, whatever has become of this handle.
  Capture before_launch(cudaStream_t stream) {
    const Capture capture(stream);
    hold_for_graph(mirror, held_by, capture);
    let_go().clear();
    return capture;
  }
  void after_launch(cudaStream_t stream, const Capture& capture) {
    if (!check_every_launch() || capture.active) return;
    C10_CUDA_CHECK(cudaStreamSynchronize(stream));
    poll();
  }
};
using KVCachePtr = std::shared_ptr<KVCache>;

Tensor rows16(const Tensor& t) { return aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Copies that a call has made of arguments live as long as the call: the allocator orders their next use behind it on this stream.
const int32_t* int_row(const OptTensor& o, int64_t B, const Tensor& like, const char* name, Tensor& hold) {
  if (!o.has_value()) return nullptr;
  KD_VALUE(o->dim() == 1 && o->size(0) == B && o->scalar_type() == at::kInt, name, " must be an int32 tensor of shape (batch,) = (", B, ",)");
  KD_VALUE(o->device() == like.device(), name, " must live on ", like.device());
  hold = o->contiguous();
  return hold.data_ptr<int32_t>();
}

const int32_t* table_rows(const Tensor& table, int64_t B, const Tensor& like, const char* name, Tensor& hold, int64_t* stride) {
  KD_VALUE(table.dim() == 2 && table.size(0) == B && table.scalar_type() == at::kInt, name, " must be an int32 tensor of shape (batch, blocks)");
  KD_VALUE(table.device() == like.device(), name, " must live on ", like.device());
  KD_VALUE(table.size(1) <= (1 << 24), name, " has more than 2^24 blocks");
  hold = table.size(1) <= 1 || table.stride(1) == 1 ? table : table.contiguous();
  *stride = hold.stride(0);
  return hold.data_ptr<int32_t>();
}

struct Sequences {
  Tensor table, lens;
  kd_cache_seqs abi{};
  Sequences(const KVCache& c, int64_t B, const Tensor& table_, const Tensor& lens_) {
    KD_VALUE(B <= INT32_MAX, "too many sequences");
    abi.table = table_rows(table_, B, c.k, "page_table", table, &abi.table_stride);
    abi.lens = int_row(lens_, B, c.k, "lens", lens);
    abi.B = static_cast<int32_t>(B);
    abi.blocks = static_cast<int32_t>(table.size(1));
  }
};

void refuse_gradients(const char* name, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && t->requires_grad()), name, " has no backward: the cache holds no history. Call it under torch.no_grad()");
    refuse_forward_ad(name, *t);
  }
  refuse_tracing(name);
}

void check_heads(const KVCache& c, const Tensor& t, const char* name, int64_t heads) {
  KD_VALUE(t.dim() == 4, name, " must be (batch, heads, time, head_dim)");
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor; there is no CPU path");
  KD_VALUE(t.device() == c.k.device(), name, " must live on ", c.k.device());
  KD_VALUE(t.size(3) == c.k.size(3), name, " has head_dim ", t.size(3), ", the cache ", c.k.size(3));
  KD_VALUE(heads == 0 || t.size(1) == heads, name, " has ", t.size(1), " heads, the cache ", heads);
  KD_VALUE(t.size(2) <= (1 << 30), name, " has too many tokens");
}

void cache_append(KVCache& c, const Tensor& k_, const Tensor& v_, const Tensor& table, const Tensor& lens, const OptTensor& n_new, const OptTensor& in_span,
                  const OptTensor& span_id, const OptTensor& is_prefix) {
  check_heads(c, k_, "k", c.abi.H);
  check_heads(c, v_, "v", c.abi.H);
  KD_VALUE(v_.sizes() == k_.sizes(), "k and v must have the same shape, got ", k_.sizes(), ", ", v_.sizes());
  const auto type = k_.scalar_type();
  KD_VALUE((type == at::kHalf || type == at::kBFloat16 || type == at::kFloat) && v_.scalar_type() == type, "k and v must share dtype float16, bfloat16 or float32");
  refuse_gradients("cache_append", {&k_, &v_});
  KD_VALUE(c.desc.has_value() || !(in_span.has_value() || span_id.has_value() || is_prefix.has_value()), "this cache holds no metadata (desc)");
  const int64_t B = k_.size(0), T = k_.size(2);
  const Sequences s(c, B, table, lens);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor k = rows16(k_), v = rows16(v_);
  kd_cache_tokens t{};
  Tensor held[4];
  t.k = desc(k);
  t.v = desc(v);
  t.T = static_cast<int32_t>(T);
  t.dtype = dtype_code(type);
  t.n_new = int_row(n_new, B, c.k, "new_lens", held[3]);
  auto per_token = [&](const OptTensor& o, at::ScalarType want, const char* name, Tensor& hold, int64_t* stride) -> const void* {
    if (!o.has_value()) return nullptr;
    KD_VALUE(o->dim() == 2 && o->size(0) == B && o->size(1) == T, name, " must have shape (batch, time) = (", B, ", ", T, "), got ", o->sizes());
    KD_VALUE(o->device() == c.k.device(), name, " must live on ", c.k.device());
    if (want == at::kBool) KD_VALUE(o->scalar_type() == at::kBool, name, " must be a torch.bool tensor (the rule negates it logically)");
    hold = o->to(want);
    if (T > 1 && hold.stride(1) != 1) hold = hold.contiguous();
    *stride = hold.stride(0);
    return hold.data_ptr();
  };
  t.in_span = static_cast<const uint8_t*>(per_token(in_span, at::kBool, "in_span", held[0], &t.in_span_stride_b));
  t.span_id = static_cast<const int64_t*>(per_token(span_id, at::kLong, "span_id", held[1], &t.span_id_stride_b));
  t.is_prefix = static_cast<const uint8_t*>(per_token(is_prefix, at::kBool, "is_prefix", held[2], &t.is_prefix_stride_b));
  c.poll();
  c10::cuda::CUDAGuard guard(c.k.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const Capture capture = c.before_launch(stream);
  check(lib.cache_append(&c.abi, &s.abi, &t, stream));
  c.after_launch(stream, capture);
}

std::tuple<Tensor, Tensor> cache_attention(KVCache& c, const Tensor& q_, const Tensor& table, const Tensor& lens, const OptTensor& q_lens,
                                           std::optional<double> sm_scale, bool causal, bool return_lse, const OptTensor& weights, bool like_input) {
  check_heads(c, q_, "q", 0);
  const auto type = q_.scalar_type();
  KD_VALUE(type == at::kHalf || type == at::kBFloat16, "q must be float16 or bfloat16");
  const int64_t B = q_.size(0), H = q_.size(1), T = q_.size(2);
  KD_VALUE(H >= 1 && H % c.abi.H == 0, "q has ", H, " heads, which is no multiple of the cache's ", c.abi.H);
  refuse_gradients("cache_attention", {&q_});
  const double scale = sm_scale.has_value() ? *sm_scale : 1.0 / std::sqrt(static_cast<double>(q_.size(3)));
  KD_VALUE(scale > 0.0 && std::isfinite(scale), "sm_scale must be positive and finite");
  const Sequences s(c, B, table, lens);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor q = rows16(q_);
  Tensor held, workspace, o = empty_out(q_, like_input), lse;
  const Tensor out = aligned(o) ? o : empty_on(q.sizes(), type, q.device());
  kd_cache_queries p{};
  p.q = desc(q);
  p.o = desc(out);
  p.H = static_cast<int32_t>(H);
  p.T = static_cast<int32_t>(T);
  p.dtype = dtype_code(type);
  p.causal = causal;
  p.sm_scale = static_cast<float>(scale);
  p.q_lens = int_row(q_lens, B, c.k, "q_lens", held);
  if (weights.has_value()) {
    const Tensor& w = *weights;
    KD_VALUE(w.dim() == 3 && w.size(0) == B && w.size(1) == c.abi.H && w.scalar_type() == at::kFloat && (w.size(2) <= 1 || w.stride(2) == 1),
             "weights must be float32 (batch, cache heads, tokens) with unit stride along tokens");
    KD_VALUE(w.device() == c.k.device(), "weights must live on ", c.k.device());
    KD_VALUE(w.size(2) <= INT32_MAX, "weights has too many tokens");
    // each head's tokens behind those of the one before, in either order of the two outer dimensions
    const bool batch_first = B <= 1 || (c.abi.H > 1 && w.stride(0) >= w.stride(1));
    const int64_t inner = batch_first ? c.abi.H : B, inner_stride = w.stride(batch_first ? 1 : 0), outer = batch_first ? B : c.abi.H, outer_stride = w.stride(batch_first ? 0 : 1);
    KD_VALUE(w.numel() == 0 || ((inner <= 1 || inner_stride >= w.size(2)) && (outer <= 1 || outer_stride >= (inner <= 1 ? 0 : (inner - 1) * inner_stride) + w.size(2))),
             "weights must have memory of its own for every head");
    TORCH_CHECK(!w.requires_grad() || !at::GradMode::is_enabled(), "weights is written in place and holds no history");
    p.weights = w.data_ptr<float>();
    p.w_stride_b = w.stride(0);
    p.w_stride_h = w.stride(1);
    p.w_len = static_cast<int32_t>(w.size(2));
  }
  if (return_lse) {
    lse = empty_on({B, H, T}, at::kFloat, q.device());
    p.lse = lse.data_ptr<float>();
  }
  c10::cuda::CUDAGuard guard(c.k.device());
  size_t bytes = 0;
  check(lib.cache_attention_workspace(&c.abi, &s.abi, &p, &bytes));
  if (bytes > 0) {
    workspace = empty_on({static_cast<int64_t>(bytes)}, at::kByte, q.device());
    p.workspace = workspace.data_ptr();
  }
  c.poll();
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const Capture capture = c.before_launch(stream);
  check(lib.cache_attention(&c.abi, &s.abi, &p, stream));
  if (!out.is_same(o)) o.copy_(out);
  c.after_launch(stream, capture);
  return {o, return_lse ? lse : Tensor()};
}

std::tuple<Tensor, Tensor, Tensor> cache_evict(KVCache& c, const Tensor& table, const Tensor& lens, const Tensor& weights, const Tensor& out_table, int64_t keep,
                                               int64_t recent, int64_t first) {
  KD_VALUE(weights.dim() == 3 && weights.size(1) == c.abi.H && weights.scalar_type() == at::kFloat, "weights must be float32 (batch, cache heads, tokens)");
  KD_VALUE(weights.device() == c.k.device(), "weights must live on ", c.k.device());
  KD_VALUE(weights.size(2) <= INT32_MAX, "weights has too many tokens");
  KD_VALUE(keep >= 1 && keep <= (1 << 30), "keep must be from 1 to 2^30, got ", keep);
  KD_VALUE(recent >= 0 && first >= 0 && recent <= keep && first <= keep - recent, "recent and first must not be negative, nor more than keep together, got ", recent,
           " and ", first, " of ", keep);
  refuse_gradients("cache_evict", {&weights});
  const int64_t B = weights.size(0), H = c.abi.H;
  const Sequences s(c, B, table, lens);
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor w = weights.size(2) <= 1 || weights.stride(2) == 1 ? weights : weights.contiguous();
  kd_cache_eviction e{};
  Tensor held, index = empty_on({B, H, keep}, at::kInt, w.device()), out_w = empty_on({B, H, keep}, at::kFloat, w.device()), out_lens = empty_on({B}, at::kInt, w.device());
  e.weights = w.data_ptr<float>();
  e.w_stride_b = w.stride(0);
  e.w_stride_h = w.stride(1);
  e.w_len = static_cast<int32_t>(w.size(2));
  e.keep = static_cast<int32_t>(keep);
  e.recent = static_cast<int32_t>(recent);
  e.first = static_cast<int32_t>(first);
  e.out_table = table_rows(out_table, B, c.k, "out_table", held, &e.out_table_stride);
  KD_VALUE(held.size(1) * KD_CACHE_PAGE >= keep, "out_table must name ", (keep + KD_CACHE_PAGE - 1) / KD_CACHE_PAGE, " pages for each sequence, got ", held.size(1));
  e.index = index.data_ptr<int32_t>();
  e.out_weights = out_w.data_ptr<float>();
  e.out_lens = out_lens.data_ptr<int32_t>();
  c.poll();
  c10::cuda::CUDAGuard guard(c.k.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const Capture capture = c.before_launch(stream);
  check(lib.cache_evict(&c.abi, &s.abi, &e, stream));
  c.after_launch(stream, capture);
  return {index, out_lens, out_w};
}

std::tuple<Tensor, Tensor> cache_read(KVCache& c, const Tensor& table, const Tensor& lens, int64_t count, const OptTensor& start, at::ScalarType type) {
  KD_VALUE(type == at::kHalf || type == at::kBFloat16 || type == at::kFloat, "dtype must be float16, bfloat16 or float32");
  KD_VALUE(count >= 0 && count <= (1 << 30), "count must be from 0 to 2^30, got ", count);
  KD_VALUE(lens.dim() == 1, "lens must be an int32 tensor of shape (batch,)");
  refuse_tracing("cache_read");
  const int64_t B = lens.size(0);
  const Sequences s(c, B, table, lens);
  Tensor held;
  const int32_t* from = int_row(start, B, c.k, "start", held);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor k = empty_on({B, c.abi.H, count, c.abi.D}, type, c.k.device()), v = empty_on({B, c.abi.H, count, c.abi.D}, type, c.k.device());
  const kd_tensor kt = desc(k), vt = desc(v);
  c.poll();
  c10::cuda::CUDAGuard guard(c.k.device());
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const Capture capture = c.before_launch(stream);
  check(lib.cache_read(&c.abi, &s.abi, from, static_cast<int32_t>(count), dtype_code(type), &kt, &vt, stream));
  c.after_launch(stream, capture);
  return {k, v};
}
