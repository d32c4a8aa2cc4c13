// q8_model.h -- a model in 8 bits: the launch sequence of its rows on the
// operators of q8.h, its weights, workspace and caches. Included by
// defer_gpu.hip behind the batched path, whose rows, logits and sampling it
// shares.
//
// Every row's arithmetic depends on the row alone (the products' sums are
// exact, every other sum's order goes by the row's own position), so a prompt
// fed at once, token by token or beside other sessions gives the same bits, as
// the f32 model's does.
#pragma once

struct Q8Matrix {
  int8_t* w = nullptr;  // [m][k]
  float* s = nullptr;   // [m]
  uint32_t m = 0, k = 0;
};

struct Q8Model {
  std::vector<Q8Matrix> qkv, o, gu, down;
  Q8Matrix lm;
  char* buf = nullptr;  // all of the above
  // workspace, grown with the batched path's
  uint32_t rows = 0, lm_rows = 0;
  int8_t* codes = nullptr;   // [rows][max(h, q, ff)]
  float* scale = nullptr;    // [rows]
  float *att = nullptr, *delta = nullptr;  // [rows][max(q, h)], [rows][h]
  float* logits = nullptr;   // [lm_rows][V]
  char* work = nullptr;      // the attention's
  size_t work_cap = 0;
  // positions hidden from the next single row (a masked forward), or null
  const uint8_t* hidden = nullptr;
  uint32_t hidden_len = 0;
};

static void q8_ws_free(Q8Model* q) {
  void* ps[] = {q->codes, q->scale, q->att, q->delta, q->logits, q->work};
  for (void* p : ps) (void)hipFree(p);
  q->codes = nullptr;
  q->scale = q->att = q->delta = q->logits = nullptr;
  q->work = nullptr;
  q->rows = q->lm_rows = 0;
  q->work_cap = 0;
}
static void q8_free(Q8Model* q) {
  if (!q) return;
  q8_ws_free(q);
  (void)hipFree(q->buf);
  delete q;
}

static int q8_ensure_ws(defer_gpu_model* m, uint32_t rows, uint32_t lm) {
  Q8Model& q = *m->q8;
  if (rows <= q.rows && lm <= q.lm_rows) return DEFER_GPU_OK;
  const Dims& d = m->d;
  const uint32_t R = std::max(rows, q.rows), L = std::max({lm, q.lm_rows, 1u});
  q8_ws_free(&q);
  // the logits' rows go through the codes, too
  const size_t rc = std::max(R, L);
  HIP_TRY(counted_malloc(&q.codes, rc * std::max({d.h, d.q, d.ff})));
  HIP_TRY(counted_malloc(&q.scale, rc * sizeof(float)));
  HIP_TRY(counted_malloc(&q.att, rc * std::max(d.q, d.h) * sizeof(float)));
  HIP_TRY(counted_malloc(&q.delta, rc * d.h * sizeof(float)));
  HIP_TRY(counted_malloc(&q.logits, (size_t)L * d.V * sizeof(float)));
  q.rows = R;
  q.lm_rows = L;
  return DEFER_GPU_OK;
}

// ------------------------------------------------------------------ weights

// A layer's matrices in the order of their launches, then the head's.
static Q8Matrix* q8_matrix(Q8Model* q, uint32_t l, uint32_t which) {
  Q8Matrix* const of[] = {&q->qkv[l], &q->o[l], &q->gu[l], &q->down[l], &q->lm};
  return of[which];
}

// Rows of a host matrix into 8 bits at row `at` of `to`, a stretch of rows at a
// time through `stage` (device, `cap` floats), on the null stream like the
// rest of a model's upload.
static hipError_t q8_upload(const Q8Matrix& to, size_t at, const float* src, size_t rows, float* stage, size_t cap) {
  const size_t most = std::max<size_t>(1, cap / to.k);
  for (size_t r = 0; r < rows; r += most) {
    const size_t n = std::min(most, rows - r);
    hipError_t e = hipMemcpy(stage, src + r * to.k, n * to.k * sizeof(float), hipMemcpyHostToDevice);
    if (e != hipSuccess) return e;
    if (q8::quantize(DEFER_GPU_F32, stage, to.k, (uint32_t)n, to.k, to.w + (at + r) * to.k, to.s + at + r, nullptr))
      return hipErrorLaunchFailure;
  }
  return hipSuccess;
}

// Room for every matrix, in one allocation.
static hipError_t q8_alloc(defer_gpu_model* m) {
  const Dims& d = m->d;
  Q8Model* q = m->q8 = new Q8Model();
  q->qkv.resize(d.L);
  q->o.resize(d.L);
  q->gu.resize(d.L);
  q->down.resize(d.L);
  size_t off = 0;
  std::vector<std::pair<Q8Matrix*, size_t>> at;
  auto take = [&](Q8Matrix& x, uint32_t rows, uint32_t k) {
    x.m = rows;
    x.k = k;
    at.push_back({&x, off});
    off += align256((size_t)rows * k) + align256((size_t)rows * sizeof(float));
  };
  for (uint32_t l = 0; l < d.L; ++l) {
    take(q->qkv[l], d.qkv_rows, d.h);
    take(q->o[l], d.h, d.q);
    take(q->gu[l], 2 * d.ff, d.h);
    take(q->down[l], d.h, d.ff);
  }
  take(q->lm, d.V, d.h);
  const hipError_t e = counted_malloc(&q->buf, off);
  if (e != hipSuccess) return e;
  for (auto& x : at) {
    x.first->w = reinterpret_cast<int8_t*>(q->buf + x.second);
    x.first->s = reinterpret_cast<float*>(q->buf + x.second + align256((size_t)x.first->m * x.first->k));
  }
  return hipSuccess;
}

// ------------------------------------------------------------------ caches

// One allocation: keys, values, key scales, value scales, each [L][pages][...].
static uint32_t q8_cache_pages(const defer_gpu_cache* c) { return (c->cap + q8::PAGE - 1) / q8::PAGE; }
static size_t q8_cache_bytes(const defer_gpu_cache* c) {
  const Dims& d = c->m->d;
  const size_t pos = (size_t)d.L * q8_cache_pages(c) * d.nkv * q8::PAGE;
  return 2 * pos * (q8::padded(d.hd) + sizeof(float));
}
static q8::SeqPages q8_cache_view(const defer_gpu_cache* c) {
  const Dims& d = c->m->d;
  const size_t pos = (size_t)d.L * q8_cache_pages(c) * d.nkv * q8::PAGE, dp = q8::padded(d.hd);
  q8::SeqPages s;
  s.keys = c->q8buf;
  s.values = c->q8buf + pos * dp;
  s.key_scale = reinterpret_cast<float*>(c->q8buf + 2 * pos * dp);
  s.value_scale = s.key_scale + pos;
  s.pages = q8_cache_pages(c);
  return s;
}

// defer_gpu_cache_read of a cache in 8 bits: the values its codes stand for.
static int q8_cache_read(defer_gpu_cache* c, uint32_t layer, float* keys, float* values) {
  const Dims& d = c->m->d;
  const hipStream_t s = c->m->stream;
  const size_t n = (size_t)c->pos * d.kv;
  if (!c->d_tmp) HIP_TRY(counted_malloc(&c->d_tmp, 2 * (size_t)c->cap * d.kv * sizeof(float)));
  if (!c->d_q8args) HIP_TRY(counted_malloc(&c->d_q8args, sizeof(Q8CacheArgs)));
  Q8CacheArgs a;
  a.view = q8_cache_view(c);
  a.row_start[0] = 0;
  a.row_start[1] = a.kv_len = (int32_t)c->pos;
  auto queue = [&]() -> int {
    HIP_TRY(hipMemcpyAsync(c->d_q8args, &a, sizeof(a), hipMemcpyHostToDevice, s));
    q8::Pages p{};
    p.heads = d.nkv;
    p.dp = q8::padded(d.hd);
    p.seqs = &c->d_q8args->view;
    p.seq_layer = layer;
    const q8::Rows r{c->d_q8args->row_start, &c->d_q8args->kv_len, 1, c->pos, c->pos};
    float* v = c->d_tmp + (size_t)c->cap * d.kv;
    const int rc = q8::kv_read(p, r, DEFER_GPU_F32, c->d_tmp, v, d.hd, s);
    if (rc) return rc;
    if (keys) HIP_TRY(hipMemcpyAsync(keys, c->d_tmp, n * sizeof(float), hipMemcpyDeviceToHost, s));
    if (values) HIP_TRY(hipMemcpyAsync(values, v, n * sizeof(float), hipMemcpyDeviceToHost, s));
    return DEFER_GPU_OK;
  };
  const int rc = queue();
  HIP_TRY(hipStreamSynchronize(s));  // nothing writes the caller's arrays after the call
  return rc;
}

// ------------------------------------------------------------------ kernels

__global__ void k_q8_embed(const BRow* __restrict__ rows, const uint32_t* __restrict__ dtok,
                           const float* __restrict__ embed, uint32_t h, float* __restrict__ X) {
  const uint32_t b = blockIdx.x;
  const float* e = embed + (size_t)(dtok ? dtok[b] : rows[b].token) * h;
  for (uint32_t i = threadIdx.x; i < h; i += blockDim.x) X[(size_t)b * h + i] = e[i];
}

// The projections' rows: biases added, queries and keys rotated by halves
// (model.rs:438-465), in place. A thread takes a pair.
__global__ void k_q8_rope(const BRow* __restrict__ rows, const float2* __restrict__ rope,
                          const float* __restrict__ bias, Dims d, float* __restrict__ Y) {
  const uint32_t b = blockIdx.y, i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= d.qkv_rows / 2) return;
  const uint32_t hb = i / d.half, e = i % d.half, r0 = hb * d.hd + e, r1 = r0 + d.half;
  float* y = Y + (size_t)b * d.qkv_rows;
  float x0 = y[r0], x1 = y[r1];
  if (bias) {
    x0 = x0 + bias[r0];
    x1 = x1 + bias[r1];
  }
  if (hb < d.nh + d.nkv) {
    const float2 cs = rope[(size_t)rows[b].pos * d.half + e];
    y[r0] = x0 * cs.x - x1 * cs.y;
    y[r1] = x1 * cs.x + x0 * cs.y;
  } else if (bias) {
    y[r0] = x0;
    y[r1] = x1;
  }
}

// act(gate) * up, over the gate's place.
__global__ void k_q8_act(float* __restrict__ Y, uint32_t ff, uint32_t act) {
  const uint32_t b = blockIdx.y, i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= ff) return;
  float* y = Y + (size_t)b * 2 * ff;
  y[i] = act_fn(y[i], act) * y[ff + i];
}

// The rows whose logits are wanted: residual and last product, side by side.
__global__ void k_q8_select(const uint32_t* __restrict__ sel, const float* __restrict__ X,
                            const float* __restrict__ D, uint32_t h, float* __restrict__ x, float* __restrict__ dl) {
  const size_t from = (size_t)sel[blockIdx.x] * h, to = (size_t)blockIdx.x * h;
  for (uint32_t i = threadIdx.x; i < h; i += blockDim.x) {
    x[to + i] = X[from + i];
    dl[to + i] = D[from + i];
  }
}

// Logits as the sampler reads them: words tagged with their row's generation.
__global__ void k_q8_tag(const float* __restrict__ logits, const uint32_t* __restrict__ gen, uint32_t V,
                         u64* __restrict__ out) {
  const uint32_t i = blockIdx.y;
  const u64 g = (u64)gen[i] << 32;
  for (uint32_t v = blockIdx.x * blockDim.x + threadIdx.x; v < V; v += gridDim.x * blockDim.x)
    out[(size_t)i * V + v] = g | __float_as_uint(logits[(size_t)i * V + v]);
}

// ------------------------------------------------------------------ rows

// batch_run for a model in 8 bits: the same arguments and results.
static int q8_run(defer_gpu_model* m, const BRow* rows, defer_gpu_cache* const* rcache, uint32_t n,
                  const uint32_t* sel, uint32_t nl, const uint32_t* dtok, bool deferred) {
  const Dims& d = m->d;
  const hipStream_t s = m->stream;
  int rc = ensure_ws(m, n, nl);
  if (rc == DEFER_GPU_OK) rc = q8_ensure_ws(m, n, nl);
  if (rc) return rc;
  BatchWs& w = *m->bw;
  Q8Model& q = *m->q8;
  // Neighbouring rows of one cache at consecutive positions are a sequence.
  std::vector<q8::SeqPages> seqs;
  std::vector<int32_t> start, len;
  uint32_t most_rows = 0, most_len = 0;
  for (uint32_t b = 0; b < n; ++b) {
    if (b == 0 || rcache[b] != rcache[b - 1] || rows[b].pos != rows[b - 1].pos + 1) {
      start.push_back((int32_t)b);
      len.push_back(0);
      seqs.push_back(q8_cache_view(rcache[b]));
    }
    len.back() = (int32_t)rows[b].pos + 1;
    most_rows = std::max(most_rows, b + 1 - (uint32_t)start.back());
    most_len = std::max(most_len, rows[b].pos + 1);
  }
  start.push_back((int32_t)n);
  std::vector<uint32_t> lgen(nl);
  for (uint32_t i = 0; i < nl; ++i) lgen[i] = gen_lm(d, rows[sel[i]].tick);
  const BRow* drows = up_put(w, rows, n);
  const q8::SeqPages* d_seqs = up_put(w, seqs.data(), seqs.size());
  const int32_t* d_start = up_put(w, start.data(), start.size());
  const int32_t* d_len = up_put(w, len.data(), len.size());
  const uint32_t* d_sel = up_put(w, sel, nl);
  const uint32_t* d_lgen = up_put(w, lgen.data(), nl);
  if (!drows || !d_seqs || !d_start || !d_len || !d_sel || !d_lgen)
    return fail(DEFER_GPU_E_HIP, "batch staging of %zu bytes exceeded", w.up_cap);
  rc = up_send(w, s);
  if (rc) return rc;
  const q8::Rows r{d_start, d_len, (uint32_t)seqs.size(), n, most_rows};
  const size_t need = q8::attention_workspace(r, d.nh, d.nkv, d.hd, most_len);
  if (need > q.work_cap) {
    (void)hipFree(q.work);
    q.work = nullptr;
    q.work_cap = 0;
    HIP_TRY(counted_malloc(&q.work, need));
    q.work_cap = need;
  }
  if (!deferred) k_begin<<<1, 1, 0, s>>>(w.st);
  double attn_flop = 0.0;
  for (uint32_t b = 0; b < n; ++b) attn_flop += 4.0 * d.nh * d.hd * (rows[b].pos + 1.0);
  auto product = [&](const Q8Matrix& x, uint32_t nr, float* y) {
    ProfSpan ps(m, 0, 2.0 * x.m * x.k * nr);
    return q8::linear(q.codes, x.k, q.scale, x.w, x.k, x.s, nr, x.m, x.k, DEFER_GPU_F32, y, x.m, s);
  };
  k_q8_embed<<<n, 256, 0, s>>>(drows, dtok, m->embed, d.h, w.X);
  for (uint32_t l = 0; l < d.L && !rc; ++l) {
    // the last layer's product joins the residual as the norm reads it
    rc = q8::rms_norm(DEFER_GPU_F32, w.X, d.h, l ? q.delta : nullptr, d.h, m->layers[l].attn_norm, d.eps, n, d.h,
                      l ? w.X : nullptr, d.h, q.codes, q.scale, s);
    if (!rc) rc = product(q.qkv[l], n, w.Y);
    if (rc) break;
    k_q8_rope<<<dim3((d.qkv_rows / 2 + 255) / 256, n), 256, 0, s>>>(drows, m->rope, m->layers[l].bqkv, d, w.Y);
    q8::Pages p{};
    p.heads = d.nkv;
    p.dp = q8::padded(d.hd);
    p.seqs = d_seqs;
    p.seq_layer = l;
    rc = q8::kv_write(p, r, DEFER_GPU_F32, w.Y + d.q, d.qkv_rows, w.Y + d.q + d.kv, d.qkv_rows, d.hd, s);
    if (rc) break;
    {
      ProfSpan ps(m, 1, attn_flop);
      q8::Attention a{};
      a.type = DEFER_GPU_F32;
      a.q = w.Y;
      a.q_stride = d.qkv_rows;
      a.out = q.att;
      a.out_stride = d.q;
      a.heads = d.nh;
      a.head_dim = d.hd;
      a.scale = d.scale;
      a.most_len = most_len;
      a.hidden = q.hidden;
      a.hidden_len = q.hidden_len;
      rc = q8::attention(p, r, a, q.work, q.work_cap, s);
    }
    if (!rc) rc = q8::quantize(DEFER_GPU_F32, q.att, d.q, n, d.q, q.codes, q.scale, s);
    if (!rc) rc = product(q.o[l], n, q.delta);
    if (!rc)
      rc = q8::rms_norm(DEFER_GPU_F32, w.X, d.h, q.delta, d.h, m->layers[l].ffn_norm, d.eps, n, d.h, w.X, d.h, q.codes,
                        q.scale, s);
    if (!rc) rc = product(q.gu[l], n, w.Y);
    if (rc) break;
    k_q8_act<<<dim3((d.ff + 255) / 256, n), 256, 0, s>>>(w.Y, d.ff, d.act);
    rc = q8::quantize(DEFER_GPU_F32, w.Y, 2 * (int64_t)d.ff, n, d.ff, q.codes, q.scale, s);
    if (!rc) rc = product(q.down[l], n, q.delta);
  }
  if (!rc && nl) {
    k_q8_select<<<nl, 256, 0, s>>>(d_sel, w.X, q.delta, d.h, q.att, w.Y);
    rc = q8::rms_norm(DEFER_GPU_F32, q.att, d.h, w.Y, d.h, m->norm, d.eps, nl, d.h, nullptr, d.h, q.codes, q.scale, s);
    if (!rc) rc = product(q.lm, nl, q.logits);
    if (!rc) {
      k_q8_tag<<<dim3(std::min((d.V + 1023) / 1024, 64u), nl), 256, 0, s>>>(q.logits, d_lgen, d.V, w.LOGT);
      k_b_chunkmax<<<dim3((d.nvc + 4 * CM_CPW - 1) / (4 * CM_CPW), nl), 256, 0, s>>>(d, w.LOGT, d_lgen, w.VMAX, w.VARG,
                                                                                     nl);
    }
  }
  if (rc) {
    (void)hipStreamSynchronize(s);
    return rc;
  }
  HIP_TRY(hipGetLastError());
  HIP_TRY(hipMemcpyAsync(w.h_st, w.st, sizeof(DevState), hipMemcpyDeviceToHost, s));
  if (deferred && !m->prof) return DEFER_GPU_OK;
  HIP_TRY(hipStreamSynchronize(s));
  if (m->prof) prof_collect(m);
  if (w.h_st->abort) return fail(DEFER_GPU_E_TIMEOUT, "a device-side wait exceeded its bound");
  return DEFER_GPU_OK;
}

// ------------------------------------------------------------------ calls

// defer_gpu_forward: one row; masked positions are hidden from its attention.
static int q8_forward(defer_gpu_model* m, defer_gpu_cache* c, uint32_t token, const uint32_t* masked, size_t n_masked,
                      float* logits_out) {
  Q8Model& q = *m->q8;
  const hipStream_t s = m->stream;
  std::vector<uint8_t> hide;
  for (size_t i = 0; i < n_masked; ++i)
    if (masked[i] < c->pos) {
      hide.resize(c->pos, 0);
      hide[masked[i]] = 1;
    }
  int rc = up_reset(m);
  if (rc) return rc;
  if (!hide.empty()) {
    if (!c->d_hidden) HIP_TRY(counted_malloc(&c->d_hidden, c->cap));
    HIP_TRY(hipMemcpyAsync(c->d_hidden, hide.data(), hide.size(), hipMemcpyHostToDevice, s));
    q.hidden = c->d_hidden;
    q.hidden_len = (uint32_t)hide.size();
  }
  rc = forward_batch_impl(m, &c, &token, nullptr, nullptr, 1, logits_out);
  q.hidden = nullptr;
  q.hidden_len = 0;
  return rc;
}

// defer_gpu_generate and _cb: a step at a time (arguments checked by the
// callers). on_token is called as each token's forward is done.
static int q8_generate(defer_gpu_model* m, defer_gpu_cache* c, uint32_t n, uint32_t max_tokens, float T,
                       const uint32_t* words, const uint32_t* stop, size_t n_stop, uint32_t* out, uint32_t* n_out,
                       defer_gpu_token_fn on_token, void* user) {
  double ms = 0.0;
  bool halt = false;
  uint32_t i = 0;
  while (i < n && !halt) {
    const int rc = defer_gpu_step_batch(m, &c, 1, T, T != 0.0f ? words + i : nullptr, out + i);
    if (rc) return rc;
    ms += m->last_ms;
    m->last_ms = ms;
    const uint32_t tok = out[i++];
    if (n_out) *n_out = i;
    if (on_token) {
      const int e = on_token(user, i - 1, tok);
      if (e) return fail(DEFER_GPU_E_CALLBACK, "on_token returned %d at token %u", e, i - 1);
    }
    for (size_t k = 0; k < n_stop && !halt; ++k) halt = stop[k] == tok;
  }
  if (n < max_tokens && !halt) return fail(DEFER_GPU_E_CONTEXT, "context length %u exceeded", m->cfg.max_seq_len);
  return DEFER_GPU_OK;
}
