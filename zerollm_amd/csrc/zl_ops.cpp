// C entry points of the long-context operators: argument checks, handles, launches.
#include <math.h>

#include <algorithm>
#include <memory>
#include <vector>

#include "zl_api.h"
#include "zl_ops.h"
#include "zl_rope_freq.h"

using namespace zl;

struct zl_kv4 {
  Kv4View v{};
  int dev = 0;
  int64_t bytes = 0;
  ~zl_kv4() {
    if (v.base) {
      hipDeviceSynchronize();
      hipFree(v.base);
    }
  }
};

struct zl_rope {
  double *turns = nullptr;
  double gain = 1.0;
  int n_rot = 0, neox = 0, dev = 0;
  ~zl_rope() {
    if (turns) {
      hipDeviceSynchronize();
      hipFree(turns);
    }
  }
};

namespace zl {

static void need_type(const char *f, int type) {
  ZL_REQUIRE(value_bytes(type) > 0, ZL_ERR_UNSUPPORTED, std::string(f) + ": values must be F32, F16 or BF16 (got type " + std::to_string(type) + ")");
}

constexpr int64_t MOST_ROWS = 1 << 26;  // tokens or query rows of a call: the launchers keep their grids within 2^32 threads up to here

// The batch; heads and sequences are grid dimensions of at most 65535. Returns whether there is anything to do.
static bool take_batch(const char *f, const zl_batch *b, OpBatch *o) {
  ZL_REQUIRE(b, ZL_ERR_ARG, std::string(f) + ": null argument");
  ZL_REQUIRE(b->n_seq >= 0 && b->n_tok >= 0, ZL_ERR_ARG, std::string(f) + ": negative batch size");
  ZL_REQUIRE(b->n_seq <= 65535, ZL_ERR_ARG, std::string(f) + ": at most 65535 sequences (got " + std::to_string(b->n_seq) + ")");
  if (b->n_seq == 0 || b->n_tok == 0) return false;
  ZL_REQUIRE((int64_t)b->n_seq * b->n_tok <= MOST_ROWS, ZL_ERR_ARG, std::string(f) + ": at most " + std::to_string(MOST_ROWS) + " tokens a call");
  ZL_REQUIRE(b->pos, ZL_ERR_ARG, std::string(f) + ": positions missing");
  *o = OpBatch{b->n_seq, b->n_tok, b->pos, b->count, b->slot};
  return true;
}
static OpRows take_rows(const char *f, const zl_rows *r, int type) {
  ZL_REQUIRE(r && r->p, ZL_ERR_ARG, std::string(f) + ": rows missing");
  ZL_REQUIRE((uintptr_t)r->p % value_bytes(type) == 0, ZL_ERR_ARG, std::string(f) + ": rows not aligned to their values");
  return OpRows{r->p, r->seq, r->tok, r->head};
}

static void check_logprobs(int rows, int vocab, int n_top) {
  ZL_REQUIRE(rows >= 0 && rows < (1 << 24) && vocab >= 1 && vocab <= (1 << 30), ZL_ERR_ARG, "logprobs: bad row count or vocabulary");
  ZL_REQUIRE(n_top >= 0 && n_top <= LOGPROB_MAX_TOP && n_top <= vocab, ZL_ERR_ARG,
             "logprobs: n_top must be 0 to " + std::to_string(LOGPROB_MAX_TOP) + " and at most the vocabulary (got " + std::to_string(n_top) + ")");
}

}  // namespace zl

extern "C" {

int zl_kv4_create(int n_slot, int n_head_kv, int head_dim, int64_t capacity, zl_kv4 **out) {
  ZL_API_BEGIN
  ZL_REQUIRE(out, ZL_ERR_ARG, "null argument");
  ZL_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, ZL_ERR_UNSUPPORTED,
             "4-bit cache: head_dim must be 64, 128 or 256 (got " + std::to_string(head_dim) + ")");
  ZL_REQUIRE(n_slot >= 1 && n_slot <= 65535 && n_head_kv >= 1 && n_head_kv <= 65535 && capacity >= 1 && capacity <= INT32_MAX, ZL_ERR_ARG,
             "4-bit cache: bad slot count, head count or capacity");
  ensure_init();
  std::unique_ptr<zl_kv4> c(new zl_kv4());
  c->dev = device();
  OnDevice on(c->dev);
  c->v.nslot = n_slot; c->v.nkv = n_head_kv; c->v.hd = head_dim; c->v.cap = capacity;
  c->v.ngroup = kv4_groups(capacity);
  c->bytes = kv4_bytes(n_slot, n_head_kv, head_dim, capacity);
  ZL_HIP(hipMalloc(&c->v.base, c->bytes));
  zero_now(c->v.base, c->bytes);
  *out = c.release();
  ZL_API_END
}

int zl_kv4_free(zl_kv4 *c) {
  ZL_API_BEGIN
  if (c) {
    OnDevice on(c->dev);
    delete c;
  }
  ZL_API_END
}

int zl_kv4_bytes(const zl_kv4 *c, int64_t *bytes) {
  ZL_API_BEGIN
  ZL_REQUIRE(c && bytes, ZL_ERR_ARG, "null argument");
  *bytes = c->bytes;
  ZL_API_END
}

int zl_kv4_append(zl_kv4 *c, const zl_batch *b, int type, const zl_rows *k, const zl_rows *v, void *stream) {
  ZL_API_BEGIN
  const char *f = "zl_kv4_append";
  ZL_REQUIRE(c, ZL_ERR_ARG, "null argument");
  need_type(f, type);
  OpBatch ob;
  if (take_batch(f, b, &ob)) {
    ZL_REQUIRE(ob.slot || ob.nseq <= c->v.nslot, ZL_ERR_ARG, std::string(f) + ": " + std::to_string(ob.nseq) + " sequences in a cache of " + std::to_string(c->v.nslot) + " slots");
    OnDevice on(c->dev);
    launch_kv4_append(c->v, ob, type, take_rows(f, k, type), take_rows(f, v, type), (hipStream_t)stream);
  }
  ZL_API_END
}

int zl_kv4_read(const zl_kv4 *c, const zl_batch *b, int type, const zl_rows *k, const zl_rows *v, void *stream) {
  ZL_API_BEGIN
  const char *f = "zl_kv4_read";
  ZL_REQUIRE(c, ZL_ERR_ARG, "null argument");
  need_type(f, type);
  OpBatch ob;
  if (take_batch(f, b, &ob)) {
    ZL_REQUIRE(ob.slot || ob.nseq <= c->v.nslot, ZL_ERR_ARG, std::string(f) + ": " + std::to_string(ob.nseq) + " sequences in a cache of " + std::to_string(c->v.nslot) + " slots");
    OnDevice on(c->dev);
    launch_kv4_read(c->v, ob, type, take_rows(f, k, type), take_rows(f, v, type), (hipStream_t)stream);
  }
  ZL_API_END
}

static void check_heads(const char *f, const zl_kv4 *c, int n_seq, int n_tok, int n_head) {
  ZL_REQUIRE(n_head >= 1 && n_head % c->v.nkv == 0 && n_head <= 65535, ZL_ERR_ARG,
             std::string(f) + ": " + std::to_string(n_head) + " query heads over " + std::to_string(c->v.nkv) + " KV heads");
  ZL_REQUIRE((int64_t)n_seq * n_tok <= MOST_ROWS / n_head, ZL_ERR_ARG, std::string(f) + ": at most " + std::to_string(MOST_ROWS) + " query rows a call");
}

int zl_kv4_attention_work(const zl_kv4 *c, int n_seq, int n_tok, int n_head, int64_t *bytes) {
  ZL_API_BEGIN
  ZL_REQUIRE(c && bytes, ZL_ERR_ARG, "null argument");
  ZL_REQUIRE(n_seq >= 0 && n_tok >= 0, ZL_ERR_ARG, "zl_kv4_attention_work: negative batch size");
  check_heads("zl_kv4_attention_work", c, n_seq, n_tok, n_head);
  *bytes = kv4_attention_work(c->v, n_seq, n_tok, n_head);
  ZL_API_END
}

int zl_kv4_attention(const zl_kv4 *c, const zl_batch *b, int type, const zl_rows *q, int n_head, float scale, const zl_rows *out,
                     void *work, int64_t work_bytes, void *stream) {
  ZL_API_BEGIN
  const char *f = "zl_kv4_attention";
  ZL_REQUIRE(c, ZL_ERR_ARG, "null argument");
  need_type(f, type);
  ZL_REQUIRE(b, ZL_ERR_ARG, std::string(f) + ": null argument");
  check_heads(f, c, std::max(b->n_seq, 0), std::max(b->n_tok, 0), n_head);
  ZL_REQUIRE(scale >= 0.0f && scale < INFINITY, ZL_ERR_ARG, std::string(f) + ": the scale must be finite and not negative");
  Kv4Attn a{};
  if (take_batch(f, b, &a.b)) {
    ZL_REQUIRE(a.b.slot || a.b.nseq <= c->v.nslot, ZL_ERR_ARG, std::string(f) + ": " + std::to_string(a.b.nseq) + " sequences in a cache of " + std::to_string(c->v.nslot) + " slots");
    const int64_t need = kv4_attention_work(c->v, a.b.nseq, a.b.ntok, n_head);
    ZL_REQUIRE(work && work_bytes >= need, ZL_ERR_ARG, std::string(f) + ": a work space of " + std::to_string(need) + " bytes is needed (got " + std::to_string(work ? work_bytes : 0) + ")");
    ZL_REQUIRE((uintptr_t)work % 16 == 0, ZL_ERR_ARG, std::string(f) + ": the work space must be aligned to 16 bytes");
    a.c = c->v;
    a.q = take_rows(f, q, type);
    a.out = take_rows(f, out, type);
    a.nhead = n_head;
    a.scale = scale > 0.0f ? scale : (float)(1.0 / sqrt((double)c->v.hd));
    a.work = work;
    OnDevice on(c->dev);
    launch_kv4_attention(a, type, (hipStream_t)stream);
  }
  ZL_API_END
}

int zl_rope_create(const zl_rope_opts *o, zl_rope **out) {
  ZL_API_BEGIN
  ZL_REQUIRE(o && out, ZL_ERR_ARG, "null argument");
  std::vector<double> th;
  double gain = 1.0;
  rope_angles(*o, &th, &gain);
  ensure_init();
  std::unique_ptr<zl_rope> r(new zl_rope());
  r->dev = device();
  r->n_rot = o->n_rot;
  r->neox = o->neox ? 1 : 0;
  r->gain = gain;
  for (double &t : th) t /= 2.0 * M_PI;
  OnDevice on(r->dev);
  ZL_HIP(hipMalloc(&r->turns, th.size() * sizeof(double)));
  ZL_HIP(hipMemcpy(r->turns, th.data(), th.size() * sizeof(double), hipMemcpyHostToDevice));
  *out = r.release();
  ZL_API_END
}

int zl_rope_free(zl_rope *r) {
  ZL_API_BEGIN
  if (r) {
    OnDevice on(r->dev);
    delete r;
  }
  ZL_API_END
}

int zl_rope_apply(const zl_rope *r, const zl_batch *b, int type, int head_dim, const zl_rows *q, const zl_rows *q_out, int n_head,
                  const zl_rows *k, const zl_rows *k_out, int n_head_kv, void *stream) {
  ZL_API_BEGIN
  const char *f = "zl_rope_apply";
  ZL_REQUIRE(r, ZL_ERR_ARG, "null argument");
  need_type(f, type);
  ZL_REQUIRE(head_dim >= r->n_rot && head_dim <= 65536, ZL_ERR_ARG, std::string(f) + ": head_dim " + std::to_string(head_dim) + " below the " + std::to_string(r->n_rot) + " rotated values, or above 65536");
  ZL_REQUIRE(!k == !k_out, ZL_ERR_ARG, std::string(f) + ": k and k_out come together");
  ZL_REQUIRE(n_head >= 1 && n_head <= 65535 && (!k || (n_head_kv >= 1 && n_head_kv <= 65535 - n_head)), ZL_ERR_ARG, std::string(f) + ": bad head count");
  RopeArgs a{};
  if (take_batch(f, b, &a.b)) {
    a.turns = r->turns; a.gain = (float)r->gain; a.half = r->n_rot / 2; a.neox = r->neox; a.hd = head_dim;
    a.nq = n_head; a.nk = k ? n_head_kv : 0;
    a.q = take_rows(f, q, type); a.qo = take_rows(f, q_out, type);
    if (k) { a.k = take_rows(f, k, type); a.ko = take_rows(f, k_out, type); }
    OnDevice on(r->dev);
    launch_rope(a, type, (hipStream_t)stream);
  }
  ZL_API_END
}

int zl_logprobs_work(int rows, int vocab, int n_top, int64_t *bytes) {
  ZL_API_BEGIN
  ZL_REQUIRE(bytes, ZL_ERR_ARG, "null argument");
  check_logprobs(rows, vocab, n_top);
  *bytes = logprobs_work(rows, vocab, n_top);
  ZL_API_END
}

int zl_logprobs(const void *logits, int type, int64_t ld, int rows, int vocab, const int32_t *tokens, int n_top, float *lp,
                float *entropy, int32_t *top_ids, float *top_lp, void *work, int64_t work_bytes, void *stream) {
  ZL_API_BEGIN
  const char *f = "zl_logprobs";
  need_type(f, type);
  check_logprobs(rows, vocab, n_top);
  ZL_REQUIRE(ld >= vocab, ZL_ERR_ARG, std::string(f) + ": row stride below the vocabulary");
  if (rows > 0) {
    ZL_REQUIRE(logits && (uintptr_t)logits % value_bytes(type) == 0, ZL_ERR_ARG, std::string(f) + ": logits missing or not aligned to their values");
    ZL_REQUIRE(!lp || tokens, ZL_ERR_ARG, std::string(f) + ": log probabilities of given tokens need the tokens");
    const int64_t need = logprobs_work(rows, vocab, n_top);
    ZL_REQUIRE(work && work_bytes >= need, ZL_ERR_ARG, std::string(f) + ": a work space of " + std::to_string(need) + " bytes is needed (got " + std::to_string(work ? work_bytes : 0) + ")");
    ZL_REQUIRE((uintptr_t)work % 16 == 0, ZL_ERR_ARG, std::string(f) + ": the work space must be aligned to 16 bytes");
    ensure_init();
    OnDevice on(device());
    launch_logprobs(LogprobArgs{logits, ld, rows, vocab, n_top, tokens, lp, entropy, top_ids, top_lp, work}, type, (hipStream_t)stream);
  }
  ZL_API_END
}

}  // extern "C"
