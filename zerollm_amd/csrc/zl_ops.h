// Operators of long contexts (zl_kv4.hip, zl_rope.hip, zl_logprob.hip): argument structures and launchers. The entry points
// (zl_ops.cpp) check the arguments; the launchers assume them checked.
#pragma once
#include "zl_kernels.h"

namespace zl {

// ---- values of the callers' types
template <int TYPE> struct ValueOf;
template <> struct ValueOf<T_F32> { typedef float t; };
template <> struct ValueOf<T_F16> { typedef uint16_t t; };
template <> struct ValueOf<T_BF16> { typedef uint16_t t; };
template <int TYPE>
__device__ __forceinline__ float load_value(typename ValueOf<TYPE>::t v) {
  if constexpr (TYPE == T_F32) return v;
  else if constexpr (TYPE == T_F16) return h2f(v);
  else return __uint_as_float((uint32_t)v << 16);
}
// (rounded to nearest, ties to even: half a step of the output's own type, once per output)
template <int TYPE>
__device__ __forceinline__ typename ValueOf<TYPE>::t store_value(float f) {
  if constexpr (TYPE == T_F32) return f;
  else if constexpr (TYPE == T_F16) return f2h(f);
  else {
    const uint32_t u = __float_as_uint(f);
    if (f != f) return (uint16_t)((u >> 16) | 0x40);
    return (uint16_t)((u + 0x7fff + ((u >> 16) & 1)) >> 16);
  }
}
inline int value_bytes(int type) { return type == T_F32 ? 4 : type == T_F16 || type == T_BF16 ? 2 : 0; }

// ---- 4-bit KV cache. Per (slot, KV head) a run of records of 32 positions, each 36 HD bytes: [keys 16 HD][values 16 HD]
// [key scales 2 HD][value scales 2 HD], so that one record is one contiguous piece of memory for the wave that reads it.
// Codes lie in the order of the matrix instructions' operands (16 x 16 x 32, f16): for a 16-position tile t and dimension
// block b of 32, lane l holds position 16 t + l % 16, dimensions 32 b + 8 (l / 16) + e, e = 0 .. 7, one nibble each; for 16
// dimensions w, lane l holds dimension 16 w + l % 16 at positions 16 (e / 4) + 4 (l / 16) + e % 4, which is where the score
// product leaves the scores of those positions. A lane's words, in fours, are its 16-byte loads. Nibble e / 2 + 4 (e % 2) of
// a word holds e: shifting the word by 4 r and masking both halves gives the pair (2 r, 2 r + 1). Scales (f16): [position
// / 4 % 4][position / 16][block][position % 4], 16 bytes for each two blocks of four positions.
constexpr int KV4_GROUP = 32;
__host__ __device__ constexpr int kv4_record(int hd) { return 36 * hd; }
__host__ __device__ constexpr int kv4_word(int w, int lane) { return ((w >> 2) * 64 + lane) * 4 + (w & 3); }
__host__ __device__ constexpr int kv4_nibble(int e) { return (e >> 1) + 4 * (e & 1); }
__host__ __device__ constexpr int kv4_scale(int p, int b, int nb) { return ((((p >> 2) & 3) * 2 + ((p >> 4) & 1)) * nb + b) * 4 + (p & 3); }

// Q4_0 of a block of 32 values, eight on each of four neighbouring lanes: the value of largest magnitude (the lowest index among
// equals) gives d = mx / -8, and code = clamp(trunc(x / d + 8.5), 0, 15) with 1/d, the product and the sum each rounded in f64, as
// the library's Q4_0 quantiser. Returns d in f16; NaN for a block with a value that is not finite or beyond f16.
__device__ __forceinline__ uint16_t kv4_quant(const float (&y)[8], int lane, int (&code)[8]) {
  float am = 0.0f;
  uint32_t neg = 0;
  bool bad = false;
  #pragma unroll
  for (int e = 0; e < 8; e++) {
    const float m = fabsf(y[e]);
    bad |= !(m <= 65504.0f);
    if (m > am) { am = m; neg = __float_as_uint(y[e]) >> 31; }
  }
  const float two = fmaxf(am, dpp_move<0xB1>(am)), all = fmaxf(two, dpp_move<0x4E>(two));
  // the first lane that reached it, and its sign, as one number; bad blocks
  uint32_t first = am == all ? 2 * (lane & 3) + neg : 8;
  first = min(first, dpp_move<0xB1>(first));
  first = min(first, dpp_move<0x4E>(first));
  uint32_t nan = bad;
  nan |= dpp_move<0xB1>(nan);
  nan |= dpp_move<0x4E>(nan);
  const float mx = first & 1 ? -all : all;
  const double d = (double)mx / -8.0, inv = d != 0.0 ? 1.0 / d : 0.0;
  #pragma unroll
  for (int e = 0; e < 8; e++) code[e] = nan ? 8 : min(15, max(0, (int)((double)y[e] * inv + 8.5)));
  return nan ? (uint16_t)0x7e00 : f2h((float)d);
}
// A key word: the lane's eight codes.
__device__ __forceinline__ uint32_t kv4_pack(const int (&code)[8]) {
  uint32_t w = 0;
  #pragma unroll
  for (int e = 0; e < 8; e++) w |= (uint32_t)code[e] << (4 * kv4_nibble(e));
  return w;
}

struct Kv4View {
  uint8_t *base;
  int nslot, nkv, hd;
  long cap;        // positions a caller may use
  long ngroup;     // records per (slot, head): whole pairs of them (a span of the attention)
};

inline long kv4_groups(long cap) { return (cap + 63) / 64 * 2; }
inline int64_t kv4_bytes(int nslot, int nkv, int hd, long cap) { return (int64_t)nslot * nkv * kv4_groups(cap) * kv4_record(hd); }

// The batch and its rows (strides in values).
struct OpRows { void *p; long seq, tok, head; };
struct OpBatch {
  int nseq, ntok;
  const int *pos, *count, *slot;
  int tok0 = 0;  // attention: the tokens are tok0 .. tok0 + ntok - 1 of each sequence
};

void launch_kv4_append(const Kv4View &c, const OpBatch &b, int type, const OpRows &k, const OpRows &v, hipStream_t st);
void launch_kv4_read(const Kv4View &c, const OpBatch &b, int type, const OpRows &k, const OpRows &v, hipStream_t st);

struct Kv4Attn {
  Kv4View c;
  OpBatch b;
  OpRows q, out;
  int nhead;
  float scale;
  void *work;
  // set by the launcher: records per row in work, spans of a sequence up to which they are spans', whether the queries are whole
  // 16-byte pieces; b is a slab of the call
  int nrec, spanmax;
  bool qvec, direct;  // direct: no records, a row's only ones are its output
};
long kv4_attention_work(const Kv4View &c, int nseq, int ntok, int nhead);
void launch_kv4_attention(const Kv4Attn &a, int type, hipStream_t st);
// f32 queries of one sequence, outputs to a model's rows (a.out is not used).
void launch_kv4_attention_model(const Kv4Attn &a, const HeadOut &out, hipStream_t st);
// A layer's attention of a model whose cache is in 4 bits (zl_attn.hip).
void launch_attention_q4(const AttnArgs &a, const Kv4View &c, void *work, int B, hipStream_t st);

// ---- rotary positions
struct RopeArgs {
  const double *turns;  // device: turns per position of each pair (angle / 2 pi)
  float gain;           // factor of cos and sin
  int half, neox, hd;
  OpBatch b;
  int nq, nk;           // heads (nk 0: none)
  OpRows q, qo, k, ko;
};
void launch_rope(const RopeArgs &a, int type, hipStream_t st);

// ---- log probabilities
struct LogprobArgs {
  const void *x;
  long ld;
  int rows, vocab, ntop;
  const int *tokens;
  float *lp, *ent;
  int *ids;
  float *toplp;
  void *work;
};
constexpr int LOGPROB_MAX_TOP = 64;
long logprobs_work(int rows, int vocab, int ntop);
void launch_logprobs(const LogprobArgs &a, int type, hipStream_t st);

}  // namespace zl
