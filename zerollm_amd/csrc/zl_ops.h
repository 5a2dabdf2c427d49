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
struct OpBatch { int nseq, ntok; const int *pos, *count, *slot; };

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
  // 16-byte pieces
  int nrec, spanmax;
  bool qvec;
};
void kv4_prepare(int hd);  // once before launches of this head size
long kv4_attention_work(const Kv4View &c, int nseq, int ntok, int nhead);
void launch_kv4_attention(const Kv4Attn &a, int type, hipStream_t st);

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
