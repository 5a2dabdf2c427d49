// KV cache in 4 bits: append, read-back and causal attention (layout in zl_ops.h).
#include "zl_ops.h"
#include <algorithm>

namespace zl {

__device__ __forceinline__ uint8_t *record_of(const Kv4View &c, int slot, int head, long group) {
  return c.base + (((long)slot * c.nkv + head) * c.ngroup + group) * kv4_record(c.hd);
}
__device__ __forceinline__ int count_of(const OpBatch &b, int s) { return b.count ? max(0, min(b.count[s], b.ntok)) : b.ntok; }
__device__ __forceinline__ int slot_of(const OpBatch &b, int s) { return b.slot ? b.slot[s] : s; }

// ---------------------------------------------------------------------------------------------- append
// One block per (32-position record that a sequence may touch, KV head, sequence). 32 lanes hold one block of 32 values:
// the value of largest magnitude (the lowest index among equals) gives d = mx / -8, and code = clamp(trunc(x / d + 8.5), 0, 15)
// with 1/d, the product and the sum each rounded in f64, as the library's Q4_0 quantiser. Key words are put together across
// 8 lanes; value words hold 8 positions, so the block gathers its record's codes in LDS and merges them into the words,
// whose other positions it keeps. The block of the first sequence that touches a record of a slot takes all of them, in order.
template <int TYPE>
__global__ __launch_bounds__(256) void k_kv4_append(const Kv4View c, const OpBatch b, const OpRows k, const OpRows v) {
  typedef typename ValueOf<TYPE>::t T;
  extern __shared__ uint8_t vn[];   // [32 positions][hd] value codes
  const int s0 = blockIdx.z, head = blockIdx.y, tid = threadIdx.x, hd = c.hd, nb = hd >> 5;
  const int slot = slot_of(b, s0);
  if (slot < 0 || slot >= c.nslot || count_of(b, s0) == 0) return;
  // (in 64 bits: positions near the ends of int32 must not wrap)
  const long g = ((long)b.pos[s0] >> 5) + blockIdx.x;
  if (g < 0 || g * KV4_GROUP >= c.cap) return;
  auto touches = [&](int s, long *p0, long *p1) {  // positions of sequence s inside the record
    *p0 = max((long)b.pos[s], g * KV4_GROUP);
    *p1 = min(min((long)b.pos[s] + count_of(b, s), (g + 1) * KV4_GROUP), c.cap);
    return *p0 < *p1;
  };
  long p0, p1;
  if (!touches(s0, &p0, &p1)) return;
  if (b.slot)
    for (int s = 0; s < s0; s++) {
      long x, y;
      if (b.slot[s] == slot && touches(s, &x, &y)) return;
    }
  uint8_t *rec = record_of(c, slot, head, g);
  const int grp = tid >> 5, e32 = tid & 31;
  for (int s = s0; s < (b.slot ? b.nseq : s0 + 1); s++) {
    if (s != s0 && (b.slot[s] != slot || !touches(s, &p0, &p1))) continue;
    const int n = (int)(p1 - p0), q0 = (int)(p0 - g * KV4_GROUP);
    const long t0 = p0 - b.pos[s];
    for (int u = grp; u < 2 * n * nb; u += 8) {  // (key | value, position, block)
      const int isv = u >= n * nb, r = isv ? u - n * nb : u, i = r / nb, blk = r - i * nb, p = q0 + i;
      const OpRows &rows = isv ? v : k;
      const float x = load_value<TYPE>(((const T *)rows.p)[s * rows.seq + (t0 + i) * rows.tok + head * rows.head + blk * 32 + e32]);
      const float a = fabsf(x), am = group_fmax(a, 32);
      const int half = tid & 32;
      const uint32_t at = (uint32_t)(__ballot(a == am) >> half);
      const bool bad = (uint32_t)(__ballot(!(a <= 65504.0f)) >> half) != 0;
      const float mx = __shfl(x, at ? __ffs(at) - 1 : 0, 32);
      const double d = (double)mx / -8.0, inv = d != 0.0 ? 1.0 / d : 0.0;
      int code = bad ? 8 : (int)((double)x * inv + 8.5);
      code = min(15, max(0, code));
      const uint16_t dh = bad ? (uint16_t)0x7e00 : f2h((float)d);
      if (e32 == 0) ((uint16_t *)(rec + (isv ? 34 : 32) * hd))[kv4_scale(p, blk, nb)] = dh;
      if (isv) vn[p * hd + blk * 32 + e32] = (uint8_t)code;
      else {
        const int e = e32 & 7;
        uint32_t w = (uint32_t)code << (4 * kv4_nibble(e));
        w |= dpp_move<0xB1>(w); w |= dpp_move<0x4E>(w); w |= dpp_move<0x141>(w);
        if (e == 0) ((uint32_t *)rec)[kv4_word((p >> 4) * nb + blk, (p & 15) + 16 * (e32 >> 3))] = w;
      }
    }
    __syncthreads();
    uint32_t *vw = (uint32_t *)(rec + 16 * hd);
    for (int i = tid; i < 4 * hd; i += 256) {  // words: (dimension, four positions of each tile)
      const int dim = i % hd, gq = i / hd;
      uint32_t w = 0, m = 0;
      #pragma unroll
      for (int e = 0; e < 8; e++) {
        const int p = 16 * (e >> 2) + 4 * gq + (e & 3);
        if (p >= q0 && p < q0 + n) {
          w |= (uint32_t)vn[p * hd + dim] << (4 * kv4_nibble(e));
          m |= 0xfu << (4 * kv4_nibble(e));
        }
      }
      if (!m) continue;
      uint32_t *at = vw + kv4_word(dim >> 4, (dim & 15) + 16 * gq);
      *at = m == 0xffffffffu ? w : (*at & ~m) | w;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------- read-back
__device__ __forceinline__ float kv4_value(const uint8_t *rec, int hd, int isv, int p, int dim) {
  const int nb = hd >> 5;
  const uint32_t *w = (const uint32_t *)(rec + isv * 16 * hd);
  const float d = h2f(((const uint16_t *)(rec + (32 + 2 * isv) * hd))[kv4_scale(p, dim >> 5, nb)]);
  uint32_t x;
  int e;
  if (isv) {
    x = w[kv4_word(dim >> 4, (dim & 15) + 16 * ((p >> 2) & 3))];
    e = 4 * (p >> 4) + (p & 3);
  } else {
    x = w[kv4_word((p >> 4) * nb + (dim >> 5), (p & 15) + 16 * ((dim >> 3) & 3))];
    e = dim & 7;
  }
  return d * (float)((int)((x >> (4 * kv4_nibble(e))) & 15) - 8);
}

// One block per (token, head, sequence), a thread per dimension.
template <int TYPE>
__global__ __launch_bounds__(256) void k_kv4_read(const Kv4View c, const OpBatch b, const OpRows k, const OpRows v) {
  typedef typename ValueOf<TYPE>::t T;
  const int t = blockIdx.x, head = blockIdx.y, s = blockIdx.z, dim = threadIdx.x;
  if (t >= count_of(b, s) || dim >= c.hd) return;
  const int slot = slot_of(b, s);
  const long p = (long)b.pos[s] + t;
  const bool ok = slot >= 0 && slot < c.nslot && p >= 0 && p < c.cap;
  const uint8_t *rec = ok ? record_of(c, slot, head, p >> 5) : nullptr;
  #pragma unroll
  for (int isv = 0; isv < 2; isv++) {
    const OpRows &o = isv ? v : k;
    const float x = ok ? kv4_value(rec, c.hd, isv, (int)(p & 31), dim) : NAN;
    ((T *)o.p)[s * o.seq + t * o.tok + head * o.head + dim] = store_value<TYPE>(x);
  }
}

// ---------------------------------------------------------------------------------------------- attention
// softmax(scale q K) V of a row (a token's query head) over positions 0 .. last, in f32 with the exponentials to base 2. The
// positions are cut, by their index alone, into spans of 64, chunks of 512 (8 spans) and parts of 2048 (4 chunks). A span has
// a softmax of its own: its reference m (the largest score less 3, so that weights reach 8), l = sum of weights and
// o = sum of weights times values. Spans are folded into their chunk in order, chunks into their part, parts into the row:
//   M' = max(M, m), L = L 2^(M - M') + l 2^(m - M'), O = O 2^(M - M') + o 2^(m - M').
// Whichever block or kernel forms a piece, it does these operations, so a row has the same bits in a batch of any size and
// in a cache of any capacity.
//
// Products run on the matrix cores (v_mfma_f32_16x16x32_f16) for 16 rows at a time: keys times queries first, which leaves
// lane l with the scores of row l % 16 at four neighbouring positions, then values (as the left operand) times weights,
// which takes those positions as they lie. Codes less 8 are exact in f16. Queries are scaled per row by a power of two to
// below 2^14 and split into two f16 parts (22 bits, or all the bits of 16-bit queries); a weight times its value's scale
// likewise where the output is f32 or f16 (a single f16 part would add an error as large as the rounding of an f16
// output). Scores are scaled by their key's scale in f32, block by block.
constexpr int SPAN = 64, CHUNK = 512, PART = 2048;
constexpr int SPANS = CHUNK / SPAN, CHUNKS = PART / CHUNK;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The eight codes of a word less 8, as f16: pair r of (word >> 4 r) under the exponent of 1024, less 1032. k: 0x64006400 in a
// vector register, so that and and or are one instruction (which takes a single scalar operand). Codes as they lie are f16
// denormals, which the matrix cores take as well and which cost no and-or and no subtraction; but sums that start at -8 sum q
// to make up for it lose five bits (outputs 7e-6 off float64's, against 2e-7), and the time is the same.
__device__ __forceinline__ h8 unpack8(uint32_t w, uint32_t k) {
  h8 x;
  #pragma unroll
  for (int r = 0; r < 4; r++) {
    const h2 p = __builtin_bit_cast(h2, ((w >> (4 * r)) & 0x000f000fu) | k) - (h2){1032, 1032};
    x[2 * r] = p[0];
    x[2 * r + 1] = p[1];
  }
  return x;
}
// Scale v (of four positions) of entry i (position tile and block) of a lane's loads: taken out of its register where it is
// used, as an operand half.
template <int N>
__device__ __forceinline__ float scale_at(const u4 (&s)[N], int i, int v) {
  const uint32_t w = s[i >> 1][2 * (i & 1) + (v >> 1)];  // (a value of its own: a cast of the element itself takes element 0)
  return (float)__builtin_bit_cast(h2, w)[v & 1];
}
// Weights p times the value scales of their positions (f16 pairs d), rounded to f16, and with LOW the rest, rounded to f16:
// v_fma_mixlo / mixhi round the exact product once, a product in f32 and a conversion twice. The compiler takes either for the
// same source, from one kernel (and one element) to the next; a row's bits must not depend on that, so the instructions are
// written out. (Register halves are read again four instructions after they were written at the earliest.)
template <bool LOW>
__device__ __forceinline__ void weigh8(const float (&p)[8], const uint32_t (&d)[4], u4 &hi, u4 &lo) {
  uint32_t h[4], r[4] = {0, 0, 0, 0};
  #define ZL_MIX(W, A, B, C, SEL) "v_fma_mix" W "_f16 " A ", " B ", " C SEL "\n\t"
  __asm__(ZL_MIX("lo", "%0", "%4", "%12, 0", " op_sel_hi:[0,1,0]") ZL_MIX("lo", "%1", "%6", "%13, 0", " op_sel_hi:[0,1,0]")
          ZL_MIX("lo", "%2", "%8", "%14, 0", " op_sel_hi:[0,1,0]") ZL_MIX("lo", "%3", "%10", "%15, 0", " op_sel_hi:[0,1,0]")
          ZL_MIX("hi", "%0", "%5", "%12, 0", " op_sel:[0,1,0] op_sel_hi:[0,1,0]") ZL_MIX("hi", "%1", "%7", "%13, 0", " op_sel:[0,1,0] op_sel_hi:[0,1,0]")
          ZL_MIX("hi", "%2", "%9", "%14, 0", " op_sel:[0,1,0] op_sel_hi:[0,1,0]") ZL_MIX("hi", "%3", "%11", "%15, 0", " op_sel:[0,1,0] op_sel_hi:[0,1,0]")
          "s_nop 1"
          : "=&v"(h[0]), "=&v"(h[1]), "=&v"(h[2]), "=&v"(h[3])
          : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]), "v"(d[0]), "v"(d[1]), "v"(d[2]), "v"(d[3]));
  if (LOW)
    __asm__(ZL_MIX("lo", "%0", "%4", "%12, -%16", " op_sel_hi:[0,1,1]") ZL_MIX("lo", "%1", "%6", "%13, -%17", " op_sel_hi:[0,1,1]")
            ZL_MIX("lo", "%2", "%8", "%14, -%18", " op_sel_hi:[0,1,1]") ZL_MIX("lo", "%3", "%10", "%15, -%19", " op_sel_hi:[0,1,1]")
            ZL_MIX("hi", "%0", "%5", "%12, -%16", " op_sel:[0,1,1] op_sel_hi:[0,1,1]") ZL_MIX("hi", "%1", "%7", "%13, -%17", " op_sel:[0,1,1] op_sel_hi:[0,1,1]")
            ZL_MIX("hi", "%2", "%9", "%14, -%18", " op_sel:[0,1,1] op_sel_hi:[0,1,1]") ZL_MIX("hi", "%3", "%11", "%15, -%19", " op_sel:[0,1,1] op_sel_hi:[0,1,1]")
            "s_nop 1"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
            : "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]), "v"(p[5]), "v"(p[6]), "v"(p[7]), "v"(d[0]), "v"(d[1]), "v"(d[2]), "v"(d[3]),
              "v"(h[0]), "v"(h[1]), "v"(h[2]), "v"(h[3]));
  #undef ZL_MIX
  hi = u4{h[0], h[1], h[2], h[3]};
  lo = u4{r[0], r[1], r[2], r[3]};
}
__device__ __forceinline__ int wave_max(int v) { return group_reduce(v, 64, [](int x, int y) { return max(x, y); }); }
__device__ __forceinline__ float sum4(float x) { x += swizzle_xor16(x); return x + __shfl_xor(x, 32, 64); }
__device__ __forceinline__ float max4(float x) { x = fmaxf(x, swizzle_xor16(x)); return fmaxf(x, __shfl_xor(x, 32, 64)); }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// A softmax sum in progress; O holds N of the row's dimensions.
template <int N>
struct Sum {
  float m = -INFINITY, l = 0.0f, o[N];
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.0f;
    #pragma unroll
    for (int i = 0; i < N; i++) o[i] = 0.0f;
  }
  // (a piece that saw nothing leaves the sum as it is; one of NaN has l NaN)
  __device__ __forceinline__ void fold(const Sum &p) {
    if (p.m == -INFINITY && p.l == 0.0f) return;
    const float M = fmaxf(m, p.m), r = M == -INFINITY ? 0.0f : M, a = exp2_(m - r), b = exp2_(p.m - r);
    m = M;
    l = fmaf(l, a, p.l * b);
    #pragma unroll
    for (int i = 0; i < N; i++) o[i] = fmaf(o[i], a, p.o[i] * b);
  }
};

// The queries of a tile of 16 rows as right operands: lane l has row l % 16, dimensions 32 b + 8 (l / 16) + e; and the factor
// from the products (code units, scaled queries) to scores in powers of two.
template <int NB>
struct Queries {
  h8 hi[NB], lo[NB];
  float c;
};
template <int NB, int TYPE>
__device__ __forceinline__ void load_queries(Queries<NB> &q, const typename ValueOf<TYPE>::t *row, float scale, int lane) {
  typedef typename ValueOf<TYPE>::t T;
  float v[NB][8], am = 0.0f;
  bool bad = false;
  const T *p = row + 8 * (lane >> 4);
  #pragma unroll
  for (int b = 0; b < NB; b++)
    #pragma unroll
    for (int e = 0; e < 8; e++) v[b][e] = load_value<TYPE>(p[32 * b + e]);
  #pragma unroll
  for (int b = 0; b < NB; b++)
    #pragma unroll
    for (int e = 0; e < 8; e++) {
      am = fmaxf(am, fabsf(v[b][e]));
      bad |= !(fabsf(v[b][e]) < INFINITY);
    }
  am = max4(bad ? INFINITY : am);
  int ex = 0;
  if (am > 0.0f && am < INFINITY) frexpf(am, &ex);
  ex = 14 - ex;  // am 2^ex is in [2^13, 2^14)
  const bool fine = am < INFINITY;  // (a row with a value that is not finite is NaN)
  #pragma unroll
  for (int b = 0; b < NB; b++) {
    #pragma unroll
    for (int e = 0; e < 8; e++) {
      const float x = fine ? ldexpf(v[b][e], ex) : NAN;
      q.hi[b][e] = (_Float16)x;
      q.lo[b][e] = (_Float16)(x - (float)q.hi[b][e]);
    }
  }
  q.c = fmaxf((float)ldexp((double)scale * 1.4426950408889634, -ex), 1.17549435e-38f);  // (not 0: it multiplies -inf)
}

// One span: records rec and rec + 36 HD, of which the lane's row sees positions 0 .. lim (63 or more: all). o[4 j + v] is
// dimension 16 j + 4 (l / 16) + v of row l % 16.
template <int NB, bool LOQ, bool LOW>
__device__ __forceinline__ void span_sum(Sum<8 * NB> &r, const uint8_t *rec, const Queries<NB> &q, int lim, int lane) {
  constexpr int HD = 32 * NB, REC = 36 * HD, NV = NB / 2;
  const int g = lane >> 4;
  uint32_t k1024 = 0x64006400u;
  __asm__("" : "+v"(k1024));
  u4 kw[2][NV], vw[2][NV], ks[2][NB], vs[2][NB];
  #pragma unroll
  for (int i = 0; i < 2; i++) {
    #pragma unroll
    for (int j = 0; j < NV; j++) kw[i][j] = ((const u4 *)(rec + i * REC))[j * 64 + lane];
    #pragma unroll
    for (int j = 0; j < NB; j++) ks[i][j] = ((const u4 *)(rec + i * REC + 32 * HD))[g * NB + j];
  }
  auto load_values = [&]() {
    #pragma unroll
    for (int i = 0; i < 2; i++) {
      #pragma unroll
      for (int j = 0; j < NV; j++) vw[i][j] = ((const u4 *)(rec + i * REC + 16 * HD))[j * 64 + lane];
      #pragma unroll
      for (int j = 0; j < NB; j++) vs[i][j] = ((const u4 *)(rec + i * REC + 34 * HD))[g * NB + j];
    }
  };
  if (NB <= 4) load_values();  // (heads of 256 would not leave registers for them)
  __builtin_amdgcn_sched_barrier(0);
  f4 s[2][2];
  #pragma unroll
  for (int i = 0; i < 2; i++)
    #pragma unroll
    for (int t = 0; t < 2; t++) {
      s[i][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
      #pragma unroll
      for (int b = 0; b < NB; b++) {
        const h8 k = unpack8(kw[i][(t * NB + b) >> 2][(t * NB + b) & 3], k1024);
        f4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q.hi[b], f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
        if (LOQ) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q.lo[b], acc, 0, 0, 0);
        #pragma unroll
        for (int v = 0; v < 4; v++) s[i][t][v] = fmaf(acc[v], scale_at(ks[i], t * NB + b, v), s[i][t][v]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  if (NB > 4) load_values();
  // positions that a row of the tile does not see: no weight, and a scale of 0 (a stale one may be NaN)
  if (__ballot(lim < SPAN - 1)) {
    #pragma unroll
    for (int i = 0; i < 2; i++)
      #pragma unroll
      for (int t = 0; t < 2; t++) {
        const int n = lim - 32 * i - 16 * t - 4 * g;  // the last of the lane's four positions that is seen
        #pragma unroll
        for (int v = 0; v < 4; v++) s[i][t][v] = v > n ? -INFINITY : s[i][t][v];
        const uint32_t m0 = n >= 1 ? 0xffffffffu : n >= 0 ? 0xffffu : 0u, m1 = n >= 3 ? 0xffffffffu : n >= 2 ? 0xffffu : 0u;
        #pragma unroll
        for (int b = 0; b < NB; b++) {
          const int e = t * NB + b;
          vs[i][e >> 1][2 * (e & 1)] &= m0;
          vs[i][e >> 1][2 * (e & 1) + 1] &= m1;
        }
      }
  }
  float m = -INFINITY;
  #pragma unroll
  for (int i = 0; i < 2; i++)
    #pragma unroll
    for (int t = 0; t < 2; t++)
      #pragma unroll
      for (int v = 0; v < 4; v++) {
        m = fmaxf(m, s[i][t][v]);
      }
  m = max4(m);
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  #pragma unroll
  for (int i = 0; i < 2; i++)
    #pragma unroll
    for (int t = 0; t < 2; t++)
      #pragma unroll
      for (int v = 0; v < 4; v++) {
        s[i][t][v] = exp2_(fmaf(s[i][t][v] - ref, q.c, 3.0f));
        l += s[i][t][v];
      }
  r.m = m * q.c - 3.0f;
  r.l = sum4(l);
  __builtin_amdgcn_sched_barrier(0);
  f4 o[2 * NB];
  #pragma unroll
  for (int j = 0; j < 2 * NB; j++) o[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  #pragma unroll
  for (int i = 0; i < 2; i++)
    #pragma unroll
    for (int b = 0; b < NB; b++) {
      u4 hu, lu;
      const float p[8] = {s[i][0][0], s[i][0][1], s[i][0][2], s[i][0][3], s[i][1][0], s[i][1][1], s[i][1][2], s[i][1][3]};
      const uint32_t d[4] = {vs[i][b >> 1][2 * (b & 1)], vs[i][b >> 1][2 * (b & 1) + 1], vs[i][(NB + b) >> 1][2 * (b & 1)],
                             vs[i][(NB + b) >> 1][2 * (b & 1) + 1]};
      weigh8<LOW>(p, d, hu, lu);
      const h8 hi = __builtin_bit_cast(h8, hu), lo = __builtin_bit_cast(h8, lu);
      #pragma unroll
      for (int j = 2 * b; j < 2 * b + 2; j++) {
        const h8 x = unpack8(vw[i][j >> 2][j & 3], k1024);
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, hi, o[j], 0, 0, 0);
        if (LOW) o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, lo, o[j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  #pragma unroll
  for (int j = 0; j < 2 * NB; j++)
    #pragma unroll
    for (int v = 0; v < 4; v++) r.o[4 * j + v] = o[j][v];
}

// The rows of a block: tile t of KV head kvh of sequence s. A row's last position; below 0 it sees nothing.
constexpr int ROW_NONE = -1, ROW_BAD = -2, ROW_ABSENT = -3;
struct Tile {
  int s, kvh, group, ntok, slot, base;  // base: the tile's first row
  bool ok;
  __device__ __forceinline__ Tile(const Kv4Attn &a, int s_, int kvh_, int base_) : s(s_), kvh(kvh_), base(base_) {
    group = a.nhead / a.c.nkv;
    ntok = count_of(a.b, s);
    slot = slot_of(a.b, s);
    ok = slot >= 0 && slot < a.c.nslot;
  }
  __device__ __forceinline__ int last(const Kv4Attn &a, int r, int *tok, int *head) const {
    const int i = base + r, t = i / group;
    *tok = t;
    *head = kvh * group + i - t * group;
    if (t >= ntok) return ROW_ABSENT;
    const long p = (long)a.b.pos[s] + t;
    return !ok || p >= a.c.cap ? ROW_BAD : p < 0 ? ROW_NONE : (int)p;
  }
};

// A chunk's (part's) records: the sums' o [row][record][HD], then their (m, l). Rows count over [sequence][token][head].
__device__ __forceinline__ long row_index(const Kv4Attn &a, int s, int tok, int head) { return ((long)s * a.b.ntok + tok) * a.nhead + head; }
__device__ __forceinline__ float *record_o(const Kv4Attn &a, long row, int rec) { return (float *)a.work + (row * a.nrec + rec) * a.c.hd; }
__device__ __forceinline__ float2 *record_ml(const Kv4Attn &a, long row, int rec) {
  const long rows = (long)a.b.nseq * a.b.ntok * a.nhead;
  return (float2 *)((float *)a.work + rows * a.nrec * a.c.hd) + row * a.nrec + rec;
}
template <int TYPE>
__device__ __forceinline__ void emit(const Kv4Attn &a, int s, int tok, int head, int dim, float o) {
  typedef typename ValueOf<TYPE>::t T;
  ((T *)a.out.p)[s * a.out.seq + tok * a.out.tok + head * a.out.head + dim] = store_value<TYPE>(o);
}

// Few rows: a block takes one tile of 16 rows and a chunk at a time (chunks x, x + X, ...), one span per wave, and folds the
// spans in LDS. Rows that see a single chunk are finished here, the others leave the chunk's record.
template <int NB, int TYPE>
__global__ __launch_bounds__(64 * SPANS) void k_kv4_chunks(const Kv4Attn a, int tiles) {
  constexpr int HD = 32 * NB, LDO = HD + 4;
  constexpr bool LOQ = TYPE == T_F32, LOW = TYPE != T_BF16;
  extern __shared__ __align__(16) float lds[];  // [spans][rows][LDO], then (m, l) [spans][16]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const Tile tl(a, blockIdx.z, blockIdx.y / tiles, blockIdx.y % tiles * 16);
  const int nr = min(16, a.b.ntok * tl.group - tl.base);
  int tok, head;
  const int last = tl.last(a, n, &tok, &head);
  const int most = wave_max(last);
  // the fold's rows: 32 lanes each
  const int fr = tid >> 5, fl = tid & 31;
  int ft, fh;
  const int flast = fr < nr ? tl.last(a, fr, &ft, &fh) : ROW_ABSENT;
  if (blockIdx.x == 0 && (flast == ROW_NONE || flast == ROW_BAD))
    for (int i = 0; i < NB; i++) emit<TYPE>(a, tl.s, ft, fh, 32 * i + fl, flast == ROW_NONE ? 0.0f : NAN);
  if (most < 0 || (int)blockIdx.x * CHUNK > most) return;
  typedef typename ValueOf<TYPE>::t T;
  Queries<NB> q;
  load_queries<NB, TYPE>(q, (const T *)a.q.p + tl.s * a.q.seq + (last >= 0 ? tok * a.q.tok + head * a.q.head : 0), a.scale, lane);
  float2 *ml = (float2 *)(lds + SPANS * nr * LDO);
  for (int c = blockIdx.x; c * CHUNK <= most; c += gridDim.x) {
    const int p0 = c * CHUNK + wave * SPAN;
    if (p0 <= most) {
      Sum<8 * NB> r;
      const uint8_t *rec = record_of(a.c, tl.slot, tl.kvh, p0 / KV4_GROUP);
      const int lim = last - p0;
      span_sum<NB, LOQ, LOW>(r, rec, q, lim, lane);
      if (n < nr) {
        float *d = lds + (wave * nr + n) * LDO + 4 * g;
        #pragma unroll
        for (int j = 0; j < 2 * NB; j++) *(float4 *)(d + 16 * j) = make_float4(r.o[4 * j], r.o[4 * j + 1], r.o[4 * j + 2], r.o[4 * j + 3]);
        if (g == 0) ml[wave * 16 + n] = make_float2(r.m, r.l);
      }
    }
    __syncthreads();
    if (flast >= c * CHUNK) {
      const int ns = min(SPANS, (most - c * CHUNK) / SPAN + 1);
      Sum<NB> f, p;
      f.clear();
      for (int w = 0; w < ns; w++) {
        const float2 v = ml[w * 16 + fr];
        p.m = v.x;
        p.l = v.y;
        #pragma unroll
        for (int i = 0; i < NB; i++) p.o[i] = lds[(w * nr + fr) * LDO + 32 * i + fl];
        f.fold(p);
      }
      if (flast < CHUNK) {
        #pragma unroll
        for (int i = 0; i < NB; i++) emit<TYPE>(a, tl.s, ft, fh, 32 * i + fl, f.o[i] / f.l);
      } else {
        const long row = row_index(a, tl.s, ft, fh);
        float *o = record_o(a, row, c);
        #pragma unroll
        for (int i = 0; i < NB; i++) o[32 * i + fl] = f.o[i];
        if (fl == 0) *record_ml(a, row, c) = make_float2(f.m, f.l);
      }
    }
    __syncthreads();
  }
}

// Rows of several records: 32 lanes per row; `per` records fold into a part, parts into the row. Rows that see at most
// `done` positions have been finished.
template <int NB, int TYPE>
__global__ __launch_bounds__(256) void k_kv4_join(const Kv4Attn a, int done, int reclen) {
  const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int fl = threadIdx.x & 31;
  if (row >= (long)a.b.nseq * a.b.ntok * a.nhead) return;
  const int head = (int)(row % a.nhead), tok = (int)(row / a.nhead % a.b.ntok), s = (int)(row / a.nhead / a.b.ntok);
  const Tile tl(a, s, 0, 0);
  const long last = (long)a.b.pos[s] + tok;
  if (!tl.ok || tok >= tl.ntok || last < done || last >= a.c.cap) return;
  const int nrec = (int)(last / reclen) + 1, per = PART / reclen;
  Sum<NB> f, u, p;
  f.clear();
  u.clear();
  for (int c = 0; c < nrec; c++) {
    const float2 v = *record_ml(a, row, c);
    const float *o = record_o(a, row, c);
    p.m = v.x;
    p.l = v.y;
    #pragma unroll
    for (int i = 0; i < NB; i++) p.o[i] = o[32 * i + fl];
    u.fold(p);
    if (c % per == per - 1 || c == nrec - 1) {
      f.fold(u);
      u.clear();
    }
  }
  #pragma unroll
  for (int i = 0; i < NB; i++) emit<TYPE>(a, s, tok, head, 32 * i + fl, f.o[i] / f.l);
}

// Many rows: a wave takes a tile of 16 rows through the spans of one part, a block four tiles; the parts' records are joined.
template <int NB, int TYPE>
__global__ __launch_bounds__(256) void k_kv4_parts(const Kv4Attn a, int tiles4) {
  constexpr bool LOQ = TYPE == T_F32, LOW = TYPE != T_BF16;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const Tile tl(a, blockIdx.z, blockIdx.y / tiles4, (blockIdx.y % tiles4 * 4 + wave) * 16);
  int tok, head;
  const int last = tl.last(a, n, &tok, &head);
  const int most = wave_max(last), part = blockIdx.x;
  if (part == 0 && (last == ROW_NONE || last == ROW_BAD))
    for (int j = 0; j < 2 * NB; j++)
      for (int v = 0; v < 4; v++) emit<TYPE>(a, tl.s, tok, head, 16 * j + 4 * g + v, last == ROW_NONE ? 0.0f : NAN);
  if (most < part * PART) return;
  typedef typename ValueOf<TYPE>::t T;
  Queries<NB> q;
  load_queries<NB, TYPE>(q, (const T *)a.q.p + tl.s * a.q.seq + (last >= 0 ? tok * a.q.tok + head * a.q.head : 0), a.scale, lane);
  Sum<8 * NB> f, u, r;
  f.clear();
  for (int c = part * CHUNKS; c < (part + 1) * CHUNKS && c * CHUNK <= most; c++) {
    u.clear();
    for (int p0 = c * CHUNK; p0 < (c + 1) * CHUNK && p0 <= most; p0 += SPAN) {
      const uint8_t *rec = record_of(a.c, tl.slot, tl.kvh, p0 / KV4_GROUP);
      const int lim = last - p0;
      span_sum<NB, LOQ, LOW>(r, rec, q, lim, lane);
      u.fold(r);
    }
    f.fold(u);
  }
  if (last < part * PART) return;
  if (last < PART) {
    #pragma unroll
    for (int j = 0; j < 2 * NB; j++)
      #pragma unroll
      for (int v = 0; v < 4; v++) emit<TYPE>(a, tl.s, tok, head, 16 * j + 4 * g + v, f.o[4 * j + v] / f.l);
  } else {
    const long row = row_index(a, tl.s, tok, head);
    float *o = record_o(a, row, part);
    #pragma unroll
    for (int j = 0; j < 2 * NB; j++) *(float4 *)(o + 16 * j + 4 * g) = make_float4(f.o[4 * j], f.o[4 * j + 1], f.o[4 * j + 2], f.o[4 * j + 3]);
    if (g == 0) *record_ml(a, row, part) = make_float2(f.m, f.l);
  }
}

// Whether a call's rows fill the GPU with a wave per (tile, part).
static bool many_rows(const Kv4View &c, int nseq, int ntok, int nhead) {
  const long tiles = ((long)ntok * (nhead / c.nkv) + 15) / 16 * c.nkv * nseq;
  return tiles >= 128;
}
static int record_count(const Kv4View &c, bool many) { return (int)((c.cap + (many ? PART : CHUNK) - 1) / (many ? PART : CHUNK)); }

long kv4_attention_work(const Kv4View &c, int nseq, int ntok, int nhead) {
  const long rows = (long)nseq * ntok * nhead, rec = record_count(c, many_rows(c, nseq, ntok, nhead));
  return std::max(16L, rows * rec * (c.hd + 2) * 4);
}

template <int NB, int TYPE>
static void launch_attention_k(Kv4Attn a, hipStream_t st) {
  const bool many = many_rows(a.c, a.b.nseq, a.b.ntok, a.nhead);
  const int group = a.nhead / a.c.nkv, reclen = many ? PART : CHUNK;
  a.nrec = record_count(a.c, many);
  const long rows = (long)a.b.ntok * group;
  if (many) {
    const long t4 = (rows + 63) / 64;
    hipLaunchKernelGGL((k_kv4_parts<NB, TYPE>), dim3(a.nrec, (unsigned)(t4 * a.c.nkv), a.b.nseq), dim3(256), 0, st, a, (int)t4);
  } else {
    const int tiles = (int)((rows + 15) / 16);
    const size_t lds = (SPANS * std::min(16L, rows) * (32 * NB + 4) + SPANS * 16 * 2) * 4;
    hipLaunchKernelGGL((k_kv4_chunks<NB, TYPE>), dim3(a.nrec, tiles * a.c.nkv, a.b.nseq), dim3(64 * SPANS), lds, st, a, tiles);
  }
  ZL_HIP(hipGetLastError());
  if (a.nrec > 1) {
    const long n = rows * a.c.nkv * a.b.nseq;
    hipLaunchKernelGGL((k_kv4_join<NB, TYPE>), dim3((unsigned)((n + 7) / 8)), dim3(256), 0, st, a, reclen, reclen);
    ZL_HIP(hipGetLastError());
  }
}

// Dynamic LDS above 64 KB is requested per kernel, once per GPU, when a cache is created: no launch changes an attribute.
template <int NB, int TYPE>
static void prepare_k() {
  const int lds = (SPANS * 16 * (32 * NB + 4) + SPANS * 16 * 2) * 4;
  ZL_HIP(hipFuncSetAttribute((const void *)k_kv4_chunks<NB, TYPE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
}
template <int NB>
static void prepare_nb() {
  prepare_k<NB, T_F32>();
  prepare_k<NB, T_F16>();
  prepare_k<NB, T_BF16>();
}
void kv4_prepare(int hd) {
  if (hd == 64) prepare_nb<2>();
  else if (hd == 128) prepare_nb<4>();
  else prepare_nb<8>();
}

template <int NB>
static void launch_attention_t(const Kv4Attn &a, int type, hipStream_t st) {
  if (type == T_F32) launch_attention_k<NB, T_F32>(a, st);
  else if (type == T_F16) launch_attention_k<NB, T_F16>(a, st);
  else launch_attention_k<NB, T_BF16>(a, st);
}
void launch_kv4_attention(const Kv4Attn &a, int type, hipStream_t st) {
  if (a.c.hd == 64) launch_attention_t<2>(a, type, st);
  else if (a.c.hd == 128) launch_attention_t<4>(a, type, st);
  else launch_attention_t<8>(a, type, st);
}

#define ZL_BY_TYPE(type, K, ...)                                             \
  do {                                                                       \
    if ((type) == T_F32) hipLaunchKernelGGL((K<T_F32>), __VA_ARGS__);        \
    else if ((type) == T_F16) hipLaunchKernelGGL((K<T_F16>), __VA_ARGS__);   \
    else hipLaunchKernelGGL((K<T_BF16>), __VA_ARGS__);                       \
    ZL_HIP(hipGetLastError());                                               \
  } while (0)

void launch_kv4_append(const Kv4View &c, const OpBatch &b, int type, const OpRows &k, const OpRows &v, hipStream_t st) {
  const dim3 grid((b.ntok + 30) / KV4_GROUP + 1, c.nkv, b.nseq);  // (a window of n positions touches at most this many records)
  ZL_BY_TYPE(type, k_kv4_append, grid, dim3(256), 32 * c.hd, st, c, b, k, v);
}
void launch_kv4_read(const Kv4View &c, const OpBatch &b, int type, const OpRows &k, const OpRows &v, hipStream_t st) {
  ZL_BY_TYPE(type, k_kv4_read, dim3(b.ntok, c.nkv, b.nseq), dim3(c.hd), 0, st, c, b, k, v);
}
}  // namespace zl
