// KV cache in 4 bits: append, read-back and causal attention (layout in zl_ops.h).
#include "zl_ops.h"
#include <algorithm>

namespace zl {

__device__ __forceinline__ uint8_t *record_of(const Kv4View &c, int slot, int head, long group) {
  return c.base + (((long)slot * c.nkv + head) * c.ngroup + group) * kv4_record(c.hd);
}
// The batch's tokens of sequence s, and the position of the first.
__device__ __forceinline__ int count_of(const OpBatch &b, int s) { return b.count ? max(0, min(b.count[s], b.tok0 + b.ntok) - b.tok0) : b.ntok; }
__device__ __forceinline__ long pos_of(const OpBatch &b, int s) { return (long)b.pos[s] + b.tok0; }
__device__ __forceinline__ int slot_of(const OpBatch &b, int s) { return b.slot ? b.slot[s] : s; }

// ---------------------------------------------------------------------------------------------- append
// One block per (32-position record that a sequence may touch, KV head, sequence). A lane takes 8 values, four lanes a block
// of 32 (kv4_quant). The codes go to LDS and from there in whole words: a key word is one lane's 8 values; a value word holds 8
// positions, and those that are not appended keep their codes. With slots, the block of the first sequence that touches a record of
// its slot takes all of them, in order, found 256 at a time (one by one, 4096 sequences of 8 heads took 17 ms for 0.4, and their square
// beyond).
// Bound by the loads' latency: all of a record's are requested together (2048 tokens of 8 heads of 128, bf16: 37 us with a
// value per lane and a load at a time).
template <int TYPE, bool VEC>
__device__ __forceinline__ void load8(const typename ValueOf<TYPE>::t *p, float (&x)[8]) {
  typedef typename ValueOf<TYPE>::t T;
  constexpr int W = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(W)));
  if constexpr (VEC) {
    #pragma unroll
    for (int i = 0; i < 8 / W; i++) {
      const vec v = ((const vec *)p)[i];
      #pragma unroll
      for (int e = 0; e < W; e++) x[i * W + e] = load_value<TYPE>(v[e]);
    }
  } else {
    #pragma unroll
    for (int e = 0; e < 8; e++) x[e] = load_value<TYPE>(p[e]);
  }
}

__device__ __forceinline__ unsigned long long uniform(unsigned long long x) {
  return (unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

template <int NB, int TYPE, bool VEC>
__global__ __launch_bounds__(256) void k_kv4_append(const Kv4View c, const OpBatch b, const OpRows k, const OpRows v) {
  typedef typename ValueOf<TYPE>::t T;
  constexpr int HD = 32 * NB, UNITS = 32 * 4 * NB / 256;  // a lane's pieces of 8 keys (of 8 values) of a whole record
  __shared__ uint32_t kw[4 * HD];
  __shared__ uint64_t vn[32][HD / 8];  // value codes, a byte each
  const int s0 = blockIdx.z, head = blockIdx.y, tid = threadIdx.x;
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
  uint8_t *rec = record_of(c, slot, head, g);
  // with slots: the sequences of the slot that touch the record, 256 at a time; one before s0 has a block that takes them all
  __shared__ unsigned long long same[4];
  for (int base = b.slot ? 0 : s0; base < (b.slot ? b.nseq : s0 + 1); base += 256) {
    if (b.slot) {
      const int s = base + tid;
      long x, y;
      const unsigned long long m = __ballot(s < b.nseq && b.slot[s] == slot && touches(s, &x, &y));
      if ((tid & 63) == 0) same[tid >> 6] = m;
      __syncthreads();
    }
    for (int sw = 0; sw < (b.slot ? 4 : 1); sw++)
      for (unsigned long long left = b.slot ? uniform(same[sw]) : 1; left; left &= left - 1) {
        const int s = base + 64 * sw + __ffsll(left) - 1;
        if (s < s0) return;
        touches(s, &p0, &p1);
        const int n = (int)(p1 - p0), q0 = (int)(p0 - g * KV4_GROUP);
        const long t0 = p0 - b.pos[s];
        float x[2][UNITS][8];
        #pragma unroll
        for (int isv = 0; isv < 2; isv++)
          #pragma unroll
          for (int u = 0; u < UNITS; u++) {
            const int i = u * 256 + tid, t = i / (4 * NB), d8 = i % (4 * NB);
            const OpRows &r = isv ? v : k;
            if (t < n) load8<TYPE, VEC>((const T *)r.p + s * r.seq + (t0 + t) * r.tok + head * r.head + 8 * d8, x[isv][u]);
          }
        #pragma unroll
        for (int isv = 0; isv < 2; isv++)
          #pragma unroll
          for (int u = 0; u < UNITS; u++) {
            const int i = u * 256 + tid, t = i / (4 * NB), d8 = i % (4 * NB), p = q0 + t;
            if (t >= n) continue;  // (four lanes of a block of 32 go together)
            int code[8];
            const uint16_t scale = kv4_quant(x[isv][u], tid, code);
            if ((tid & 3) == 0) ((uint16_t *)(rec + (isv ? 34 : 32) * HD))[kv4_scale(p, d8 >> 2, NB)] = scale;
            uint64_t bytes = 0;
            #pragma unroll
            for (int e = 0; e < 8; e++) bytes |= (uint64_t)code[e] << (8 * e);
            if (isv) vn[p][d8] = bytes;
            else kw[kv4_word((p >> 4) * NB + (d8 >> 2), (p & 15) + 16 * (d8 & 3))] = kv4_pack(code);
          }
        __syncthreads();
        uint32_t *kd = (uint32_t *)rec, *vd = (uint32_t *)(rec + 16 * HD);
        #pragma unroll
        for (int u = 0; u < 4 * HD / 256; u++) {
          const int i = u * 256 + tid, lane = i >> 2 & 63, w4 = (i >> 8) * 4 + (i & 3);  // dword i of the words
          const int p = (lane & 15) + 16 * (w4 / NB);
          if (p >= q0 && p < q0 + n) kd[i] = kw[i];
          const int dim = 16 * w4 + (lane & 15), gq = lane >> 4;
          uint32_t w = 0, m = 0;
          #pragma unroll
          for (int e = 0; e < 8; e++) {
            const int q = 16 * (e >> 2) + 4 * gq + (e & 3);
            if (q >= q0 && q < q0 + n) {
              w |= (uint32_t)((const uint8_t *)vn[q])[dim] << (4 * kv4_nibble(e));
              m |= 0xfu << (4 * kv4_nibble(e));
            }
          }
          if (m) vd[i] = m == 0xffffffffu ? w : (vd[i] & ~m) | w;
        }
        __syncthreads();
      }
    if (b.slot) __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------- read-back
// One block per (32 tokens, KV head, sequence); a lane takes 8 values of a token's key, then of its value.
template <int NB, int TYPE, bool VEC>
__global__ __launch_bounds__(256) void k_kv4_read(const Kv4View c, const OpBatch b, const OpRows k, const OpRows v) {
  typedef typename ValueOf<TYPE>::t T;
  constexpr int HD = 32 * NB, W = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(W)));
  const int head = blockIdx.y, s = blockIdx.z, n = count_of(b, s), slot = slot_of(b, s);
  #pragma unroll
  for (int i = threadIdx.x; i < 32 * 4 * NB; i += 256) {
    const int t = blockIdx.x * 32 + i / (4 * NB), d8 = i % (4 * NB);
    if (t >= n) continue;
    const long pos = (long)b.pos[s] + t;
    const bool ok = slot >= 0 && slot < c.nslot && pos >= 0 && pos < c.cap;
    const int p = (int)(pos & 31);
    const uint8_t *rec = ok ? record_of(c, slot, head, pos >> 5) : nullptr;
    #pragma unroll
    for (int isv = 0; isv < 2; isv++) {
      const OpRows &o = isv ? v : k;
      T *out = (T *)o.p + s * o.seq + t * o.tok + head * o.head + 8 * d8;
      T y[8];
      #pragma unroll
      for (int e = 0; e < 8; e++) y[e] = store_value<TYPE>(NAN);
      if (ok) {
        const uint32_t *w = (const uint32_t *)(rec + isv * 16 * HD);
        const float d = h2f(((const uint16_t *)(rec + (32 + 2 * isv) * HD))[kv4_scale(p, d8 >> 2, NB)]);
        const uint32_t kword = isv ? 0 : w[kv4_word((p >> 4) * NB + (d8 >> 2), (p & 15) + 16 * (d8 & 3))];
        #pragma unroll
        for (int e = 0; e < 8; e++) {
          const int dim = 8 * d8 + e;
          const uint32_t x = isv ? w[kv4_word(dim >> 4, (dim & 15) + 16 * ((p >> 2) & 3))] : kword;
          y[e] = store_value<TYPE>(d * (float)((int)((x >> (4 * kv4_nibble(isv ? 4 * (p >> 4) + (p & 3) : e))) & 15) - 8));
        }
      }
      if constexpr (VEC) {
        #pragma unroll
        for (int j = 0; j < 8 / W; j++) {
          vec u;
          #pragma unroll
          for (int e = 0; e < W; e++) u[e] = y[j * W + e];
          ((vec *)out)[j] = u;
        }
      } else {
        #pragma unroll
        for (int e = 0; e < 8; e++) out[e] = y[e];
      }
    }
  }
}

// Whether every head of the rows starts on a 16-byte boundary.
static bool whole_pieces(const OpRows &r, int type) {
  const int w = 16 / value_bytes(type);
  return (uintptr_t)r.p % 16 == 0 && r.seq % w == 0 && r.tok % w == 0 && r.head % w == 0;
}
template <int NB, int TYPE, bool VEC>
static void launch_kv(bool read, const Kv4View &c, const OpBatch &b, const OpRows &k, const OpRows &v, hipStream_t st) {
  // (a window of n positions touches at most (n + 30) / 32 + 1 records)
  if (read) hipLaunchKernelGGL((k_kv4_read<NB, TYPE, VEC>), dim3((b.ntok - 1) / 32 + 1, c.nkv, b.nseq), dim3(256), 0, st, c, b, k, v);
  else hipLaunchKernelGGL((k_kv4_append<NB, TYPE, VEC>), dim3((unsigned)(((long)b.ntok + 30) / KV4_GROUP + 1), c.nkv, b.nseq), dim3(256), 0, st, c, b, k, v);
  ZL_HIP(hipGetLastError());
}
template <int NB, int TYPE>
static void launch_kv_v(bool read, const Kv4View &c, const OpBatch &b, const OpRows &k, const OpRows &v, hipStream_t st) {
  if (whole_pieces(k, TYPE) && whole_pieces(v, TYPE)) launch_kv<NB, TYPE, true>(read, c, b, k, v, st);
  else launch_kv<NB, TYPE, false>(read, c, b, k, v, st);
}
template <int NB>
static void launch_kv_t(bool read, const Kv4View &c, const OpBatch &b, int type, const OpRows &k, const OpRows &v, hipStream_t st) {
  if (type == T_F32) launch_kv_v<NB, T_F32>(read, c, b, k, v, st);
  else if (type == T_F16) launch_kv_v<NB, T_F16>(read, c, b, k, v, st);
  else launch_kv_v<NB, T_BF16>(read, c, b, k, v, st);
}
static void launch_kv_nb(bool read, const Kv4View &c, const OpBatch &b, int type, const OpRows &k, const OpRows &v, hipStream_t st) {
  if (c.hd == 64) launch_kv_t<2>(read, c, b, type, k, v, st);
  else if (c.hd == 128) launch_kv_t<4>(read, c, b, type, k, v, st);
  else launch_kv_t<8>(read, c, b, type, k, v, st);
}
void launch_kv4_append(const Kv4View &c, const OpBatch &b, int type, const OpRows &k, const OpRows &v, hipStream_t st) {
  launch_kv_nb(false, c, b, type, k, v, st);
}
void launch_kv4_read(const Kv4View &c, const OpBatch &b, int type, const OpRows &k, const OpRows &v, hipStream_t st) {
  launch_kv_nb(true, c, b, type, k, v, st);
}

// ---------------------------------------------------------------------------------------------- attention
// softmax(scale q K) V of a row (a token's query head) over positions 0 .. last, in f32 with the exponentials to base 2. The
// positions are cut, by their index alone, into spans of 64, chunks of 256 (4 spans) and parts of 1024 (4 chunks). A span has
// a softmax of its own: its reference m (the largest score less 3, so that weights reach 8), l = sum of weights and
// o = sum of weights times values. Spans are folded into their chunk in order, chunks into their part:
//   M' = max(M, m), L = L 2^(M - M') + l 2^(m - M'), O = O 2^(M - M') + o 2^(m - M').
// Parts are joined into the row (JOIN_PARTS).
// Whichever block or kernel forms a piece, it does these operations, so a row has the same bits in a batch of any size and
// in a cache of any capacity.
//
// Products run on the matrix cores (v_mfma_f32_16x16x32_f16) for 16 rows at a time: keys times queries first, which leaves
// lane l with the scores of row l % 16 at four neighbouring positions, then values (as the left operand) times weights,
// which takes those positions as they lie. Codes less 8 are exact in f16. Queries are scaled per row by a power of two to
// below 2^14 and split into two f16 parts (22 bits; 16-bit queries need one); a weight times its value's scale likewise, whatever the
// output's type: rounded to one f16 part, and the product again, it would be off by 2^-11 twice, more than an f16 output's own
// rounding, and 7 to 9 % of bf16 outputs would be other numbers than the rounded f32 ones. Scores are scaled by their key's scale in
// f32, block by block.
constexpr int SPAN = 64, CHUNK = 256, PART = 1024;
constexpr int CHUNKS = PART / CHUNK;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The eight codes of a word, less 8, as f16 operands: pair r of (word >> 4 r), under an exponent and less the sum of both: 1024 where
// the code is in the lowest bits, 64 where it is four higher (no shift; 36 cycles a word). (Codes as they lie, as f16 denormals, take
// 12, but the matrix cores' sums of those lose bits: outputs of f16 rows other than the rounded f32 ones 2 to 4 % instead of 0.1 to
// 0.4, for 190 us instead of 200 a call of 256 tokens after 12000 positions.)
// The constants are in vector registers: a 32-bit operation takes 2 cycles of a SIMD from two waves' vector operands and 4 with a
// scalar one, and and-or takes a single scalar one.
struct Unpack {
  uint32_t mask = 0x000f000fu, k1024 = 0x64006400u, mask4 = 0x00f000f0u, k64 = 0x54005400u;
  __device__ __forceinline__ Unpack() { __asm__("" : "+v"(mask), "+v"(k1024), "+v"(mask4), "+v"(k64)); }
};
__device__ __forceinline__ h8 unpack8(uint32_t w, const Unpack &k) {
  u4 x;
  #pragma unroll
  for (int r = 0; r < 4; r++) {
    const uint32_t v = r < 2 ? w : w >> 8;
    const h2 p = r & 1 ? __builtin_bit_cast(h2, (v & k.mask4) | k.k64) - (h2){72, 72} : __builtin_bit_cast(h2, (v & k.mask) | k.k1024) - (h2){1032, 1032};
    x[r] = __builtin_bit_cast(uint32_t, p);
  }
  return __builtin_bit_cast(h8, x);
}
// Scale v (of four positions) of entry i (position tile and block) of a lane's loads: taken out of its register where it is
// used, as an operand half.
template <int N>
__device__ __forceinline__ float scale_at(const u4 (&s)[N], int i, int v) {
  const uint32_t w = s[i >> 1][2 * (i & 1) + (v >> 1)];  // (a value of its own: a cast of the element itself takes element 0)
  return (float)__builtin_bit_cast(h2, w)[v & 1];
}
__device__ __forceinline__ int wave_max(int v) { return group_reduce(v, 64, [](int x, int y) { return max(x, y); }); }
// Over the four lanes l % 16 + 0, 16, 32, 48: rows of 16 lanes are swapped pairwise (16, then 32 apart), no trip through LDS.
template <class T, class Op>
__device__ __forceinline__ T over4(T x, Op op) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x);
  const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t p0 = p[0], p1 = p[1], b = __builtin_bit_cast(uint32_t, op(__builtin_bit_cast(T, p0), __builtin_bit_cast(T, p1)));
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const uint32_t q0 = q[0], q1 = q[1];
  return op(__builtin_bit_cast(T, q0), __builtin_bit_cast(T, q1));
}
__device__ __forceinline__ float sum4(float x) { return over4(x, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ float max4(float x) { return over4(x, [](float a, float b) { return fmaxf(a, b); }); }
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
  // (a piece that saw nothing has m = -inf and l = o = 0, and adds 0; one of NaN has l NaN)
  __device__ __forceinline__ void fold(const Sum &p) {
    const float M = fmaxf(m, p.m), r = M == -INFINITY ? 0.0f : M, a = exp2_(m - r), b = exp2_(p.m - r);
    m = M;
    l = fmaf(p.l, b, l * a);
    #pragma unroll
    for (int i = 0; i < N; i++) o[i] = fmaf(p.o[i], b, o[i] * a);
  }
};

// K pieces at once, the first `n` of them: what folding them one by one gives, with the factors formed side by side.
template <int K, int N>
__device__ __forceinline__ void fold_all(Sum<N> &f, const float2 (&ml)[K], const float (&o)[K][N], int n) {
  float M = f.m, a[K], b[K];
  #pragma unroll
  for (int k = 0; k < K; k++) {
    const float to = fmaxf(M, k < n ? ml[k].x : -INFINITY), r = to == -INFINITY ? 0.0f : to;
    a[k] = exp2_(M - r);
    b[k] = exp2_(ml[k].x - r);
    M = to;
  }
  f.m = M;
  #pragma unroll
  for (int k = 0; k < K; k++) {
    if (k >= n) break;
    f.l = fmaf(ml[k].y, b[k], f.l * a[k]);
    #pragma unroll
    for (int i = 0; i < N; i++) f.o[i] = fmaf(o[k][i], b[k], f.o[i] * a[k]);
  }
}

// The queries of a tile of 16 rows as right operands: lane l has row l % 16, dimensions 32 b + 8 (l / 16) + e; and the factor
// from the products (code units, scaled queries) to scores in powers of two.
template <int NB>
struct Queries {
  h8 hi[NB], lo[NB];
  float c;
};
template <int NB, int TYPE>
__device__ __forceinline__ void fetch_queries(float (&v)[NB][8], const typename ValueOf<TYPE>::t *row, bool vec, int lane) {
  const typename ValueOf<TYPE>::t *p = row + 8 * (lane >> 4);
  if (vec) {
    #pragma unroll
    for (int b = 0; b < NB; b++) load8<TYPE, true>(p + 32 * b, v[b]);
  } else {
    #pragma unroll
    for (int b = 0; b < NB; b++) load8<TYPE, false>(p + 32 * b, v[b]);
  }
}
template <int NB>
__device__ __forceinline__ void set_queries(Queries<NB> &q, const float (&v)[NB][8], float scale) {
  float am = 0.0f, any = 0.0f;
  #pragma unroll
  for (int b = 0; b < NB; b++)
    #pragma unroll
    for (int e = 0; e < 8; e++) {
      am = fmaxf(am, fabsf(v[b][e]));
      any = fmaf(v[b][e], 0.0f, any);  // 0, or NaN where a value is not finite: the row is NaN then
    }
  am = max4(am);
  any = sum4(any);
  // a power of two that takes the largest value to [2^13, 2^14); rows below 2^-112 stay smaller: their scores are 0 all the same
  int ex = 0;
  if (am > 0.0f) frexpf(am, &ex);
  ex = min(126, 14 - ex);
  const float up = __uint_as_float((uint32_t)(127 + ex) << 23) + any;
  #pragma unroll
  for (int b = 0; b < NB; b++) {
    u4 hi, lo;
    #pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x0 = v[b][2 * e] * up, x1 = v[b][2 * e + 1] * up;
      const h2 h = {(_Float16)x0, (_Float16)x1};
      const h2 r = {(_Float16)fmaf(-1.0f, (float)h[0], x0), (_Float16)fmaf(-1.0f, (float)h[1], x1)};
      hi[e] = __builtin_bit_cast(uint32_t, h);
      lo[e] = __builtin_bit_cast(uint32_t, r);
    }
    q.hi[b] = __builtin_bit_cast(h8, hi);
    q.lo[b] = __builtin_bit_cast(h8, lo);
  }
  // (neither 0 nor infinite: it multiplies infinities and zeros)
  q.c = fminf(fmaxf((float)ldexp((double)scale * 1.4426950408889634, -ex), 1.17549435e-38f), 3.40282347e38f);
}

// A lane's share of a span (two records): code words and scales, loaded with every lane's 16-byte loads side by side.
template <int NB>
struct SpanWords {
  static constexpr int HD = 32 * NB, REC = 36 * HD, NV = NB / 2;
  u4 kw[2][NV], ks[2][NB], vw[2][NV], vs[2][NB];
  __device__ __forceinline__ void load_keys(const uint8_t *rec, int lane) {
    #pragma unroll
    for (int i = 0; i < 2; i++) {
      #pragma unroll
      for (int j = 0; j < NV; j++) kw[i][j] = ((const u4 *)(rec + i * REC))[j * 64 + lane];
      #pragma unroll
      for (int j = 0; j < NB; j++) ks[i][j] = ((const u4 *)(rec + i * REC + 32 * HD))[(lane >> 4) * NB + j];
    }
  }
  __device__ __forceinline__ void load_values(const uint8_t *rec, int lane) {
    #pragma unroll
    for (int i = 0; i < 2; i++) {
      #pragma unroll
      for (int j = 0; j < NV; j++) vw[i][j] = ((const u4 *)(rec + i * REC + 16 * HD))[j * 64 + lane];
      #pragma unroll
      for (int j = 0; j < NB; j++) vs[i][j] = ((const u4 *)(rec + i * REC + 34 * HD))[(lane >> 4) * NB + j];
    }
  }
};

// Scores of 16 positions (tile t of a record) in code units, from the tile's operands k(b) and key scales.
template <int NB, bool LOQ, class K>
__device__ __forceinline__ f4 tile_scores(const K &k, const u4 (&ks)[NB], int t, const Queries<NB> &q) {
  f4 s = f4{0.0f, 0.0f, 0.0f, 0.0f};
  #pragma unroll
  for (int b = 0; b < NB; b++) {
    const h8 x = k(b);
    f4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.hi[b], f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
    if (LOQ) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.lo[b], acc, 0, 0, 0);
    #pragma unroll
    for (int v = 0; v < 4; v++) s[v] = fmaf(acc[v], scale_at(ks, t * NB + b, v), s[v]);
  }
  return s;
}

// Positions that the lane's row does not see (those behind lim of the span): no weight, ... (in spans at the rows' ends only:
// the empty asm, which lim depends on, keeps the compiler from making selects of it that every span would pay for)
__device__ __forceinline__ void mask_scores(f4 (&s)[2][2], int lim, int g) {
  __asm__ volatile("" : "+v"(lim));
  #pragma unroll
  for (int i = 0; i < 2; i++)
    #pragma unroll
    for (int t = 0; t < 2; t++)
      #pragma unroll
      for (int v = 0; v < 4; v++) s[i][t][v] = 32 * i + 16 * t + 4 * g + v > lim ? -INFINITY : s[i][t][v];
}
// ... and a scale of 0 (a stale one may be NaN): record i's value scales.
template <int NB>
__device__ __forceinline__ void mask_scales(u4 (&vs)[NB], int i, int lim, int g) {
  __asm__ volatile("" : "+v"(lim));
  #pragma unroll
  for (int t = 0; t < 2; t++) {
    const int n = lim - 32 * i - 16 * t - 4 * g;  // the last of the lane's four positions that is seen
    const uint32_t m0 = n >= 1 ? 0xffffffffu : n >= 0 ? 0xffffu : 0u, m1 = n >= 3 ? 0xffffffffu : n >= 2 ? 0xffffu : 0u;
    #pragma unroll
    for (int b = 0; b < NB; b++) {
      const int e = t * NB + b;
      vs[e >> 1][2 * (e & 1)] &= m0;
      vs[e >> 1][2 * (e & 1) + 1] &= m1;
    }
  }
}

// Value scales d of a block that are all below 2^-5: a weight times such a scale would end, in two f16 parts, at 2^-25 of the
// weights' 8, few bits below that (values of 1e-5 made outputs 4e-3 off). Where a span's largest one that the lane's row sees is below, they
// are taken times 2^15, twice if that leaves them there (denormals), which is exact, and the block's sums times the same less. It goes by
// the row and the span's positions alone, so that a row's bits do not depend on the batch. Returns two bits a block, the times. The look
// costs 2 to 3 % of a call, the raising 17 to 25 % (256 tokens after 12000 positions, f16: 197 us, values of 0.05 242).
constexpr uint32_t SMALL_SCALE = 0x2800;  // 2^-5 in f16
// Whether a block of the span may be such a one for any row that sees the span: none is where every lane has a scale of 2^-5 or more
// among its four positions of tile 0 of record 0, in every block. The rest is left out then, which changes no bit.
template <int NB>
__device__ __forceinline__ bool maybe_small(const u4 (&vs)[NB], int lim) {
  uint32_t all = 0x80008000u;
  #pragma unroll
  for (int b = 0; b < NB; b++) {
    // (no carry from the lower half: 0x7fff + 0x5800 < 2^16)
    constexpr uint32_t up = (0x8000u - SMALL_SCALE) * 0x10001u;
    uint32_t x = ((vs[b >> 1][2 * (b & 1)] & 0x7fff7fffu) + up) | ((vs[b >> 1][2 * (b & 1) + 1] & 0x7fff7fffu) + up);
    x |= x << 16;
    all &= x;
  }
  return __ballot((all >> 31) == 0 && lim >= 0) != 0;
}
template <int NB>
__device__ __forceinline__ uint32_t raise_small(u4 (&v0)[NB], u4 (&v1)[NB]) {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  uint32_t times = 0;
  #pragma unroll 1
  for (int round = 0; round < 2; round++) {
    #pragma unroll
    for (int b = 0; b < NB; b++) {
      us2 m = {0, 0};
      #pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint32_t x = v0[((k >> 1) * NB + b) >> 1][2 * (b & 1) + (k & 1)] & 0x7fff7fffu, y = v1[((k >> 1) * NB + b) >> 1][2 * (b & 1) + (k & 1)] & 0x7fff7fffu;
        m = __builtin_elementwise_max(m, __builtin_elementwise_max(__builtin_bit_cast(us2, x), __builtin_bit_cast(us2, y)));
      }
      const uint32_t top = over4((uint32_t)max(m[0], m[1]), [](uint32_t x, uint32_t y) { return max(x, y); });  // (NaN above all)
      const bool small = top < SMALL_SCALE;
      const h2 f = small ? (h2){32768, 32768} : (h2){1, 1};
      times += (small ? 1u : 0u) << (2 * b);
      #pragma unroll
      for (int k = 0; k < 4; k++) {
        const int i = ((k >> 1) * NB + b) >> 1, j = 2 * (b & 1) + (k & 1);
        const uint32_t w0 = v0[i][j], w1 = v1[i][j];
        v0[i][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, w0) * f);
        v1[i][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, w1) * f);
      }
    }
    if (!__ballot(times != 0)) break;
  }
  return times;
}
template <int NB>
__device__ __forceinline__ void lower_sums(f4 (&o)[2 * NB], uint32_t times) {
  #pragma unroll
  for (int b = 0; b < NB; b++) {
    const float f = __uint_as_float((127u - 15u * (times >> (2 * b) & 3u)) << 23);
    #pragma unroll
    for (int v = 0; v < 4; v++) o[2 * b][v] *= f, o[2 * b + 1][v] *= f;
  }
}

// Weights of a lane's positions (four neighbouring ones of each tile of both records) in two f16 parts.
struct Weights {
  h2 hi[2][2][2], lo[2][2][2];  // [record][tile][pair]
};
// Scores to weights; the span's reference and the sum of its weights.
__device__ __forceinline__ void span_softmax(const f4 (&s)[2][2], float c, Weights &w, float &m, float &l) {
  float x = -INFINITY;
  #pragma unroll
  for (int i = 0; i < 2; i++)
    #pragma unroll
    for (int t = 0; t < 2; t++)
      #pragma unroll
      for (int v = 0; v < 4; v++) x = fmaxf(x, s[i][t][v]);
  x = max4(x);
  const float ref = x == -INFINITY ? 0.0f : x;
  l = 0.0f;
  #pragma unroll
  for (int i = 0; i < 2; i++)
    #pragma unroll
    for (int t = 0; t < 2; t++)
      #pragma unroll
      for (int v = 0; v < 4; v += 2) {
        const float p0 = exp2_(fmaf(s[i][t][v] - ref, c, 3.0f)), p1 = exp2_(fmaf(s[i][t][v + 1] - ref, c, 3.0f));
        l += p0;
        l += p1;
        const h2 h = {(_Float16)p0, (_Float16)p1};
        w.hi[i][t][v >> 1] = h;
        // (the differences are exact, so that they are rounded once in whatever instructions they are formed)
        w.lo[i][t][v >> 1] = (h2){(_Float16)fmaf(-1.0f, (float)h[0], p0), (_Float16)fmaf(-1.0f, (float)h[1], p1)};
      }
  m = x * c - 3.0f;
  l = sum4(l);
}

// Weights of record i times the value scales d of block b, as right operands, in packed f16: hi = f16(ph d), and the rest
// lo = f16(f16(ph d - hi) + pl d), the inner difference exact. Every step rounds once, in whichever kernel it is.
template <int NB>
__device__ __forceinline__ void weigh(const Weights &w, const u4 (&vs)[NB], int i, int b, h8 &hi, h8 &lo) {
  const uint32_t d[4] = {vs[b >> 1][2 * (b & 1)], vs[b >> 1][2 * (b & 1) + 1], vs[(NB + b) >> 1][2 * (b & 1)], vs[(NB + b) >> 1][2 * (b & 1) + 1]};
  #pragma unroll
  for (int k = 0; k < 4; k++) {
    const h2 e = __builtin_bit_cast(h2, d[k]), p = w.hi[i][k >> 1][k & 1], h = p * e;
    hi[2 * k] = h[0];
    hi[2 * k + 1] = h[1];
    const h2 r = __builtin_elementwise_fma(w.lo[i][k >> 1][k & 1], e, __builtin_elementwise_fma(p, e, -h));
    lo[2 * k] = r[0];
    lo[2 * k + 1] = r[1];
  }
}

// Blocks of a one-dimensional grid, which the GPU deals to its 8 XCDs in turn: `groups` of n blocks that read the same records, each
// on one XCD, whose L2 then holds them.
__host__ __device__ inline long deal_blocks(long groups, int n) { return (groups + 7) / 8 * 8 * n; }
__device__ __forceinline__ bool dealt(long groups, int n, long *group, int *i) {
  const long j = blockIdx.x >> 3;
  *i = (int)(j % n);
  *group = j / n * 8 + (blockIdx.x & 7);
  return *group < groups;
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
    const long p = pos_of(a.b, s) + t;
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
// Where outputs go: rows of the caller's type, or a model's (32 dimensions on 32 lanes).
// (+ 0: a sum of -0 comes out the same whether it was folded with empty pieces or not)
template <int TYPE>
struct ToRows {
  OpRows r;
  __device__ __forceinline__ void emit(int s, int tok, int head, int dim, float o) const {
    ((typename ValueOf<TYPE>::t *)r.p)[s * r.seq + tok * r.tok + head * r.head + dim] = store_value<TYPE>(o + 0.0f);
  }
  void skip(int seqs) { r.p = (char *)r.p + seqs * r.seq * value_bytes(TYPE); }
};
struct ToModel {
  HeadOut h;
  __device__ __forceinline__ void emit(int, int tok, int head, int dim, float o) const { attn_emit(h, tok, head, dim, o + 0.0f); }
  void skip(int) {}  // (one sequence)
};

// A span's products of block b and record: values times weights.
__device__ __forceinline__ void weighted_sums(f4 &o0, f4 &o1, h8 x0, h8 x1, h8 hi, h8 lo) {
  o0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x0, hi, o0, 0, 0, 0);
  o1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x1, hi, o1, 0, 0, 0);
  o0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x0, lo, o0, 0, 0, 0);
  o1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x1, lo, o1, 0, 0, 0);
}

// Positions per record of a sequence's rows (of k_kv4_rows<.., false>): by the sequence's last position, so that all its rows agree.
__device__ __forceinline__ int record_len(const Kv4Attn &a, int s) {
  const long last = min(pos_of(a.b, s) + count_of(a.b, s), a.c.cap) - 1;
  return last < (long)a.spanmax * SPAN ? SPAN : CHUNK;
}

// A tile's finished sums: the rows' outputs where a call has one record per row, else record `rec` of the rows that see it. Lane
// l has row l % 16, dimensions 16 j + 4 (l / 16) + v.
template <int NB, int TYPE>
__device__ __forceinline__ void leave(const Kv4Attn &a, const Tile &tl, int last, int tok, int head, int rec, int first, const Sum<8 * NB> &f, int g) {
  if (a.direct) {
    if (last == ROW_ABSENT) return;
    const ToRows<TYPE> out{a.out};
    #pragma unroll
    for (int j = 0; j < 2 * NB; j++)
      #pragma unroll
      for (int v = 0; v < 4; v++)
        out.emit(tl.s, a.b.tok0 + tok, head, 16 * j + 4 * g + v, last >= 0 ? f.o[4 * j + v] / f.l : last == ROW_NONE ? 0.0f : NAN);
    return;
  }
  if (last < first) return;
  const long row = row_index(a, tl.s, tok, head);
  float *o = record_o(a, row, rec) + 4 * g;
  #pragma unroll
  for (int j = 0; j < 2 * NB; j++) *(f4 *)(o + 16 * j) = f4{f.o[4 * j], f.o[4 * j + 1], f.o[4 * j + 2], f.o[4 * j + 3]};
  if (g == 0) *record_ml(a, row, rec) = make_float2(f.m, f.l);
}

// A wave takes one tile of 16 rows through chunks (few rows) or parts (MANY), span by span, and leaves the piece's record; no wave
// waits for another. The next span's keys are requested when the scores are done with this one's, its values after the weighted
// sums, so that the loads run under the rest. (A chunk of 512 per block, one span per wave, folded in LDS behind a barrier: 9 tokens
// of 32 heads after 16384 positions 48 us against 41. Eight waves of a block sharing spans unpacked into LDS, one meeting a span:
// 256 tokens after 12000 positions 240 us against 189, as both were then.)
// Few rows: sequences of so few spans that a wave for each does not overfill the GPU (a.spanmax, by the call's tiles) leave a record
// per span instead: four times the waves, each a quarter as long (a token after 700 positions 13 us -> 8). A token of 32 heads of
// 128 over 8 KV heads after 131000 positions: 43 us, 151 MB at 3.5 TB/s, near a read's own rate (4.1). 9 tokens after 16384: 26 us,
// bound by the vector units, 1.5 waves a SIMD, and by the waves' start and end.
// MANY: the block's waves have neighbouring tiles of the same part, whose records they read at about the same time. 256 tokens of 32
// heads over 8 after 12000 positions, f16: 188 us, bound by the vector units: some 710 vector instructions and 48 matrix ones a span of
// a tile, with two waves to hide the matrix instructions' latency.
// Registers: heads of 64 take 173 to 187 VGPRs, heads of 128 all 256 (f32 rows spill 2 to 6 of them, 12 to 28 bytes a lane, outside the
// loop over spans), heads of 256 also 115 to 150 AGPRs, which leaves them one wave a SIMD.
template <int NB, int TYPE, bool MANY>
__global__ __launch_bounds__(256, NB <= 4 ? 2 : 1) void k_kv4_rows(const Kv4Attn a, int tiles, int gx) {
  constexpr int HD = 32 * NB;
  constexpr bool LOQ = TYPE == T_F32, AHEAD = NB <= 4;  // (heads of 256 leave no registers for loads ahead)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  // the wave's tile, and its first chunk (MANY: part) and the step to the next
  long group;  // [sequence][KV head][block of chunks (a part)]
  int tile, c0, step;
  if (!dealt((long)gx * a.c.nkv * a.b.nseq, MANY ? (tiles + 3) / 4 : tiles, &group, &tile)) return;
  if (MANY) tile = tile * 4 + wave, c0 = (int)(group % gx), step = gx;
  else c0 = (int)(group % gx) * 4 + wave, step = gx * 4;
  const Tile tl(a, (int)(group / gx / a.c.nkv), (int)(group / gx % a.c.nkv), tile * 16);
  int tok, head;
  const int last = tl.last(a, n, &tok, &head);
  const int most = __builtin_amdgcn_readfirstlane(wave_max(last));
  const int unit = MANY ? PART : record_len(a, tl.s);
  __shared__ f4 part[MANY ? 4 : 1][MANY ? 2 * NB : 1][64];  // MANY: the part's o, a column per lane (registers hold one sum, not two)
  Sum<8 * NB> u;
  u.clear();
  if (most < (long)c0 * unit) {
    if (a.direct && c0 == 0) leave<NB, TYPE>(a, tl, last, tok, head, 0, 0, u, g);
    return;
  }
  typedef typename ValueOf<TYPE>::t T;
  const Unpack uk;
  // (loads complete in order: the queries, which take a while to prepare, are requested first)
  SpanWords<NB> w;
  Queries<NB> q;
  {
    float qv[NB][8];
    fetch_queries<NB, TYPE>(qv, (const T *)a.q.p + tl.s * a.q.seq + (last >= 0 ? (a.b.tok0 + tok) * a.q.tok + head * a.q.head : 0), a.qvec, lane);
    const uint8_t *rec = record_of(a.c, tl.slot, tl.kvh, (long)c0 * (unit / KV4_GROUP));
    w.load_keys(rec, lane);
    if (AHEAD) w.load_values(rec, lane);
    __builtin_amdgcn_sched_barrier(0);
    set_queries<NB>(q, qv, a.scale);
  }
  for (int c = c0; (long)c * unit <= most; c += step) {
    const int ns = min(unit / SPAN, (most - c * unit) / SPAN + 1);
    float pm = -INFINITY, pl = 0.0f;
    if (MANY) {
      #pragma unroll
      for (int j = 0; j < 2 * NB; j++) part[wave][j][lane] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int sp = 0; sp < ns;) {
      u.clear();
      for (const int end = min(sp + CHUNK / SPAN, ns); sp < end; sp++) {
        const int p0 = c * unit + sp * SPAN, lim = last - p0;
        const int pn = sp + 1 < ns ? p0 + SPAN : (long)(c + step) * unit <= most ? (c + step) * unit : p0;  // (the last one is read again, for nothing)
        const uint8_t *rec = record_of(a.c, tl.slot, tl.kvh, p0 / KV4_GROUP), *next = record_of(a.c, tl.slot, tl.kvh, pn / KV4_GROUP);
        const bool masked = __ballot(lim < SPAN - 1) != 0;
        f4 s[2][2];
        #pragma unroll
        for (int i = 0; i < 2; i++)
          #pragma unroll
          for (int t = 0; t < 2; t++) {
            s[i][t] = tile_scores<NB, LOQ>([&](int b) { return unpack8(w.kw[i][(t * NB + b) >> 2][(t * NB + b) & 3], uk); }, w.ks[i], t, q);
            __builtin_amdgcn_sched_barrier(0);
          }
        if (AHEAD) w.load_keys(next, lane);
        else w.load_values(rec, lane);
        __builtin_amdgcn_sched_barrier(0);
        if (masked) {
          mask_scores(s, lim, g);
          mask_scales<NB>(w.vs[0], 0, lim, g);
          mask_scales<NB>(w.vs[1], 1, lim, g);
        }
        Sum<8 * NB> r;
        Weights pw;
        span_softmax(s, q.c, pw, r.m, r.l);
        // (only here, where the values' loads have had the softmax to arrive)
        const bool small = maybe_small<NB>(w.vs[0], lim);
        uint32_t times = 0;
        if (small) times = raise_small<NB>(w.vs[0], w.vs[1]);
        f4 o[2 * NB];
        #pragma unroll
        for (int j = 0; j < 2 * NB; j++) o[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        #pragma unroll
        for (int i = 0; i < 2; i++)
          #pragma unroll
          for (int b = 0; b < NB; b++) {
            h8 hi, lo;
            weigh<NB>(pw, w.vs[i], i, b, hi, lo);
            const h8 x0 = unpack8(w.vw[i][(2 * b) >> 2][(2 * b) & 3], uk), x1 = unpack8(w.vw[i][(2 * b + 1) >> 2][(2 * b + 1) & 3], uk);
            weighted_sums(o[2 * b], o[2 * b + 1], x0, x1, hi, lo);
            __builtin_amdgcn_sched_barrier(0);
          }
        if (AHEAD) w.load_values(next, lane);
        else w.load_keys(next, lane);
        __builtin_amdgcn_sched_barrier(0);
        if (small) lower_sums<NB>(o, times);
        #pragma unroll
        for (int j = 0; j < 2 * NB; j++)
          #pragma unroll
          for (int v = 0; v < 4; v++) r.o[4 * j + v] = o[j][v];
        u.fold(r);
      }
      if (MANY) {
        const float M = fmaxf(pm, u.m), ref = M == -INFINITY ? 0.0f : M, x = exp2_(pm - ref), y = exp2_(u.m - ref);
        pm = M;
        pl = fmaf(u.l, y, pl * x);
        #pragma unroll
        for (int j = 0; j < 2 * NB; j++) {
          f4 o = part[wave][j][lane];
          #pragma unroll
          for (int v = 0; v < 4; v++) o[v] = fmaf(u.o[4 * j + v], y, o[v] * x);
          part[wave][j][lane] = o;
        }
      }
    }
    if (MANY) {
      u.m = pm;
      u.l = pl;
      #pragma unroll
      for (int j = 0; j < 2 * NB; j++)
        #pragma unroll
        for (int v = 0; v < 4; v++) u.o[4 * j + v] = part[wave][j][lane][v];
    }
    leave<NB, TYPE>(a, tl, last, tok, head, c, c * unit, u, g);
  }
}

// A row of a call, its last position (as Tile::last) and whether it is the call's to write.
__device__ __forceinline__ int row_of(const Kv4Attn &a, long row, int *s, int *tok, int *head) {
  *head = (int)(row % a.nhead);
  *tok = (int)(row / a.nhead % a.b.ntok);
  *s = (int)(row / a.nhead / a.b.ntok);
  if (*tok >= count_of(a.b, *s)) return ROW_ABSENT;
  const int slot = slot_of(a.b, *s);
  const long p = pos_of(a.b, *s) + *tok;
  return slot < 0 || slot >= a.c.nslot || p >= a.c.cap ? ROW_BAD : p < 0 ? ROW_NONE : (int)p;
}

// Parts to a row: up to 128 of them (131072 positions) side by side, weighted by 2^(m - M) of their largest M and summed into eight
// sums by their index, which are added in order; such sums are folded one after the other.
constexpr int JOIN_PARTS = 128, JOIN_SUMS = 8;

// Rows of chunk or span records, few of them: a block per (row, 32 dimensions), a dimension per lane. Its groups of 32 lanes fold the
// chunks of a part each, the loads of AT parts issued together, and eight of them sum the parts up. Rows of up to 32 parts have 8
// groups, longer ones 32.
template <int GROUPS, class OUT>
__global__ __launch_bounds__(32 * GROUPS) void k_kv4_join_chunks(const Kv4Attn a, const OUT out) {
  constexpr int AT = GROUPS == 8 ? 2 : 4, MOST = GROUPS == 8 ? 32 : JOIN_PARTS;
  __shared__ float po[MOST][32], so[JOIN_SUMS][32];
  __shared__ float2 pml[MOST];
  __shared__ float sl[JOIN_SUMS];
  const int fl = threadIdx.x & 31, grp = threadIdx.x >> 5, dim = blockIdx.y * 32 + fl;
  int s, tok, head;
  const int last = row_of(a, blockIdx.x, &s, &tok, &head);
  if (last == ROW_ABSENT) return;
  if (last < 0) {
    if (grp == 0) out.emit(s, a.b.tok0 + tok, head, dim, last == ROW_NONE ? 0.0f : NAN);
    return;
  }
  const int len = record_len(a, s), nrec = last / len + 1;
  const int np = last / PART + 1;
  const float *o = record_o(a, blockIdx.x, 0) + dim;
  const float2 *ml = record_ml(a, blockIdx.x, 0);
  Sum<1> f;
  f.clear();
  for (int b0 = 0; b0 < np; b0 += MOST) {
    const int n = min(MOST, np - b0);
    if (len == CHUNK) {
      for (int i0 = grp; i0 < n; i0 += AT * GROUPS) {
        float x[AT][CHUNKS][1];
        float2 v[AT][CHUNKS];
        #pragma unroll
        for (int i = 0; i < AT; i++)
          #pragma unroll
          for (int k = 0; k < CHUNKS; k++) {
            const int c = min((b0 + i0 + i * GROUPS) * CHUNKS + k, nrec - 1);
            x[i][k][0] = o[(long)c * a.c.hd];
            v[i][k] = ml[c];
          }
        #pragma unroll
        for (int i = 0; i < AT; i++) {
          const int p = i0 + i * GROUPS;
          if (p >= n) break;
          Sum<1> u;
          u.clear();
          fold_all<CHUNKS, 1>(u, v[i], x[i], nrec - (b0 + p) * CHUNKS);
          po[p][fl] = u.o[0];
          if (fl == 0) pml[p] = make_float2(u.m, u.l);
        }
      }
    } else {
      static_assert(CHUNK / SPAN == CHUNKS, "records folded at a time");
      for (int p = grp; p < n; p += GROUPS) {
        Sum<1> u;
        u.clear();
        for (int j0 = (b0 + p) * CHUNKS; j0 < (b0 + p + 1) * CHUNKS && j0 * CHUNKS < nrec; j0 += 2) {  // two chunks' loads together
          float x[2][CHUNKS][1];
          float2 v[2][CHUNKS];
          #pragma unroll
          for (int j = 0; j < 2; j++)
            #pragma unroll
            for (int k = 0; k < CHUNKS; k++) {
              const int c = min((j0 + j) * CHUNKS + k, nrec - 1);
              x[j][k][0] = o[(long)c * a.c.hd];
              v[j][k] = ml[c];
            }
          #pragma unroll
          for (int j = 0; j < 2; j++) {
            if ((j0 + j) * CHUNKS >= nrec) break;
            Sum<1> c;
            c.clear();
            fold_all<CHUNKS, 1>(c, v[j], x[j], nrec - (j0 + j) * CHUNKS);
            u.fold(c);
          }
        }
        po[p][fl] = u.o[0];
        if (fl == 0) pml[p] = make_float2(u.m, u.l);
      }
    }
    __syncthreads();
    float M = -INFINITY;
    if (grp < JOIN_SUMS) {
      for (int p = fl; p < n; p += 32) M = fmaxf(M, pml[p].x);
      M = group_reduce(M, 32, [](float x, float y) { return fmaxf(x, y); });
      const float r = M == -INFINITY ? 0.0f : M;
      float l = 0.0f, x = 0.0f;
      for (int p = grp; p < n; p += JOIN_SUMS) {
        const float w = exp2_(pml[p].x - r);
        l = fmaf(pml[p].y, w, l);
        x = fmaf(po[p][fl], w, x);
      }
      so[grp][fl] = x;
      if (fl == 0) sl[grp] = l;
    }
    __syncthreads();
    if (grp == 0) {
      Sum<1> u;
      u.m = M;
      u.l = sl[0];
      u.o[0] = so[0][fl];
      #pragma unroll
      for (int i = 1; i < JOIN_SUMS; i++) u.l += sl[i], u.o[0] += so[i][fl];
      f.fold(u);
    }
  }
  if (grp == 0) out.emit(s, a.b.tok0 + tok, head, dim, f.o[0] / f.l);
}

// Rows of part records, many of them: 32 lanes per row.
template <int NB, class OUT>
__global__ __launch_bounds__(256) void k_kv4_join_parts(const Kv4Attn a, const OUT out) {
  const long row = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int fl = threadIdx.x & 31;
  if (row >= (long)a.b.nseq * a.b.ntok * a.nhead) return;
  int s, tok, head;
  const int last = row_of(a, row, &s, &tok, &head);
  if (last == ROW_ABSENT) return;
  Sum<NB> f;
  f.clear();
  const int np = last < 0 ? 0 : last / PART + 1;
  const float *o = record_o(a, row, 0) + fl;
  const float2 *ml = record_ml(a, row, 0);
  for (int b0 = 0; b0 < np; b0 += JOIN_PARTS) {
    const int n = min(JOIN_PARTS, np - b0);
    Sum<NB> u[JOIN_SUMS];
    float M = -INFINITY;
    for (int p = fl; p < n; p += 32) M = fmaxf(M, ml[b0 + p].x);
    M = group_reduce(M, 32, [](float x, float y) { return fmaxf(x, y); });
    const float r = M == -INFINITY ? 0.0f : M;
    #pragma unroll
    for (int k = 0; k < JOIN_SUMS; k++) u[k].clear();
    for (int p0 = 0; p0 < n; p0 += JOIN_SUMS) {
      #pragma unroll
      for (int k = 0; k < JOIN_SUMS; k++) {
        const int p = b0 + min(p0 + k, n - 1);
        const float2 v = ml[p];
        const float w = p0 + k < n ? exp2_(v.x - r) : 0.0f;
        if (p0 + k < n) {
          u[k].l = fmaf(v.y, w, u[k].l);
          #pragma unroll
          for (int i = 0; i < NB; i++) u[k].o[i] = fmaf(o[(long)p * a.c.hd + 32 * i], w, u[k].o[i]);
        }
      }
    }
    #pragma unroll
    for (int k = 1; k < JOIN_SUMS; k++) {
      u[0].l += u[k].l;
      #pragma unroll
      for (int i = 0; i < NB; i++) u[0].o[i] += u[k].o[i];
    }
    u[0].m = M;
    f.fold(u[0]);
  }
  #pragma unroll
  for (int i = 0; i < NB; i++) out.emit(s, a.b.tok0 + tok, head, 32 * i + fl, last >= 0 ? f.o[i] / f.l : last == ROW_NONE ? 0.0f : NAN);
}

// Tiles of 16 rows times KV heads times sequences.
static long tile_count(const Kv4View &c, int nseq, int ntok, int nhead) { return ((long)ntok * (nhead / c.nkv) + 15) / 16 * c.nkv * nseq; }
// Whether a call takes a wave per (tile, part): where they fill the GPU's SIMDs, and there are enough rows that the records of chunks
// would cost more than the longer runs. (f16 queries of one sequence, 32 heads over 8, us, records of chunks : of parts, 16 tokens a
// call = 32 tiles:
//   after    16 tokens  32        48        64        128       256
//   1000     21 : 40    30 : 42   38 : 42   42 : 42   57 : 43   98 : 46
//   4000     28 : 42    36 : 43   41 : 44   47 : 44   78 : 68   141 : 84
//   16000    34 : 48    54 : 51   86 : 72   91 : 74   165 : 133 337 : 241
//   60000    112 : 86   212 : 139 349 : 192 422 : 245 872 : 455 1744 : 841.) The cache's capacity stands for the length, which the
// host does not know; with fewer tiles a short sequence in a large cache would lose more than a long one gains.
// Batches of single tokens are not told apart, and mostly lose by parts: a block's four waves take four tiles of one (sequence, KV
// head), so that three of them have nothing to do. (The same heads, 4 / 8 / 16 / 32 / 64 sequences, chunks : parts after 500: 14 : 23,
// 14 : 23, 17 : 23, 24 : 23, 38 : 25; after 4000 20 : 44, 29 : 44, 32 : 46, 53 : 69, 92 : 89; after 16000 29 : 50, 45 : 73, 78 : 119,
// 143 : 220, 270 : 428; parts from 16 sequences on, and from 4 in caches of 32768.)
static bool many_rows(const Kv4View &c, int nseq, int ntok, int nhead) {
  const long tiles = tile_count(c, nseq, ntok, nhead);
  return tiles >= 128 || (tiles >= 32 && tiles * ((c.cap + PART - 1) / PART) >= 1024);
}
// Spans of a sequence up to which its rows have a record per span: as many as give about two waves a SIMD.
static int span_max(const Kv4View &c, long tiles) { return (int)std::min((c.cap + SPAN - 1) / SPAN, 2048 / tiles); }
// How a call is run: the records of a row, and slabs of `seqs` sequences and `toks` tokens one after the other in the same work space, so
// that it stays below WORK_MOST bytes (one token's records apart), however long the prompt and large the cache are, and the
// launches within 2^32 threads. A row has the same bits in any slab. (2048 tokens of 32 heads of 128 in a cache of 131072: 4.1 GB as
// one, nine slabs of 240 tokens.)
struct AttnPlan {
  bool many;
  int nrec, spanmax, seqs, toks;
};
constexpr long WORK_MOST = 1L << 29, BLOCKS_MOST = 1L << 22;
static AttnPlan attn_plan(const Kv4View &c, int nseq, int ntok, int nhead) {
  AttnPlan p;
  p.many = many_rows(c, nseq, ntok, nhead);
  p.spanmax = p.many ? 0 : span_max(c, tile_count(c, nseq, ntok, nhead));
  p.nrec = p.many ? (int)((c.cap + PART - 1) / PART) : (int)std::max((c.cap + CHUNK - 1) / CHUNK, (long)p.spanmax);
  const long token = (long)nhead * p.nrec * (c.hd + 2) * 4, fit = WORK_MOST / token;
  p.seqs = nseq;
  p.toks = ntok;
  if (fit < ntok) {
    p.seqs = 1;
    p.toks = (int)(fit >= 16 ? fit / 16 * 16 : std::max(1L, fit));  // (whole tiles)
  } else {
    p.seqs = (int)std::min((long)nseq, fit / ntok);
    const long blocks = tile_count(c, 1, ntok, nhead);  // of a sequence, at most
    p.seqs = (int)std::max(1L, std::min((long)p.seqs, BLOCKS_MOST / blocks));
  }
  return p;
}

long kv4_attention_work(const Kv4View &c, int nseq, int ntok, int nhead) {
  if (nseq == 0 || ntok == 0) return 16;
  const AttnPlan p = attn_plan(c, nseq, ntok, nhead);
  return std::max(16L, (long)p.seqs * p.toks * nhead * p.nrec * (c.hd + 2) * 4);
}

template <int NB, int TYPE, class OUT>
static void launch_slab(const Kv4Attn &a, bool many, const OUT &out, hipStream_t st) {
  const int group = a.nhead / a.c.nkv;
  const long rows = (long)a.b.ntok * group;
  const int tiles = (int)((rows + 15) / 16);
  // waves up to two a SIMD (all on the GPU at once, whichever CUs the blocks are dealt to), each with an even share of the
  // parts (chunks) beyond; or of spans
  const int units = many ? a.nrec : (int)((a.c.cap + CHUNK - 1) / CHUNK);
  const long y = (long)tiles * a.c.nkv * a.b.nseq, rounds = (units * y + 2047) / 2048;
  if (many) {
    // (not units / rounds: the last part of a cache is seldom full)
    const int gx = (int)std::min((long)units, std::max(1L, 2048 / y));
    hipLaunchKernelGGL((k_kv4_rows<NB, TYPE, true>), dim3((unsigned)deal_blocks((long)gx * a.c.nkv * a.b.nseq, (tiles + 3) / 4)), dim3(256), 0, st, a, tiles, gx);
  } else {
    const int gx = std::max((int)((units + 4 * rounds - 1) / (4 * rounds)), (a.spanmax + 3) / 4);
    hipLaunchKernelGGL((k_kv4_rows<NB, TYPE, false>), dim3((unsigned)deal_blocks((long)gx * a.c.nkv * a.b.nseq, tiles)), dim3(256), 0, st, a, tiles, gx);
  }
  ZL_HIP(hipGetLastError());
  if (!a.direct) {
    const long n = rows * a.c.nkv * a.b.nseq;
    if (many) hipLaunchKernelGGL((k_kv4_join_parts<NB, OUT>), dim3((unsigned)((n + 7) / 8)), dim3(256), 0, st, a, out);
    else if (a.c.cap > 32 * PART) hipLaunchKernelGGL((k_kv4_join_chunks<32, OUT>), dim3((unsigned)n, NB), dim3(1024), 0, st, a, out);
    else hipLaunchKernelGGL((k_kv4_join_chunks<8, OUT>), dim3((unsigned)n, NB), dim3(256), 0, st, a, out);
    ZL_HIP(hipGetLastError());
  }
}

template <int NB, int TYPE, class OUT>
static void launch_attention_k(Kv4Attn a, OUT out, bool direct, hipStream_t st) {
  const AttnPlan p = attn_plan(a.c, a.b.nseq, a.b.ntok, a.nhead);
  a.nrec = p.nrec;
  a.spanmax = p.spanmax;
  a.qvec = whole_pieces(a.q, TYPE);
  a.direct = direct && a.nrec == 1;
  const OpBatch all = a.b;
  for (int s = 0; s < all.nseq; s += p.seqs) {
    a.b.nseq = std::min(p.seqs, all.nseq - s);
    for (a.b.tok0 = 0; a.b.tok0 < all.ntok; a.b.tok0 += p.toks) {
      a.b.ntok = std::min(p.toks, all.ntok - a.b.tok0);
      launch_slab<NB, TYPE>(a, p.many, out, st);
    }
    a.b.pos += p.seqs;
    if (a.b.count) a.b.count += p.seqs;
    if (a.b.slot) {
      a.b.slot += p.seqs;
    } else {
      a.c.base += (long)p.seqs * a.c.nkv * a.c.ngroup * kv4_record(a.c.hd);
      a.c.nslot -= p.seqs;
    }
    a.q.p = (char *)a.q.p + p.seqs * a.q.seq * value_bytes(TYPE);
    if (a.direct) a.out.p = (char *)a.out.p + p.seqs * a.out.seq * value_bytes(TYPE);
    out.skip(p.seqs);
  }
}

template <int NB>
static void launch_attention_t(const Kv4Attn &a, int type, hipStream_t st) {
  if (type == T_F32) launch_attention_k<NB, T_F32>(a, ToRows<T_F32>{a.out}, true, st);
  else if (type == T_F16) launch_attention_k<NB, T_F16>(a, ToRows<T_F16>{a.out}, true, st);
  else launch_attention_k<NB, T_BF16>(a, ToRows<T_BF16>{a.out}, true, st);
}
void launch_kv4_attention(const Kv4Attn &a, int type, hipStream_t st) {
  if (a.c.hd == 64) launch_attention_t<2>(a, type, st);
  else if (a.c.hd == 128) launch_attention_t<4>(a, type, st);
  else launch_attention_t<8>(a, type, st);
}
void launch_kv4_attention_model(const Kv4Attn &a, const HeadOut &out, hipStream_t st) {
  if (a.c.hd == 64) launch_attention_k<2, T_F32>(a, ToModel{out}, false, st);
  else if (a.c.hd == 128) launch_attention_k<4, T_F32>(a, ToModel{out}, false, st);
  else launch_attention_k<8, T_F32>(a, ToModel{out}, false, st);
}

}  // namespace zl
