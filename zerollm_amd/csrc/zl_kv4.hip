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
// One block per (query head, token, sequence): 64 positions at a time, a position per lane of the first wave for the
// scores, a dimension per thread for the weighted sum.
template <int TYPE>
__global__ __launch_bounds__(256) void k_kv4_attend(const Kv4Attn a) {
  typedef typename ValueOf<TYPE>::t T;
  __shared__ float qs[256], ps[64];
  __shared__ float red;
  const Kv4View &c = a.c;
  const int h = blockIdx.x, t = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, hd = c.hd;
  if (t >= count_of(a.b, s)) return;
  const int slot = slot_of(a.b, s), kvh = h / (a.nhead / c.nkv);
  const long last = (long)a.b.pos[s] + t;
  T *out = (T *)a.out.p + s * a.out.seq + t * a.out.tok + h * a.out.head;
  const bool ok = slot >= 0 && slot < c.nslot && last < c.cap;
  const T *q = (const T *)a.q.p + s * a.q.seq + t * a.q.tok + h * a.q.head;
  if (tid < hd) qs[tid] = load_value<TYPE>(q[tid]);
  __syncthreads();
  if (!ok || last < 0) {
    if (tid < hd) out[tid] = store_value<TYPE>(ok ? 0.0f : NAN);
    return;
  }
  float M = -INFINITY, L = 0.0f, O = 0.0f;
  for (long p0 = 0; p0 <= last; p0 += 64) {
    if (tid < 64) {
      const long p = p0 + tid;
      float x = -INFINITY;
      if (p <= last) {
        const uint8_t *rec = record_of(c, slot, kvh, p >> 5);
        x = 0.0f;
        for (int i = 0; i < hd; i++) x = fmaf(qs[i], kv4_value(rec, hd, 0, (int)(p & 31), i), x);
        x *= a.scale;
      }
      ps[tid] = x;
      const float m = group_fmax(x, 64);
      if (tid == 0) red = m;
    }
    __syncthreads();
    const float M1 = fmaxf(M, red), r = M1 == -INFINITY ? 0.0f : M1, f = expf(M - r);
    L *= f;
    O *= f;
    M = M1;
    for (int j = 0; j < 64 && p0 + j <= last; j++) {
      const float e = expf(ps[j] - r);
      L += e;
      if (tid < hd) O = fmaf(e, kv4_value(record_of(c, slot, kvh, (p0 + j) >> 5), hd, 1, (int)((p0 + j) & 31), tid), O);
    }
    __syncthreads();
  }
  if (tid < hd) out[tid] = store_value<TYPE>(O / L);
}

long kv4_attention_work(const Kv4View &c, int nseq, int ntok, int nhead) { return 16; }

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
void launch_kv4_attention(const Kv4Attn &a, int type, hipStream_t st) {
  ZL_BY_TYPE(type, k_kv4_attend, dim3(a.nhead, a.b.ntok, a.b.nseq), dim3(256), 0, st, a);
}

}  // namespace zl
