// Rotary positions: queries and keys of a batch rotated in one launch.
#include "zl_ops.h"
#include <algorithm>

namespace zl {

// cos and sin of 2 pi t: t is cut to its nearest quarter turn in f64 (exact), so that the rest, at most an eighth of a turn
// either way, keeps 24 bits in f32 at any position; Taylor polynomials there (the first terms left out are below 2e-9).
__device__ __forceinline__ void turn_sincos(double t, float *c, float *s) {
  const double q = rint(4.0 * t);
  const float x = (float)((t - 0.25 * q) * 6.283185307179586), y = x * x;
  const float sn = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
  const float cs = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
  const int k = (int)(long long)q & 3;
  const float a = k & 1 ? sn : cs, b = k & 1 ? cs : sn;
  *c = k == 1 || k == 2 ? -a : a;
  *s = k >= 2 ? -b : b;
}

template <int TYPE> constexpr int value_size() { return sizeof(typename ValueOf<TYPE>::t); }
template <class T, int W> struct Piece {
  typedef T t __attribute__((ext_vector_type(W)));
  typedef t loose __attribute__((aligned(sizeof(T))));  // one that starts at any value
};

// A block takes `tb` tokens of a sequence and a share of their heads (blockIdx.z): the tokens' cos and sin go to LDS once, then
// every lane takes pieces of the rows. WHOLE: every row is whole 16-byte pieces of V values. Neighbouring pairs: a piece's pairs
// are rotated or pass through one by one. Halves: V pairs' firsts and seconds (which start anywhere), the last ones of a half one by
// one, then the pieces behind the rotated values, of which the first may start among them. Bound by HBM: each value is read and written once (16384
// tokens of 40 heads of 128, 64 rotated, bf16: 80 us, 4.2 TB/s; with whole pieces only where the parts of the head were some too,
// 2 of 64 values rotated took 59 us a call of 11269 tokens of 24 heads; they take 18 as neighbours, 35 as halves).
template <int TYPE, bool HALF, bool WHOLE>
__global__ __launch_bounds__(256) void k_rope(const RopeArgs a, int tb, int hb) {
  typedef typename ValueOf<TYPE>::t T;
  constexpr int V = WHOLE ? 16 / sizeof(T) : 1;
  typedef typename Piece<T, V>::t whole;
  typedef typename Piece<T, V>::loose loose;
  extern __shared__ float2 cs[];  // [tokens][half]
  const int s = blockIdx.y, tid = threadIdx.x, t0 = blockIdx.x * tb, half = a.half, nrot = 2 * half;
  const int nt = min(tb, (a.b.count ? max(0, min(a.b.count[s], a.b.ntok)) : a.b.ntok) - t0);
  if (nt <= 0) return;
  const int p0 = a.b.pos[s];
  for (int i = tid; i < nt * half; i += 256) {
    const int t = i / half, r = i - t * half;
    float c, n;
    turn_sincos(((double)p0 + (t0 + t)) * a.turns[r], &c, &n);
    cs[i] = make_float2(c * a.gain, n * a.gain);
  }
  __syncthreads();
  // pieces of a head: rotated ones, then those behind
  const int rp = HALF ? (half + V - 1) / V : WHOLE ? a.hd / V : half, items = rp + (HALF || !WHOLE ? a.hd / V - nrot / V : 0);
  const int h0 = blockIdx.z * hb, nh = min(hb, a.nq + a.nk - h0), total = nt * nh * items;
  for (int i = tid; i < total; i += 256) {
    const int row = i / items, r = i - row * items, t = row / nh, h = h0 + row - t * nh;
    const bool isq = h < a.nq;
    const OpRows &x = isq ? a.q : a.k, &y = isq ? a.qo : a.ko;
    const long hh = isq ? h : h - a.nq;
    const T *xp = (const T *)x.p + s * x.seq + (t0 + t) * x.tok + hh * x.head;
    T *yp = (T *)y.p + s * y.seq + (t0 + t) * y.tok + hh * y.head;
    if (r >= rp) {
      const int d = (nrot / V + r - rp) * V;
      const whole u = *(const whole *)(xp + d);
      if (d >= nrot) {
        *(whole *)(yp + d) = u;
      } else {
        typedef typename Piece<T, 2>::t two;
        #pragma unroll
        for (int e = 0; e < V; e += 2)  // (rotated values come in twos)
          if (d + e >= nrot) *(two *)(yp + d + e) = two{u[e], u[e + 1]};
      }
      continue;
    }
    const float2 *f = cs + t * half;
    if constexpr (HALF) {
      const int d = r * V;
      auto turn = [&](float x0, float x1, int i, T *y0, T *y1) {
        const float2 g = f[i];
        *y0 = store_value<TYPE>(fmaf(x0, g.x, -(x1 * g.y)));
        *y1 = store_value<TYPE>(fmaf(x0, g.y, x1 * g.x));
      };
      if (d + V <= half) {
        whole u = *(const whole *)(xp + d), v = *(const loose *)(xp + d + half);
        #pragma unroll
        for (int e = 0; e < V; e++) {
          T y0, y1;
          turn(load_value<TYPE>(u[e]), load_value<TYPE>(v[e]), d + e, &y0, &y1);
          u[e] = y0;
          v[e] = y1;
        }
        *(whole *)(yp + d) = u;
        *(loose *)(yp + d + half) = v;
      } else {
        T u[V], v[V];  // (all loads before the stores: one wait)
        #pragma unroll
        for (int e = 0; e < V - 1; e++) {
          const int i = min(d + e, half - 1);
          u[e] = xp[i];
          v[e] = xp[i + half];
        }
        #pragma unroll
        for (int e = 0; e < V - 1; e++)
          if (d + e < half) turn(load_value<TYPE>(u[e]), load_value<TYPE>(v[e]), d + e, yp + d + e, yp + d + e + half);
      }
    } else if constexpr (WHOLE) {
      const int d = r * V;
      whole u = *(const whole *)(xp + d);
      #pragma unroll
      for (int e = 0; e < V; e += 2) {
        if (d + e >= nrot) break;
        const float x0 = load_value<TYPE>(u[e]), x1 = load_value<TYPE>(u[e + 1]);
        const float2 g = f[(d + e) >> 1];
        u[e] = store_value<TYPE>(fmaf(x0, g.x, -(x1 * g.y)));
        u[e + 1] = store_value<TYPE>(fmaf(x0, g.y, x1 * g.x));
      }
      *(whole *)(yp + d) = u;
    } else {
      const float x0 = load_value<TYPE>(xp[2 * r]), x1 = load_value<TYPE>(xp[2 * r + 1]);
      const float2 g = f[r];
      yp[2 * r] = store_value<TYPE>(fmaf(x0, g.x, -(x1 * g.y)));
      yp[2 * r + 1] = store_value<TYPE>(fmaf(x0, g.y, x1 * g.x));
    }
  }
}

// Rows of 16-byte pieces: every start and stride, and the head.
static bool whole_pieces(const RopeArgs &a, int vb) {
  const int w = 16 / vb;
  auto ok = [&](const OpRows &r) {
    return (uintptr_t)r.p % 16 == 0 && r.seq % w == 0 && r.tok % w == 0 && r.head % w == 0;
  };
  return ok(a.q) && ok(a.qo) && (!a.nk || (ok(a.k) && ok(a.ko))) && a.hd % w == 0;
}

template <int TYPE, bool HALF, bool WHOLE>
static void launch_rope_k(const RopeArgs &a, hipStream_t st) {
  // Tokens and heads per block: pieces for every lane a few times over where there are many tokens, as many blocks as CUs
  // where there are few (each of which forms its tokens' cos and sin itself: 2 half values a block).
  constexpr int V = WHOLE ? 16 / value_size<TYPE>() : 1;
  const int heads = a.nq + a.nk, nrot = 2 * a.half;
  const int pieces = HALF ? (a.half + V - 1) / V + a.hd / V - nrot / V : WHOLE ? a.hd / V : a.half + a.hd - nrot;
  const long all = (long)a.b.ntok * a.b.nseq * heads * pieces;
  const long per = std::max(256L, std::min(4096L, all / 512));  // pieces per block
  const int hb = (int)std::max(1L, std::min((long)heads, per / pieces));
  // (at least the tokens that keep the grid's first dimension below 2^32 threads: up to 8 of the 2^26 a call may have)
  const int tb = (int)std::max({1L, std::min({(long)a.b.ntok, per / ((long)hb * pieces), 16L}), ((long)a.b.ntok + (1 << 23) - 1) >> 23});
  const dim3 grid((unsigned)((a.b.ntok + tb - 1) / tb), a.b.nseq, (heads + hb - 1) / hb);
  hipLaunchKernelGGL((k_rope<TYPE, HALF, WHOLE>), grid, dim3(256), (size_t)tb * a.half * sizeof(float2), st, a, tb, hb);
  ZL_HIP(hipGetLastError());
}

template <int TYPE>
static void launch_rope_t(const RopeArgs &a, hipStream_t st) {
  const bool whole = whole_pieces(a, value_size<TYPE>());
  if (a.neox) whole ? launch_rope_k<TYPE, true, true>(a, st) : launch_rope_k<TYPE, true, false>(a, st);
  else whole ? launch_rope_k<TYPE, false, true>(a, st) : launch_rope_k<TYPE, false, false>(a, st);
}
void launch_rope(const RopeArgs &a, int type, hipStream_t st) {
  if (type == T_F32) launch_rope_t<T_F32>(a, st);
  else if (type == T_F16) launch_rope_t<T_F16>(a, st);
  else launch_rope_t<T_BF16>(a, st);
}

}  // namespace zl
