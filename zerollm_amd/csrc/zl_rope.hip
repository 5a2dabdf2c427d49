// Rotary positions: queries and keys of a batch rotated in one launch.
#include "zl_ops.h"

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

// One block per (token, sequence): the pairs' cos and sin once, then every head.
template <int TYPE>
__global__ __launch_bounds__(256) void k_rope(const RopeArgs a) {
  typedef typename ValueOf<TYPE>::t T;
  __shared__ float cs[128], sn[128];
  const int t = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
  if (t >= (a.b.count ? max(0, min(a.b.count[s], a.b.ntok)) : a.b.ntok)) return;
  const double pos = (double)a.b.pos[s] + t;
  if (tid < a.half) {
    float c, n;
    turn_sincos(pos * a.turns[tid], &c, &n);
    cs[tid] = c * a.gain;
    sn[tid] = n * a.gain;
  }
  __syncthreads();
  const int nrot = 2 * a.half, items = a.half + (a.hd - nrot);  // pairs, then the values that pass through
  for (int i = tid; i < (a.nq + a.nk) * items; i += 256) {
    const int h = i / items, r = i - h * items;
    const bool isq = h < a.nq;
    const OpRows &x = isq ? a.q : a.k, &y = isq ? a.qo : a.ko;
    const int hh = isq ? h : h - a.nq;
    const T *xp = (const T *)x.p + s * x.seq + t * x.tok + hh * x.head;
    T *yp = (T *)y.p + s * y.seq + t * y.tok + hh * y.head;
    if (r >= a.half) {
      const int d = nrot + r - a.half;
      yp[d] = xp[d];
      continue;
    }
    const int i0 = a.neox ? r : 2 * r, i1 = a.neox ? r + a.half : 2 * r + 1;
    const float x0 = load_value<TYPE>(xp[i0]), x1 = load_value<TYPE>(xp[i1]), c = cs[r], n = sn[r];
    yp[i0] = store_value<TYPE>(fmaf(x0, c, -(x1 * n)));
    yp[i1] = store_value<TYPE>(fmaf(x0, n, x1 * c));
  }
}

void launch_rope(const RopeArgs &a, int type, hipStream_t st) {
  const dim3 grid(a.b.ntok, a.b.nseq);
  if (type == T_F32) hipLaunchKernelGGL((k_rope<T_F32>), grid, dim3(256), 0, st, a);
  else if (type == T_F16) hipLaunchKernelGGL((k_rope<T_F16>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_rope<T_BF16>), grid, dim3(256), 0, st, a);
  ZL_HIP(hipGetLastError());
}

}  // namespace zl
