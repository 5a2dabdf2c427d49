// Log probabilities of logits rows.
#include "zl_ops.h"

namespace zl {

// Order of the alternatives: larger value first, lower id first among equals, NaN below all, as one number.
__device__ __forceinline__ unsigned long long rank_key(float x, int id) {
  return ((unsigned long long)(x != x ? 0u : fkey(x)) << 32) | (uint32_t)~id;
}

// One block per row, a pass over the row for the maximum, one for the sums and one for each alternative.
template <int TYPE>
__global__ __launch_bounds__(256) void k_logprobs(const LogprobArgs a) {
  typedef typename ValueOf<TYPE>::t T;
  __shared__ float redf[4];
  __shared__ double redd[8];
  __shared__ unsigned long long redk[4];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T *x = (const T *)a.x + (long)r * a.ld;
  float m = -INFINITY;
  bool nan = false;
  for (int i = tid; i < a.vocab; i += 256) { const float v = load_value<TYPE>(x[i]); m = fmaxf(m, v); nan |= v != v; }
  if (nan) m = NAN;
  m = group_reduce(m, 64, [](float p, float q) { return p != p || q != q ? NAN : fmaxf(p, q); });
  if (lane == 0) redf[wave] = m;
  __syncthreads();
  m = redf[0];
  for (int w = 1; w < 4; w++) m = m != m || redf[w] != redf[w] ? NAN : fmaxf(m, redf[w]);
  double l = 0, e = 0;
  for (int i = tid; i < a.vocab; i += 256) {
    const double d = (double)load_value<TYPE>(x[i]) - (double)m;
    if (d == -INFINITY) continue;
    const double p = exp(d);
    l += p;
    e += p * d;
  }
  l = wave_sum_xor(l, 64);
  e = wave_sum_xor(e, 64);
  if (lane == 0) { redd[wave] = l; redd[4 + wave] = e; }
  __syncthreads();
  l = (redd[0] + redd[1]) + (redd[2] + redd[3]);
  e = (redd[4] + redd[5]) + (redd[6] + redd[7]);
  const double lz = m > -INFINITY ? log(l) : NAN;
  if (tid == 0) {
    if (a.lp) {
      const int id = a.tokens[r];
      a.lp[r] = id >= 0 && id < a.vocab ? (float)((double)load_value<TYPE>(x[id]) - (double)m - lz) : NAN;
    }
    if (a.ent) a.ent[r] = (float)(lz - e / l);
  }
  unsigned long long prev = ~0ull;
  for (int k = 0; k < a.ntop; k++) {
    unsigned long long best = 0;
    for (int i = tid; i < a.vocab; i += 256) {
      const unsigned long long c = rank_key(load_value<TYPE>(x[i]), i);
      if (c < prev && c > best) best = c;
    }
    best = group_reduce(best, 64, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
    __syncthreads();
    if (lane == 0) redk[wave] = best;
    __syncthreads();
    for (int w = 0; w < 4; w++) best = redk[w] > best ? redk[w] : best;
    prev = best;
    if (tid == 0) {
      const int id = (int)~(uint32_t)best;
      if (a.ids) a.ids[(long)r * a.ntop + k] = id;
      if (a.toplp) a.toplp[(long)r * a.ntop + k] = (float)((double)load_value<TYPE>(x[id]) - (double)m - lz);
    }
  }
}

long logprobs_work(int rows, int vocab, int ntop) { return 16; }

void launch_logprobs(const LogprobArgs &a, int type, hipStream_t st) {
  if (type == T_F32) hipLaunchKernelGGL((k_logprobs<T_F32>), dim3(a.rows), dim3(256), 0, st, a);
  else if (type == T_F16) hipLaunchKernelGGL((k_logprobs<T_F16>), dim3(a.rows), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_logprobs<T_BF16>), dim3(a.rows), dim3(256), 0, st, a);
  ZL_HIP(hipGetLastError());
}

}  // namespace zl
