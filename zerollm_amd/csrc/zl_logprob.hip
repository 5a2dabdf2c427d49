// Log probabilities of logits rows: the log-sum-exp, the entropy and the top alternatives in one pass over the logits.
//
// With m the largest logit seen so far, l = sum e^(x - m) and e = sum e^(x - m) (x - m): a larger m' scales l by f = e^(m - m')
// and takes e to f (e + l (m - m')). Then lse = m + ln l and the entropy is ln l - e / l: differences from the maximum all
// along, so that nothing cancels. -inf counts for nothing; NaN and +inf make l NaN, and with it every float output.
//
// Alternatives are 64-bit numbers, the ordered value above the complement of the id, so that a larger one is a better one
// and equal values go to the lowest id. The pass keeps each lane's largest logit; at least n_top logits are at or above the
// n_top-th largest of a block's. The lanes whose largest reaches that threshold, n_top of 256 but for ties, have their pieces read
// again (from the caches), and what reaches it is listed in LDS. Full lists are cut to their n_top best (a search for the
// n_top-th largest number, bit by bit with ballots). (Lists filled during the pass, under a threshold of what came before: 2048 x
// 32000 bf16, 5 alternatives, 46 us.)
//
// Bound by HBM (each logit is read once) for many rows, by the latency of two launches for few.
#include "zl_ops.h"
#include <algorithm>

namespace zl {

typedef unsigned long long rank_t;
__device__ __forceinline__ rank_t rank_key(float x, int id) {
  return ((rank_t)(x != x ? 0u : fkey(x)) << 32) | (uint32_t)~id;
}
__device__ __forceinline__ float rank_value(rank_t k) { return keyf((uint32_t)(k >> 32)); }

struct RowSum {
  float m = -INFINITY, l = 0.0f, e = 0.0f;
  __device__ __forceinline__ void raise(float to) {  // to >= m, above -inf
    if (m == -INFINITY) { m = to; return; }
    const float d = m - to, f = __builtin_amdgcn_exp2f(d * 1.44269504f);
    e = f == 0.0f ? 0.0f : f * fmaf(l, d, e);  // (f is 0 from d = -104 on, where l d may be infinite: masks of -1e38, a type's lowest value)
    l *= f;
    m = to;
  }
  __device__ __forceinline__ void add(const RowSum &o) {
    RowSum p = o;
    const float M = fmaxf(m, p.m);
    if (M > -INFINITY) {
      raise(M);
      p.raise(M);
    }
    l += p.l;
    e += p.e;
  }
  __device__ __forceinline__ void join_wave() {
    const float M = group_fmax(m, 64);
    if (M > -INFINITY) raise(M);
    l = wave_sum_xor(l, 64);
    e = wave_sum_xor(e, 64);
  }
};

constexpr int LP_CAP = 256;      // candidates of a wave
constexpr int LP_TILE = 4096;    // logits of a block at a time: 16 per lane

// A wave's candidate list: n entries in LDS, the threshold t (an entry must be larger), k wanted.
struct Candidates {
  rank_t *buf;
  int n, k;
  rank_t t;
  // Cut to the k largest (n > k). Entries are distinct, none is 0.
  template <int N>
  __device__ __forceinline__ void cut_n(int lane) {
    rank_t x[N];
    #pragma unroll
    for (int i = 0; i < N; i++) x[i] = lane + 64 * i < n ? buf[lane + 64 * i] : 0;
    rank_t v = 0;
    for (int bit = 63; bit >= 0; bit--) {
      const rank_t c = v | (1ull << bit);
      int cnt = 0;
      #pragma unroll
      for (int i = 0; i < N; i++) cnt += __popcll(__ballot(x[i] >= c));
      if (cnt >= k) v = c;
      if (cnt == k) break;
    }
    int at = 0;
    rank_t mn = ~0ull;  // the k-th largest itself: the smallest that is kept
    #pragma unroll
    for (int i = 0; i < N; i++) {
      const bool keep = x[i] >= v && x[i] != 0;
      const unsigned long long b = __ballot(keep);
      if (keep) buf[at + __popcll(b & ((1ull << lane) - 1))] = x[i];
      if (keep && x[i] < mn) mn = x[i];
      at += __popcll(b);
    }
    n = at;
    t = group_reduce(mn, 64, [](rank_t a, rank_t b) { return a < b ? a : b; });
  }
  __device__ __forceinline__ void cut(int lane) {
    if (n <= 64) cut_n<1>(lane);
    else cut_n<LP_CAP / 64>(lane);
  }
  __device__ __forceinline__ void offer(bool have, rank_t x, int lane) {  // by all lanes of the wave
    const bool take = have && x > t;
    const unsigned long long b = __ballot(take);
    if (!b) return;
    if (take) buf[n + __popcll(b & ((1ull << lane) - 1))] = x;
    n += __popcll(b);
    if (n > LP_CAP - 64) cut(lane);
  }
};

// The k-th largest of the block's 256 numbers, in all lanes; keys: 1 KB of LDS, free again afterwards.
__device__ __forceinline__ uint32_t block_threshold(uint32_t key, int k, uint32_t *keys, int lane, int wave) {
  keys[64 * wave + lane] = key;
  __syncthreads();
  uint32_t x[4], v = 0;
  if (wave == 0) {
    #pragma unroll
    for (int i = 0; i < 4; i++) x[i] = keys[lane + 64 * i];
    for (int bit = 31; bit >= 0; bit--) {
      int cnt = 0;
      #pragma unroll
      for (int i = 0; i < 4; i++) cnt += __popcll(__ballot(x[i] >= (v | (1u << bit))));
      if (cnt >= k) v |= 1u << bit;
      if (cnt == k) break;
    }
  }
  __syncthreads();
  if (wave == 0 && lane == 0) keys[0] = v;
  __syncthreads();
  v = keys[0];
  __syncthreads();
  return v;
}

// The k best of the four waves' lists, in wave 0's list, by the whole block.
__device__ __forceinline__ void merge_waves(Candidates &c, rank_t (*lists)[LP_CAP], int *counts, int lane, int wave) {
  if (c.n > 64) c.cut(lane);  // (to fit one offer)
  if (lane == 0) counts[wave] = c.n;
  __syncthreads();
  if (wave == 0) {
    for (int w = 1; w < 4; w++) c.offer(lane < counts[w], lists[w][min(lane, LP_CAP - 1)], lane);
    if (c.n > c.k) c.cut(lane);
  }
}

// Outputs of a row, by one wave: its sums and its k best.
template <int TYPE>
__device__ __forceinline__ void finish_row(const LogprobArgs &a, int row, const RowSum &s, rank_t mine, int lane) {
  typedef typename ValueOf<TYPE>::t T;
  const T *x = (const T *)a.x + (long)row * a.ld;
  const double lz = s.m > -INFINITY ? log((double)s.l) : NAN;
  if (lane == 0) {
    if (a.lp) {
      const int id = a.tokens[row];
      a.lp[row] = id >= 0 && id < a.vocab ? (float)((double)load_value<TYPE>(x[id]) - (double)s.m - lz) : NAN;
    }
    if (a.ent) a.ent[row] = (float)(lz - (double)s.e / (double)s.l);
  }
  if (a.ntop == 0) return;
  int place = 0;
  for (int j = 0; j < a.ntop; j++) place += __shfl(mine, j, 64) > mine;
  if (lane < a.ntop) {
    const int id = (int)~(uint32_t)mine;
    if (a.ids) a.ids[(long)row * a.ntop + place] = id;
    if (a.toplp) a.toplp[(long)row * a.ntop + place] = (float)((double)rank_value(mine) - (double)s.m - lz);
  }
}

// Work space: the parts' sums [row][part], then their candidates [row][part][ntop].
__device__ __forceinline__ float4 *part_sum(const LogprobArgs &a, int parts, long row) { return (float4 *)a.work + row * parts; }
__device__ __forceinline__ rank_t *part_top(const LogprobArgs &a, int parts, long row) {
  return (rank_t *)((float4 *)a.work + (long)a.rows * parts) + row * parts * a.ntop;
}

template <int TYPE>
__global__ __launch_bounds__(256) void k_logprobs(const LogprobArgs a, int parts, int span) {
  typedef typename ValueOf<TYPE>::t T;
  constexpr int VE = 16 / sizeof(T), NV = 16 / VE;  // values per 16-byte load, loads per lane
  typedef T vec __attribute__((ext_vector_type(VE)));
  __shared__ rank_t lists[4][LP_CAP];
  __shared__ float sums[4][3];
  __shared__ int counts[4];
  const int row = blockIdx.x / parts, part = blockIdx.x - row * parts, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T *x = (const T *)a.x + (long)row * a.ld;
  const int off = (int)(((uintptr_t)x % 16) / sizeof(T));  // indexes count from the 16-byte boundary at or before the row
  const T *base = x - off;
  const int i0 = part * span, i1 = min(a.vocab + off, i0 + span);
  RowSum s;
  Candidates c{lists[wave], 0, a.ntop, 0};
  float lm = -INFINITY;  // the lane's largest logit
  for (int t0 = i0; t0 < i1; t0 += LP_TILE) {
    float v[16];
    #pragma unroll
    for (int j = 0; j < NV; j++) {
      const int i = t0 + (j * 256 + tid) * VE;
      if (i >= off && i + VE <= a.vocab + off && i + VE <= i1) {
        const vec u = *(const vec *)(base + i);
        #pragma unroll
        for (int e = 0; e < VE; e++) v[j * VE + e] = load_value<TYPE>(u[e]);
      } else {
        #pragma unroll
        for (int e = 0; e < VE; e++) v[j * VE + e] = i + e >= off && i + e < i1 ? load_value<TYPE>(base[i + e]) : -INFINITY;
      }
    }
    float mx = v[0];
    #pragma unroll
    for (int e = 1; e < 16; e++) mx = fmaxf(mx, v[e]);
    if (mx > s.m) s.raise(mx);
    const float ref = s.m == -INFINITY ? 0.0f : s.m;
    #pragma unroll
    for (int e = 0; e < 16; e++) {
      const float d = v[e] - ref, p = __builtin_amdgcn_exp2f(d * 1.44269504f);
      s.l += p;
      s.e = fmaf(p, fmaxf(d, -3.0e38f), s.e);
    }
    lm = fmaxf(lm, mx);
  }
  if (a.ntop) {
    // no threshold where it is -inf: such lanes may hold nothing
    const uint32_t none = fkey(-INFINITY), kth = block_threshold(fkey(lm), a.ntop, (uint32_t *)lists[3], lane, wave);
    c.t = kth > none ? ((rank_t)kth << 32) - 1 : 0;
    // the lanes that have something at it: their pieces of every tile, a piece per lane
    const bool in = !c.t || lm >= keyf(kth);
    const unsigned long long who = __ballot(in);
    const int rank = __popcll(who & ((1ull << lane) - 1)), held = __popcll(who);
    const int list = __builtin_amdgcn_ds_permute(4 * (in ? rank : held + lane - rank), lane);  // the lanes in order, those first
    const int tiles = (i1 - i0 + LP_TILE - 1) / LP_TILE;
    for (int p0 = 0; p0 < held * tiles; p0 += 64) {
      const int p = p0 + lane, t0 = i0 + p % tiles * LP_TILE, from = wave * 64 + __shfl(list, min(p / tiles, 63), 64);
      const int end = p < held * tiles ? i1 : 0;
      // what is at the least number above the threshold, which cuts raise: its value or more, among its equals its id or before
      const rank_t least = c.t + 1;
      const uint32_t tv = (uint32_t)(least >> 32), ti = ~(uint32_t)least;
      const float tf = tv ? keyf(tv) : NAN;  // (NaN: everything)
      auto may = [&](float v, int i) { return !(v < tf) && !(v == tf && (uint32_t)(i - off) > ti); };
      uint32_t mask = 0;
      #pragma unroll
      for (int j = 0; j < NV; j++) {
        const int i = t0 + (j * 256 + from) * VE;
        if (i >= off && i + VE <= end) {
          const vec u = *(const vec *)(base + i);
          #pragma unroll
          for (int e = 0; e < VE; e++) mask |= may(load_value<TYPE>(u[e]), i + e) ? 1u << (j * VE + e) : 0u;
        } else {
          #pragma unroll
          for (int e = 0; e < VE; e++) mask |= i + e >= off && i + e < end && may(load_value<TYPE>(base[i + e]), i + e) ? 1u << (j * VE + e) : 0u;
        }
      }
      while (__ballot(mask != 0)) {
        const int e = __ffs((int)mask) - 1, i = t0 + ((e / VE) * 256 + from) * VE + e % VE;
        c.offer(mask != 0, mask ? rank_key(load_value<TYPE>(base[i]), i - off) : 0, lane);
        mask &= mask - 1;
      }
    }
  }
  s.join_wave();
  if (lane == 0) { sums[wave][0] = s.m; sums[wave][1] = s.l; sums[wave][2] = s.e; }
  if (a.ntop) merge_waves(c, lists, counts, lane, wave);
  else __syncthreads();
  if (wave) return;
  for (int w = 1; w < 4; w++) {
    RowSum o;
    o.m = sums[w][0];
    o.l = sums[w][1];
    o.e = sums[w][2];
    s.add(o);
  }
  const rank_t mine = lane < c.n ? lists[0][lane] : 0;
  if (parts == 1) {
    finish_row<TYPE>(a, row, s, mine, lane);
    return;
  }
  if (lane == 0) part_sum(a, parts, row)[part] = make_float4(s.m, s.l, s.e, 0.0f);
  if (lane < a.ntop) part_top(a, parts, row)[part * a.ntop + lane] = mine;
}

// The parts of a row.
template <int TYPE>
__global__ __launch_bounds__(256) void k_logprobs_join(const LogprobArgs a, int parts) {
  __shared__ rank_t lists[4][LP_CAP];
  __shared__ int counts[4];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Candidates c{lists[wave], 0, a.ntop, 0};
  if (a.ntop) {
    const rank_t *top = part_top(a, parts, row);
    const int total = parts * a.ntop;
    rank_t best = 0;
    for (int i = tid; i < total; i += 256) best = max(best, top[i]);
    const uint32_t kth = block_threshold((uint32_t)(best >> 32), a.ntop, (uint32_t *)lists[3], lane, wave);
    c.t = kth ? ((rank_t)kth << 32) - 1 : 0;
    for (int i0 = 0; i0 < total; i0 += 1024) {
      rank_t x[4];
      #pragma unroll
      for (int j = 0; j < 4; j++) x[j] = i0 + 256 * j + tid < total ? top[i0 + 256 * j + tid] : 0;
      #pragma unroll
      for (int j = 0; j < 4; j++) c.offer(x[j] != 0, x[j], lane);
    }
    merge_waves(c, lists, counts, lane, wave);
  }
  if (wave) return;
  RowSum s;
  for (int p = lane; p < parts; p += 64) {
    const float4 v = part_sum(a, parts, row)[p];
    RowSum o;
    o.m = v.x;
    o.l = v.y;
    o.e = v.z;
    s.add(o);
  }
  s.join_wave();
  finish_row<TYPE>(a, row, s, lane < c.n ? lists[0][lane] : 0, lane);
}

// Parts of a row: blocks of whole tiles, about a thousand blocks in all where the rows alone are fewer (four of a CU's size, to
// have loads of many waves in flight), one block per row beyond.
static int lp_span(int rows, int vocab) {
  const long tiles = (vocab + 7 + LP_TILE - 1) / LP_TILE;  // (a row may start up to 7 values behind a 16-byte boundary)
  return (int)std::max(1L, std::min(tiles, (tiles * rows + 512) / 1024)) * LP_TILE;
}
static int lp_parts(int rows, int vocab) { return (vocab + 7 + lp_span(rows, vocab) - 1) / lp_span(rows, vocab); }

long logprobs_work(int rows, int vocab, int ntop) {
  const long parts = lp_parts(std::max(rows, 1), vocab);
  return std::max(16L, parts == 1 ? 0L : rows * parts * (16 + 8L * ntop));
}

template <int TYPE>
static void launch_logprobs_t(const LogprobArgs &a, hipStream_t st) {
  const int span = lp_span(a.rows, a.vocab), parts = lp_parts(a.rows, a.vocab);
  hipLaunchKernelGGL((k_logprobs<TYPE>), dim3((unsigned)((long)a.rows * parts)), dim3(256), 0, st, a, parts, span);
  ZL_HIP(hipGetLastError());
  if (parts > 1) {
    hipLaunchKernelGGL((k_logprobs_join<TYPE>), dim3(a.rows), dim3(256), 0, st, a, parts);
    ZL_HIP(hipGetLastError());
  }
}
void launch_logprobs(const LogprobArgs &a, int type, hipStream_t st) {
  if (type == T_F32) launch_logprobs_t<T_F32>(a, st);
  else if (type == T_F16) launch_logprobs_t<T_F16>(a, st);
  else launch_logprobs_t<T_BF16>(a, st);
}

}  // namespace zl
