// Sampling with temperature, top-k, top-p and min-p from one uniform number a row.
//
// Entries of a row in descending order of their logit (equal ones: the lower index first), w_v = exp((x_v - max x) / T):
//   n_k = top_k,  n_p = the shortest prefix with C(n) >= top_p C(n_k),  n_m = #{w >= min_p},  n = min(n_k, n_p, n_m) >= 1,
//   token = the first entry of that order with C(j) > u C(n),                C(j) = w_1 + .. + w_j.
// NaN counts as -inf, a row of nothing else gives token 0 with log-probability -inf. T <= 0: the first entry.
//
// A token lies next to a border of C now and then, so weights and their sums are in 64 bits: w by a polynomial of degree 10
// (relative error 2e-13), sums in double or, where they are collected by atomics, in units of 2^-45 (whole numbers: no order
// changes them).
//
// Two launches. The first reads the row once, many workgroups a row: largest entry of each 64 (group), and of each 2048 entries
// the sums of exp. The second, a workgroup a row, never sorts the row: each filter bounds the kept entries from below before any
// of them is known,
//   top-k  the k-th largest of the groups' largest entries (k groups have an entry as large)
//   top-p  w >= (1 - p) C(V) / V: entries below it hold less than 1 - p of the mass together
//   min-p  w >= min_p
// and only groups whose largest entry passes the bound are read again. Up to CAP entries are sorted in LDS; more of them (flat
// distributions) are counted into 2048 bins of the ordered 32-bit key, the bin in which a border falls into 2048 of its own,
// until a bin is one value (three times at most).
#include "common.h"
#include "sample.h"

constexpr int SF_GROUP = 64, SF_CHUNK = 2048, SF_MAX_V = 1 << 18, SF_CAP = 4096, SF_BINS = 2048;
constexpr int SF_MAX_GROUPS = SF_MAX_V / SF_GROUP, SF_MAX_CHUNKS = SF_MAX_V / SF_CHUNK;
constexpr double SF_UNIT = 35184372088832.0;  // 2^45: 2^18 weights of 1 fit 64 bits

struct ChunkSum { double zt, z1; float m; int pad; };

struct FilterArgs {
  double T, p, m;  // of all rows, unless the pointers give each its own
  const float *Ts, *ps, *ms;
  int k;
  const int* ks;
  const float* u;
  unsigned* gmax;  // [B][groups]
  ChunkSum* sums;  // [B][chunks]
  SampleArgs s;
};

struct RowOpts { double T, p, m; int k; };  // k 0, p 1, m 0: off

__device__ __forceinline__ RowOpts row_opts(const FilterArgs& a, int b) {
  RowOpts o{a.Ts ? (double)a.Ts[b] : a.T, a.ps ? (double)a.ps[b] : a.p, a.ms ? (double)a.ms[b] : a.m, a.ks ? a.ks[b] : a.k};
  if (!(o.T > 0)) o = {1.0, 1.0, 0.0, 1};  // greedy: the first entry
  if (o.k <= 0 || o.k >= a.s.V) o.k = 0;
  if (!(o.p < 1)) o.p = 1;
  if (!(o.m > 0)) o.m = 0;
  return o;
}

__device__ __forceinline__ float entry(float x) { return x != x ? -INFINITY : x; }
__device__ __forceinline__ unsigned key_of(float x) {  // ordered as the values are; -0 as +0
  const unsigned u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// e^a for a <= 0: 2^n by the exponent, e^r (|r| <= ln 2 / 2) by its series
__device__ __forceinline__ double exp_neg(double a) {
  const double n = rint(a * 1.4426950408889634);
  const double r = fma(n, -1.9082149292705877e-10, fma(n, -0.69314718036912382, a));
  double q = 1.0 / 3628800;
  q = fma(q, r, 1.0 / 362880);
  q = fma(q, r, 1.0 / 40320);
  q = fma(q, r, 1.0 / 5040);
  q = fma(q, r, 1.0 / 720);
  q = fma(q, r, 1.0 / 120);
  q = fma(q, r, 1.0 / 24);
  q = fma(q, r, 1.0 / 6);
  q = fma(q, r, 0.5);
  q = fma(q, r, 1.0);
  q = fma(q, r, 1.0);
  return a > -700 ? ldexp(q, (int)n) : 0.0;
}

__device__ __forceinline__ double weight(float x, float top, double inv_t) {
  return x == top ? 1.0 : exp_neg(((double)x - (double)top) * inv_t);
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ------------------------------------------------------------------------------------------- first launch
template <typename L>
__global__ void __launch_bounds__(256) filter_stats_kernel(FilterArgs a) {
  __shared__ float redf[16];
  __shared__ double redd[2][4];
  const int b = blockIdx.y, V = a.s.V, tid = threadIdx.x, v0 = blockIdx.x * SF_CHUNK + tid * 8;
  const L* row = (const L*)a.s.logits + (long)b * a.s.ld;
  const RowOpts o = row_opts(a, b);
  float x[8];
  if (v0 + 8 <= V && (((size_t)(row + v0)) & 15) == 0) {
    if constexpr (sizeof(L) == 2) {
      const u32x4_t u = *(const u32x4_t*)(row + v0);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(e & 1 ? u[e >> 1] & 0xffff0000u : u[e >> 1] << 16);
    } else {
      const f32x4_t lo = *(const f32x4_t*)(row + v0), hi = *(const f32x4_t*)(row + v0 + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = e < 4 ? lo[e & 3] : hi[e & 3];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = v0 + e < V ? logit_f(row[v0 + e]) : -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = entry(x[e]);
    mx = fmaxf(mx, x[e]);
  }
  float gm = mx;  // a group is 8 lanes
  gm = fmaxf(gm, __shfl_xor(gm, 1, 64));
  gm = fmaxf(gm, __shfl_xor(gm, 2, 64));
  gm = fmaxf(gm, __shfl_xor(gm, 4, 64));
  const int NG = (V + SF_GROUP - 1) / SF_GROUP;
  if ((tid & 7) == 0 && v0 < V) a.gmax[(long)b * NG + v0 / SF_GROUP] = key_of(gm);
  const float top = block_max(mx, redf), use = top == -INFINITY ? 0.f : top;
  double z1 = 0, zt = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    // exp in fp32 with the product's rounding error put back: 2 ulp for the log-probability's sum
    const float d = x[e] == use ? 0.f : x[e] - use, t = d * 1.44269504f, lo = fmaf(d, 1.44269504f, -t) + d * 1.92596299e-8f;
    const float q = __builtin_amdgcn_exp2f(t);
    z1 += t < -150.f ? 0.f : fmaf(q, lo * 0.693147181f, q);
  }
  if (o.p < 1 && o.k == 0) {
    const double it = 1.0 / o.T;
#pragma unroll
    for (int e = 0; e < 8; ++e) zt += x[e] == -INFINITY ? 0.0 : weight(x[e], use, it);
  }
  z1 = wave_sum_d(z1);
  zt = wave_sum_d(zt);
  if ((tid & 63) == 0) { redd[0][tid >> 6] = z1; redd[1][tid >> 6] = zt; }
  __syncthreads();
  if (tid == 0)
    a.sums[(long)b * gridDim.x + blockIdx.x] = {((redd[1][0] + redd[1][1]) + redd[1][2]) + redd[1][3],
                                                ((redd[0][0] + redd[0][1]) + redd[0][2]) + redd[0][3], top, 0};
}

// ------------------------------------------------------------------------------------------- second launch
typedef unsigned long long u64;

struct PickLds {
  u64 list[SF_CAP];  // (key, ~index) of the entries; counted ones: mass[SF_BINS], count[SF_BINS]
  union {
    double C[SF_CAP];  // of sorted entries
    struct {           // the groups that pass the bound, and (counted entries) each group's entries of one value
      unsigned short group[SF_MAX_GROUPS], match[SF_MAX_GROUPS];
    };
  };
  double redd[2][16];
  unsigned redu[3][16];
  u64 redm[16];
  unsigned kappa, n_group, n_list;
  unsigned bin, c_above, c_at, found;
  u64 m_above, m_at;
};

// The workgroup's inclusive sums over its threads, in order (16 waves)
__device__ __forceinline__ double scan_d(double v, double* red, double& before) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  double s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(s, o, 64);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 63) red[wv] = s;
  __syncthreads();
  double off = 0;
  for (int i = 0; i < wv; ++i) off += red[i];
  before = off + (s - v);
  return off + s;
}

template <typename T>
__device__ __forceinline__ T scan_u(T v, T* red) {  // exclusive
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  T s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T t = __shfl_up(s, o, 64);
    if (lane >= o) s += t;
  }
  __syncthreads();
  if (lane == 63) red[wv] = s;
  __syncthreads();
  T off = 0;
  for (int i = 0; i < wv; ++i) off += red[i];
  return off + s - v;
}

__device__ __forceinline__ unsigned block_sum_u(unsigned v, unsigned* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  unsigned t = 0;
  for (int i = 0; i < 16; ++i) t += red[i];
  return t;
}

// f(key, index) for the entries of the listed groups
template <typename L, typename F>
__device__ __forceinline__ void each_entry(const L* row, int V, const PickLds& S, F f) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, n = S.n_group;
  for (int g0 = wv * 4; g0 < n; g0 += 64) {
    float x[4];
    int v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = g0 + e < n ? S.group[g0 + e] * SF_GROUP + lane : V;
      x[e] = v[e] < V ? logit_f(row[v[e]]) : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) f(v[e] < V, key_of(entry(x[e])), v[e], e, g0 + e);
  }
}

// A border in the order of a row: the r first entries of value `key`, behind all larger ones (`above` of them, of mass `mass`)
struct Border { unsigned key, r, above; u64 mass; };

// The entries with lo <= key <= hi into bins, hi's first; then the first bin by which `count` entries (or more than / at least
// `mass`) are reached, and again within it until it is one key. Nothing reached: the end of the last bin.
enum { BY_COUNT, BY_MASS, OVER_MASS };
template <typename L>
__device__ Border find_border(const L* row, int V, PickLds& S, unsigned lo, unsigned hi, float top, double it, int by,
                              unsigned count, double mass) {
  u64* mbin = S.list;
  unsigned* cbin = (unsigned*)(S.list + SF_BINS);
  const int tid = threadIdx.x;
  unsigned above = 0;
  u64 m_above = 0;
  for (;;) {
    const unsigned range = hi - lo;
    const int shift = range < SF_BINS ? 0 : 21 - __builtin_clz(range);  // range >> shift < 2048
    __syncthreads();
    for (int i = tid; i < SF_BINS; i += 1024) { mbin[i] = 0; cbin[i] = 0; }
    __syncthreads();
    each_entry(row, V, S, [&](bool in, unsigned key, int, int, int) {
      if (!in || key < lo || key > hi) return;
      const unsigned bin = (hi - key) >> shift;
      atomicAdd(&cbin[bin], 1u);
      atomicAdd(&mbin[bin], (u64)rint(weight(of_key(key), top, it) * SF_UNIT));
    });
    __syncthreads();
    const unsigned c0 = cbin[2 * tid], c1 = cbin[2 * tid + 1];
    const u64 m0 = mbin[2 * tid], m1 = mbin[2 * tid + 1];
    const unsigned cb = above + scan_u<unsigned>(c0 + c1, S.redu[0]);
    const u64 mb = m_above + scan_u<u64>(m0 + m1, S.redm);
    if (tid == 0) S.found = 0;
    __syncthreads();
    auto reached = [&](unsigned c, u64 m) {
      return by == BY_COUNT ? c >= count : by == BY_MASS ? (double)m >= mass : (double)m > mass;
    };
    // bins that hold something, the last of them if nothing is reached
    if (c0 && !reached(cb, mb) && reached(cb + c0, mb + m0)) {
      S.bin = 2 * tid; S.c_above = cb; S.c_at = c0; S.m_above = mb; S.m_at = m0; S.found = 1;
    }
    if (c1 && !reached(cb + c0, mb + m0) && reached(cb + c0 + c1, mb + m0 + m1)) {
      S.bin = 2 * tid + 1; S.c_above = cb + c0; S.c_at = c1; S.m_above = mb + m0; S.m_at = m1; S.found = 1;
    }
    __syncthreads();
    if (!S.found) {
      const unsigned all = block_sum_u(c0 + c1, S.redu[1]) + above;
      if (c0 && cb + c0 == all) { S.bin = 2 * tid; S.c_above = cb; S.c_at = c0; S.m_above = mb; S.m_at = m0; }
      if (c1 && cb + c0 + c1 == all) { S.bin = 2 * tid + 1; S.c_above = cb + c0; S.c_at = c1; S.m_above = mb + m0; S.m_at = m1; }
      __syncthreads();
    }
    above = S.c_above;
    m_above = S.m_above;
    const unsigned bin = S.bin, at = S.c_at;
    const bool found = S.found;
    hi -= bin << shift;
    if (shift == 0) {
      const double w = rint(weight(of_key(hi), top, it) * SF_UNIT);
      double r = at;
      if (found && by == BY_COUNT) r = count - above;
      else if (found && w > 0) r = by == BY_MASS ? ceil((mass - (double)m_above) / w) : floor((mass - (double)m_above) / w) + 1;
      return {hi, (unsigned)fmin(fmax(r, 1.0), (double)at), above, m_above};
    }
    const unsigned low = hi - ((1u << shift) - 1);
    if (low > lo && low <= hi) lo = low;
  }
}

__device__ __forceinline__ double border_mass(const Border& b, float top, double it) {
  return (double)(b.mass + (u64)b.r * (u64)rint(weight(of_key(b.key), top, it) * SF_UNIT));
}

template <typename L>
__device__ int pick_counted(const L* row, int V, PickLds& S, const RowOpts& o, unsigned kappa, unsigned hi, float top, double it,
                            double zt, double u) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  unsigned lo = kappa, lo_m = 0;
  if (o.m > 0) {  // the smallest key of weight min_p or more
    unsigned a = 0, b = hi;
    while (a < b) {
      const unsigned mid = a + (b - a) / 2;
      if (weight(of_key(mid), top, it) >= o.m) b = mid;
      else a = mid + 1;
    }
    lo_m = a;
    if (!(o.k && o.p < 1)) lo = max(lo, lo_m);
  }
  Border end = find_border(row, V, S, lo, hi, top, it, BY_COUNT, o.k ? (unsigned)o.k : 0xffffffffu, 0.0);
  if (o.p < 1) {
    const double mass = o.k ? border_mass(end, top, it) : zt * SF_UNIT;
    const Border e = find_border(row, V, S, lo, hi, top, it, BY_MASS, 0, fmax(o.p * mass, 1.0));  // (the first entry at least)
    if (e.key > end.key || (e.key == end.key && e.r < end.r)) end = e;
  }
  if (lo_m > end.key) end = find_border(row, V, S, lo_m, hi, top, it, BY_COUNT, 0xffffffffu, 0.0);
  const Border at = find_border(row, V, S, lo, hi, top, it, OVER_MASS, 0, u * border_mass(end, top, it));
  unsigned key = at.key, r = at.r;
  if (key < end.key || (key == end.key && r > end.r)) key = end.key, r = end.r;
  // the r-th of the entries of that value, by index: each listed group's count, in the groups' order
  const int NG = (V + SF_GROUP - 1) / SF_GROUP;
  __syncthreads();
  for (int g = tid; g < SF_MAX_GROUPS; g += 1024) S.match[g] = 0;
  __syncthreads();
  each_entry(row, V, S, [&](bool in, unsigned k, int v, int, int) {
    const u64 hit = __ballot(in && k == key);
    if (hit && lane == 0) S.match[v / SF_GROUP] = (unsigned short)__popcll(hit);
  });
  __syncthreads();
  unsigned c[4], sum = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum += c[e] = 4 * tid + e < NG ? S.match[4 * tid + e] : 0;
  unsigned before = scan_u<unsigned>(sum, S.redu[0]);
  if (tid == 0) S.bin = 0, S.c_above = 0;
  __syncthreads();
  if (before < r && before + sum >= r) {
    int e = 0;
    while (before + c[e] < r) before += c[e++];
    S.bin = 4 * tid + e;
    S.c_above = r - before;  // of its matches
  }
  __syncthreads();
  if (wv == 0) {
    const int v = S.bin * SF_GROUP + lane;
    const u64 hit = __ballot(v < V && key_of(entry(logit_f(row[min(v, V - 1)]))) == key);
    const unsigned nth = __popcll(hit & ((2ull << lane) - 1));
    if ((hit >> lane & 1) && nth == S.c_above) S.bin = v;
  }
  __syncthreads();
  return S.bin;
}

__device__ int pick_sorted(PickLds& S, unsigned count, const RowOpts& o, float top, double it, double zt, double u) {
  const int tid = threadIdx.x;
  unsigned n2 = 64;
  while (n2 < count) n2 *= 2;
  for (unsigned i = count + tid; i < n2; i += 1024) S.list[i] = 0;
  // bitonic, descending; a key and its index are no other entry's
  for (unsigned size = 2; size <= n2; size *= 2)
    for (unsigned step = size / 2; step > 0; step /= 2) {
      __syncthreads();
      for (unsigned i = tid; i < n2 / 2; i += 1024) {
        const unsigned x = 2 * i - (i & (step - 1)), y = x + step;
        const u64 p = S.list[x], q = S.list[y];
        if ((p < q) == ((x & size) == 0)) { S.list[x] = q; S.list[y] = p; }
      }
    }
  __syncthreads();
  const unsigned each = n2 > 1024 ? n2 / 1024 : 1;
  double w[4], sum = 0, before;
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) {
    const unsigned i = tid * each + e;
    w[e] = e < each && i < count ? weight(of_key((unsigned)(S.list[i] >> 32)), top, it) : 0.0;
    sum += w[e];
  }
  scan_d(sum, S.redd[0], before);
  unsigned over = 0;
#pragma unroll
  for (unsigned e = 0; e < 4; ++e) {
    const unsigned i = tid * each + e;
    before += w[e];
    if (e < each && i < count) S.C[i] = before;
    over += e < each && i < count && w[e] >= o.m;
  }
  __syncthreads();
  unsigned n = min(o.k ? (unsigned)o.k : count, count);
  if (o.p < 1) {
    const double t = o.p * (o.k ? S.C[n - 1] : zt);
    unsigned c = 0;
    for (unsigned i = tid; i < count; i += 1024) c += S.C[i] < t;
    n = min(n, block_sum_u(c, S.redu[0]) + 1);
  }
  if (o.m > 0) n = min(n, max(1u, block_sum_u(over, S.redu[1])));
  const double t = u * S.C[n - 1];
  unsigned c = 0;
  for (unsigned i = tid; i < n; i += 1024) c += S.C[i] <= t;
  const unsigned at = min(block_sum_u(c, S.redu[2]), n - 1);
  return (int)~(unsigned)S.list[at];
}

template <typename L>
__global__ void __launch_bounds__(1024) filter_pick_kernel(FilterArgs a) {
  __shared__ __attribute__((aligned(16))) PickLds S;
  const int b = blockIdx.x, V = a.s.V, tid = threadIdx.x, lane = tid & 63;
  const int NG = (V + SF_GROUP - 1) / SF_GROUP, NC = (V + SF_CHUNK - 1) / SF_CHUNK;
  const L* row = (const L*)a.s.logits + (long)b * a.s.ld;
  const RowOpts o = row_opts(a, b);
  const double it = 1.0 / o.T;
  ChunkSum cs{0, 0, -INFINITY, 0};
  if (tid < NC) cs = a.sums[(long)b * NC + tid];
  unsigned gm[4];
  unsigned least = ~0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    gm[e] = tid + 1024 * e < NG ? a.gmax[(long)b * NG + tid + 1024 * e] : 0;
    if (tid + 1024 * e < NG) least = min(least, gm[e]);
  }
  const float top = block_max(cs.m, (float*)S.redu[0]);
  if (top == -INFINITY) {
    if (tid == 0) sample_bookkeep(a.s, b, 0, -INFINITY);
    return;
  }
  double z1 = cs.m == -INFINITY ? 0.0 : cs.z1 * (cs.m == top ? 1.0 : exp_neg((double)cs.m - (double)top)), zt = 0, skip;
  if (o.p < 1 && o.k == 0) zt = cs.m == -INFINITY ? 0.0 : cs.zt * weight(cs.m, top, it);
  z1 = wave_sum_d(z1);
  zt = wave_sum_d(zt);
  if (lane == 0) { S.redd[0][tid >> 6] = z1; S.redd[1][tid >> 6] = zt; }
  if (tid == 0) S.kappa = 0, S.n_group = 0, S.n_list = 0;
  __syncthreads();
  z1 = S.redd[0][0] + S.redd[0][1];  // (up to 128 chunks: two waves)
  zt = S.redd[1][0] + S.redd[1][1];
  const unsigned hi = key_of(top);
  // ---- the bound ----
  unsigned kappa = 0;
  if (o.k && o.k <= NG) {
    // the k-th largest group's bin of 1024 between the smallest and the largest
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) least = min(least, (unsigned)__shfl_xor((int)least, x, 64));
    unsigned* cbin = (unsigned*)S.list;
    cbin[tid] = 0;
    if (lane == 0) S.redu[1][tid >> 6] = least;
    __syncthreads();
    for (int i = 0; i < 16; ++i) least = min(least, S.redu[1][i]);
    const unsigned range = hi - least;
    const int shift = range < 1024 ? 0 : 22 - __builtin_clz(range);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (tid + 1024 * e < NG) atomicAdd(&cbin[(hi - gm[e]) >> shift], 1u);
    __syncthreads();
    const unsigned mine = cbin[tid], before = scan_u<unsigned>(mine, S.redu[0]);
    if (before < (unsigned)o.k && before + mine >= (unsigned)o.k) {
      const unsigned up = ((unsigned)tid << shift) + ((1u << shift) - 1);
      S.kappa = up >= hi ? 0 : hi - up;
    }
    __syncthreads();
    kappa = S.kappa;
  }
  if (!(o.k && o.p < 1)) {  // (with both, the mass of the top k is needed)
    double least_w = o.m;
    if (o.p < 1) least_w = fmax(least_w, (1.0 - o.p) * zt / V);
    if (least_w > 0) {
      const double below = o.T * log(least_w), x = (double)top + fmin(below, 0.0);
      const float f = (float)(x - 1e-6 * (fabs((double)top) + fabs(below)));  // (safely below what rounding could do)
      if (f == f) kappa = max(kappa, key_of(f));
    }
    kappa = min(kappa, hi);
  }
  __syncthreads();
  // ---- the groups that pass it, in any order, and their entries ----
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (tid + 1024 * e < NG && gm[e] >= kappa) S.group[atomicAdd(&S.n_group, 1u)] = (unsigned short)(tid + 1024 * e);
  __syncthreads();
  each_entry(row, V, S, [&](bool in, unsigned key, int v, int, int) {
    const bool hit = in && key >= kappa;
    const u64 all = __ballot(hit);
    if (!all) return;
    unsigned at = 0;
    if (lane == 0) at = atomicAdd(&S.n_list, (unsigned)__popcll(all));
    at = __builtin_amdgcn_readfirstlane(at) + __popcll(all & ((1ull << lane) - 1));
    if (hit && at < SF_CAP) S.list[at] = ((u64)key << 32) | (unsigned)~v;
  });
  __syncthreads();
  const unsigned count = S.n_list;
  double u;
  if (a.u) u = a.u[b];
  else u = u01(a.s.seed, (a.s.ctr ? (unsigned)a.s.ctr[b] : a.s.step) * 131071u + (unsigned)b, 0u);
  u = fmin(fmax(u, 0.0), 1.0);
  const int tok = count <= SF_CAP ? pick_sorted(S, count, o, top, it, zt, u)
                                  : pick_counted(row, V, S, o, kappa, hi, top, it, zt, u);
  if (tid == 0) {
    const float x = entry(logit_f(row[tok]));
    const double d = x == top ? 0.0 : (double)x - (double)top;
    sample_bookkeep(a.s, b, tok, (float)(d - log1p(z1 - 1.0)));
  }
}

DA_EXPORT size_t da_sample_filtered_ws(int B, int V) {
  const size_t NG = (V + SF_GROUP - 1) / SF_GROUP, NC = (V + SF_CHUNK - 1) / SF_CHUNK;
  return B * (NC * sizeof(ChunkSum) + NG * 4);
}

DA_EXPORT int da_sample_filtered(const void* logits, int f32, int B, int V, int ld, double T, double p, double m, int k,
                                 const void* Ts, const void* ps, const void* ms, const void* ks, const void* u, unsigned seed,
                                 unsigned step, const void* ctr, void* ws, void* out_tok, void* out_lp, void* conf, void* active,
                                 void* pos, void* lens, void* hist, const void* start, int hist_ld, int eos0, int eos1, int eos2,
                                 int eos3, void* stream) {
  if (V < 1 || V > SF_MAX_V || B > 65535 || (hist && (!pos || !start))) return (int)hipErrorInvalidValue;
  if (B == 0) return 0;
  const int NC = (V + SF_CHUNK - 1) / SF_CHUNK;
  SampleArgs s{logits, V, ld, 0.f, seed, step, (const int*)ctr, (int*)out_tok, (float*)out_lp, (float*)conf, (int*)active,
               (int*)pos, (int*)lens, (int*)hist, (const int*)start, hist_ld, eos0, eos1, eos2, eos3};
  FilterArgs a{T, p, m, (const float*)Ts, (const float*)ps, (const float*)ms, k, (const int*)ks, (const float*)u,
               (unsigned*)((char*)ws + (size_t)B * NC * sizeof(ChunkSum)), (ChunkSum*)ws, s};
  hipStream_t st = (hipStream_t)stream;
  if (f32) filter_stats_kernel<float><<<dim3(NC, B), 256, 0, st>>>(a);
  else filter_stats_kernel<bf16_t><<<dim3(NC, B), 256, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (f32) filter_pick_kernel<float><<<B, 1024, 0, st>>>(a);
  else filter_pick_kernel<bf16_t><<<B, 1024, 0, st>>>(a);
  DA_LAUNCH_CHECK();
}
