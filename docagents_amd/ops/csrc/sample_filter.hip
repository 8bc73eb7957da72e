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
// Two launches, or one where a row has few workgroups. The first reads the row once, a wave to 512 entries: the largest entry of each
// 64 (group) and the sums of exp.
// The second, a workgroup a row, reads again only what can be kept. Each filter bounds the kept entries from below before any of them
// is known,
//   top-k  the k-th largest of the groups' largest entries (k groups have an entry as large)
//   top-p  w >= (1 - p) C(V) / V: entries below it hold less than 1 - p of the mass together
//   min-p  w >= min_p
//   all    w >= e^-44
// and only groups whose largest entry passes the bound are read again. Up to CAP entries are sorted in LDS. Of more of them, where
// top-k keeps fewer, those down to the bin of the k-th of 2048 bins of equal width are. More still (flat distributions) are counted
// into such bins with their weights; a border (of top-k, top-p or u) falls into one bin, and that bin's entries are sorted. If even
// those are too many (thousands of equal logits), the ordered 32-bit key is split by 11 bits a time.
//
// What the sums are off by, in weights of the largest entry: sorted rows V e^-44 (2e-14 at 2^18 entries) and the roundings of their
// sums; counted ones V (2^-46 + e^-32), 7e-9 at 2^18 entries and 1e-9 at 50257: each weight is rounded to a unit, and entries 32 T below
// the top are left out. A token is the definition's unless it lies that near to a border.
//
// Measured: one row of 32064 11 us in one launch (3.9 + 5.7 in two), 64 of 128256 (bf16, 16 MB) 8.0 + 9.9 (the read at 2.0 TB/s, its
// start and end in it), 128 of them in fp32 with settings of their own (66 MB) 18.5 + 12 (3.6 TB/s), latencies of launches and of some ten steps that wait
// for one another; 33 flat rows of 50257 6 + 52: 16 us weigh 40000 entries or so on one CU (vector instructions), 10 a border (search,
// read, sort). Several workgroups a row for that took a quarter of its time and twice as much again for handing over.
#include "common.h"
#include "sample.h"

constexpr int SF_GROUP = 64, SF_CHUNK = 512, SF_MAX_V = 1 << 18, SF_CAP = 2048, SF_BINS = 2048;
// Both in one launch: rows that one workgroup takes (16 chunks), a CU each, and up to 64 workgroups of longer ones, whose last goes on
// to the pick. us of calls one by one / in a graph, two launches and one: 1 - 256 rows of 8000 13.1 / 10.0 - 11.4 and 10.7 / 9.2 - 10.4 (320
// 18.3 / 18.1, 18.7 / 18.7); one row of 32064 13.1 / 10.3 and 11.5 / 10.8, 16 of them 13.6 / 10.4 and 11.9 / 11.1 (64: 13.6 / 11.2, 12.0 /
// 11.9), 4 of 128256 13.6 / 10.8 and 11.8 / 11.5 (32: 13.4 / 12.6, 21.5 / 20.7)
constexpr int SF_WG = 16, SF_JOINED_ROWS = 256, SF_JOINED = 64;
// Waves that sort 64 entries each by counting, the others having ended; above them a workgroup sorts through bins. 32 rows, the whole
// call in us: 65 entries 13.1 with one wave / 12.1 with two, 128 13.6 / 13.3, 192 14.7 / 14.5 / 14.7 with four, 256 14.4 / 15.8
constexpr int SF_FEW = 2;
// Entries of a bin that are counted against one another; in larger ones all are exchanged in pairs (2000 entries, each value 32 times
// 22 us / 33, 100 times 25 / 33, 200 times 35 / 33)
constexpr unsigned SF_CROWD = 128;
constexpr int SF_MAX_GROUPS = SF_MAX_V / SF_GROUP;
static_assert(SF_MAX_V / SF_CHUNK <= 1024 && SF_MAX_GROUPS <= 4096 && SF_CAP <= 2048, "the second launch's 1024 threads");
typedef unsigned long long u64;
constexpr double SF_UNIT = 35184372088832.0;  // 2^45: 2^18 weights of 1 fit 64 bits

struct ChunkSum { double zt; float rest, m; int n, pad; };  // sums relative to the chunk's largest entry m: n of it, the others' exp

struct FilterArgs {
  double T, p, m;  // of all rows, unless the pointers give each its own
  const float *Ts, *ps, *ms;
  int k;
  const int* ks;
  const float* u;
  unsigned* gmax;  // [B][groups]
  ChunkSum* sums;  // [B][chunks]
  int* tickets;    // [B], 0 between launches: of rows of several workgroups in one launch
  SampleArgs s;
};

struct RowOpts { double T, p, m; int k; };  // k 0, p 1, m 0: off

__device__ __forceinline__ RowOpts row_opts(const FilterArgs& a, int b) {
  RowOpts o{a.Ts ? (double)a.Ts[b] : a.T, a.ps ? (double)a.ps[b] : a.p, a.ms ? (double)a.ms[b] : a.m, a.ks ? a.ks[b] : a.k};
  if (!(o.T > 0) || o.m > 1) o = {1.0, 1.0, 0.0, 1};  // the first entry: greedy, or no weight passes min-p (which bins could not hold)
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
// (a range's last key as a value: -0's, which no entry has, would be +0)
__device__ __forceinline__ float of_key(unsigned k);
__device__ __forceinline__ float of_last(unsigned k) { return of_key(k - (k == 0x7fffffffu)); }
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// e^a for a <= 0: a = n ln 2 + r with ln 2 in two parts (Cody and Waite's reduction), 2^n by the exponent, e^r (|r| <= ln 2 / 2) by its series
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

// A wave's smallest value, in lane 63 (complements: lanes that are moved from nowhere hold 0)
__device__ __forceinline__ unsigned wave_min(unsigned s) {
  s = ~s;
  s = max(s, moved<0x111, 0xf>(s));
  s = max(s, moved<0x112, 0xf>(s));
  s = max(s, moved<0x114, 0xf>(s));
  s = max(s, moved<0x118, 0xf>(s));
  s = max(s, moved<0x142, 0xa>(s));
  return ~max(s, moved<0x143, 0xc>(s));
}

// A wave's reductions on the vector ALU: neighbours, pairs, halves of 8 and of 16 lanes (mirrored), then rows of lanes
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float max8(float v) {
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  return fmaxf(v, dpp<0x141>(v));
}
__device__ __forceinline__ float max_8_64(float v) {  // of max8
  v = fmaxf(v, dpp<0x140>(v));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_xhalf(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum64(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  v += dpp<0x140>(v);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return sum_xhalf(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Groups and chunks begin at 16 bytes whatever the row does: group g is the entries 64 g - lead .. 64 g - lead + 63 that the row has
template <typename L>
__device__ __forceinline__ int lead_of(const L* row, int V) {
  const int lead = (int)(((size_t)row & 15) / sizeof(L));
  return V + lead <= SF_MAX_V ? lead : 0;
}
__host__ __device__ constexpr int groups_of(int V) { return (V + SF_GROUP - 1) / SF_GROUP; }
__host__ __device__ constexpr int chunks_of(int V) { return (V + SF_CHUNK - 1) / SF_CHUNK; }
constexpr int SF_LEAD = 7;  // at most

// What is handed over within a launch passes the L2s of the XCDs (agent scope)
template <bool JOINED, typename T>
__device__ __forceinline__ void put(T* p, T v) {
  if constexpr (JOINED) __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else *p = v;
}
template <bool JOINED, typename T>
__device__ __forceinline__ T get(const T* p) {
  if constexpr (JOINED) return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else return *p;
}

// ------------------------------------------------------------------------------------------- statistics
// A wave's 512 entries of row b
template <typename L, bool JOINED>
__device__ __forceinline__ void chunk_stats(const FilterArgs& a, int b, int chunk) {
  const int V = a.s.V, lane = threadIdx.x & 63;
  const L* row = (const L*)a.s.logits + (long)b * a.s.ld;
  const int lead = lead_of(row, V), v0 = chunk * SF_CHUNK + lane * 8 - lead;
  if (chunk >= chunks_of(V + lead)) return;
  float x[8];
  if (v0 >= 0 && v0 + 8 <= V) {
    u32x4_t u[sizeof(L) / 2];
    __builtin_memcpy(u, row + v0, sizeof(u));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (sizeof(L) == 2) x[e] = __uint_as_float(e & 1 ? u[0][e >> 1] & 0xffff0000u : u[0][e >> 1] << 16);
      else x[e] = __uint_as_float((unsigned)u[e >> 2][e & 3]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (unsigned)(v0 + e) < (unsigned)V ? logit_f(row[v0 + e]) : -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = entry(x[e]);
    mx = fmaxf(mx, x[e]);
  }
  mx = max8(mx);  // a group is 8 lanes
  if ((lane & 7) == 0 && v0 < V) put<JOINED>(a.gmax + (long)b * groups_of(V + SF_LEAD) + chunk * 8 + (lane >> 3), key_of(mx));
  const float top = max_8_64(mx), use = top == -INFINITY ? 0.f : top;
  // 2^t and what t's rounding left, or a term would be off by 2^-24 |t|
  float rest = 0.f;
  int n = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = fmaxf(x[e] - use, -1e4f), t = d * 1.44269504f, q = __builtin_amdgcn_exp2f(t);
    const float left = fmaf(d, 1.92596303e-8f, fmaf(d, 1.44269504f, -t));
    const u64 same = __ballot(x[e] == use);
    n += __popcll(same);
    rest += x[e] == use ? 0.f : fmaf(q, left * 0.693147181f, q);
  }
  rest = sum64(rest);
  const RowOpts o = row_opts(a, b);
  double zt = 0;
  if (o.p < 1 && o.k == 0) {
    const double it = 1.0 / o.T;
#pragma unroll
    for (int e = 0; e < 8; ++e) zt += x[e] == -INFINITY ? 0.0 : weight(x[e], use, it);
    zt = wave_scan(zt);
  }
  if (lane == 63) {
    u64* to = (u64*)(a.sums + (long)b * chunks_of(V + SF_LEAD) + chunk);
    put<JOINED>(to, __builtin_bit_cast(u64, zt));
    put<JOINED>(to + 1, (u64)__float_as_uint(rest) | (u64)__float_as_uint(top) << 32);
    put<JOINED>(to + 2, (u64)(unsigned)n);
  }
}

template <typename L>
__global__ void __launch_bounds__(256) filter_stats_kernel(FilterArgs a) {
  chunk_stats<L, false>(a, blockIdx.y, blockIdx.x * 4 + (threadIdx.x >> 6));
}

// ------------------------------------------------------------------------------------------- the pick
struct PickLds {
  u64 list[SF_CAP];  // (key, ~index) of entries
  union {
    double C[SF_CAP];               // of sorted entries
    unsigned match[SF_MAX_GROUPS];  // each listed group's entries of one value
  };
  u64 mass[SF_BINS];
  unsigned count[SF_BINS];
  unsigned short group[SF_MAX_GROUPS];  // the groups that pass the bound
  double redd[2][16];
  unsigned redu[3][16];
  int redt[8];
  float topw[16];
  u64 redm[16];
  unsigned kappa, n_list;
  int n_group, lead;
  unsigned bin, c_above, c_at, found, range[2];
  u64 m_above;
};

// A value that all lanes hold, in scalar registers: what a function is given is in vector ones, and a branch on it is taken both ways
template <typename T>
__device__ __forceinline__ T uniform(T v) {
  constexpr int N = sizeof(T) / 4;
  unsigned q[N];
  __builtin_memcpy(q, &v, sizeof(T));
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = __builtin_amdgcn_readfirstlane(q[i]);
  __builtin_memcpy(&v, q, sizeof(T));
  return v;
}

// Bins a unit of logit, of a range of them (one of 0 or inf: one bin; finite, or the top's 0 would not be in the first bin)
__device__ __forceinline__ float bins_over(float range) { return range > 0.f ? fminf((SF_BINS - 1) / range, 3e38f) : 0.f; }

// The workgroup's sums over its threads, in order (16 waves): before the thread's own
template <typename T>
__device__ __forceinline__ T scan_before(T v, T* red) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const T s = wave_scan(v);
  __syncthreads();
  if (lane == 63) red[wv] = s;
  __syncthreads();
  T off = 0;
#pragma unroll
  for (int i = 0; i < 15; ++i) off += i < wv ? red[i] : T(0);
  return off + (s - v);
}

__device__ __forceinline__ unsigned block_sum_u(unsigned v, unsigned* red) {
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
  __syncthreads();
  unsigned t = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) t += red[i];
  return t;
}

// A lane's 8 neighbours of a wave's 8 listed groups, as they are in memory (NaN: the row has none there), in words: nothing waits
// for them here
template <typename L>
struct Eight {
  u32x4_t q[sizeof(L) / 2];
  int v;  // the first one's index
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (sizeof(L) == 2) return __uint_as_float(e & 1 ? q[0][e >> 1] & 0xffff0000u : q[0][e >> 1] << 16);
    else {
      const unsigned u = q[e >> 2][e & 3];
      return __uint_as_float(u);
    }
  }
  __device__ __forceinline__ unsigned there(int V) const {  // a bit each
    return v < 0 ? 0xffu << -v & 0xffu >> max(v + 8 - V, 0) : 0xffu >> min(max(v + 8 - V, 0), 8);
  }
};
template <typename L>
__device__ __forceinline__ Eight<L> load_entries(const L* row, int V, const PickLds& S, int g0) {
  const int lane = threadIdx.x & 63, g = g0 + (lane >> 3);
  Eight<L> x;
  x.v = g < S.n_group ? S.group[g] * SF_GROUP + (lane & 7) * 8 - S.lead : V;
  if (x.v >= 0 && x.v + 8 <= V) {
    __builtin_memcpy(x.q, row + x.v, sizeof(x.q));
  } else {
    L q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (sizeof(L) == 2) q[e] = (unsigned)(x.v + e) < (unsigned)V ? row[x.v + e] : (L)0x7fff;
      else q[e] = (unsigned)(x.v + e) < (unsigned)V ? row[x.v + e] : __builtin_nanf("");
    }
    __builtin_memcpy(x.q, q, sizeof(x.q));
  }
  return x;
}

// f(x, index) for the entries of the listed groups (and x = NaN beside them), by whole waves; in a loop where f is long: a
// launch fetches its instructions anew
template <typename L, typename F>
__device__ __forceinline__ void each_entry(const L* row, int V, const PickLds& S, F f) {
  const int n = S.n_group;
  int g0 = (threadIdx.x >> 6) * 8;
  Eight<L> next = load_entries(row, V, S, g0);
  for (; g0 < n; g0 += 128) {
    const Eight<L> now = next;
    next = load_entries(row, V, S, g0 + 128);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = entry(now[e]);  // (a median of -inf and inf would be folded to a minimum, and NaN be inf)
    const unsigned there = now.there(V);
    if (there != 0xff) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = there >> e & 1 ? x[e] : __builtin_nanf("");
    }
#pragma unroll 1
    for (int e = 0; e < 4; ++e) {
      f(x[0], now.v + e);
      f(x[4], now.v + 4 + e);
#pragma unroll
      for (int i = 0; i < 3; ++i) { x[i] = x[i + 1]; x[4 + i] = x[5 + i]; }
    }
  }
}

// (key, ~index) of the listed groups' entries with lo <= key <= hi into the list (n_list of them; those past CAP are only counted,
// and with `stop` no longer once they are). Bound by the vector ALU: three instructions an entry, the counts are scalar
template <typename L>
__device__ __forceinline__ void collect(const L* row, int V, PickLds& S, unsigned lo, unsigned hi, bool stop) {
  const float from = of_key(lo), to = of_last(hi);
  const int n = S.n_group, lane = threadIdx.x & 63;
  int g0 = (threadIdx.x >> 6) * 8;
  Eight<L> next = load_entries(row, V, S, g0);
  for (; g0 < n; g0 += 128) {
    if (stop && *(volatile unsigned*)&S.n_list > SF_CAP) return;
    const Eight<L> now = next;
    next = load_entries(row, V, S, g0 + 128);
    u64 hits[8];
    unsigned all = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) hits[e] = __ballot(__builtin_amdgcn_fmed3f(now[e], from, to) == now[e]);
    if (from == -INFINITY) {  // and NaN
      const unsigned there = now.there(V);
#pragma unroll
      for (int e = 0; e < 8; ++e) hits[e] |= __ballot(now[e] != now[e] && (there >> e & 1));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) all += __popcll(hits[e]);
    if (!all) continue;
    unsigned at = 0;
    if (lane == 0) at = atomicAdd(&S.n_list, all);
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!hits[e]) continue;
      const unsigned mine = at + __builtin_amdgcn_mbcnt_hi((unsigned)(hits[e] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hits[e], 0u));
      if ((hits[e] >> lane & 1) && mine < SF_CAP) S.list[mine] = ((u64)key_of(entry(now[e])) << 32) | (unsigned)~(now.v + e);
      at += __popcll(hits[e]);
    }
  }
}

// The list's first `want` entries in descending order (what is behind them is not in order); a key and its index are no other entry's
__device__ __forceinline__ void sort_list(PickLds& S, unsigned count, unsigned want) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  unsigned n2 = 64, p = 16;  // p threads an entry
  while (n2 < count) n2 *= 2, p /= 2;
  if (n2 <= 128) {  // each entry's rank by counting the larger ones
    const unsigned i = tid / p;
    const u64 mine = i < count ? S.list[i] : 0;
    unsigned rank = 0;
    for (unsigned j = tid & (p - 1); j < count; j += p) rank += S.list[j] > mine;
    for (unsigned o = p / 2; o > 0; o >>= 1) rank += __shfl_xor(rank, o, 64);
    __syncthreads();
    if ((tid & (p - 1)) == 0) S.list[i < count ? rank : i] = mine;
    __syncthreads();
    return;
  }
  // into 2048 bins of equal width between the largest and the smallest value, then each bin's by counting
  unsigned *const held = (unsigned*)S.C, *const start = held + SF_BINS;
  u64 mine[2];
  unsigned lo = ~0u, hi = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const unsigned i = tid + 1024 * e, key = i < count ? (unsigned)(S.list[i] >> 32) : 0;
    mine[e] = i < count ? S.list[i] : 0;
    hi = max(hi, key);
    if (key > 0x007fffffu) lo = min(lo, key);  // (of -inf)
    held[i] = 0;
  }
  lo = wave_min(lo);
  hi = ~wave_min(~hi);
  if (lane == 63) { S.redu[0][wv] = lo; S.redu[1][wv] = hi; }
  if (tid == 0) S.found = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) { lo = min(lo, S.redu[0][i]); hi = max(hi, S.redu[1][i]); }
  const float top = of_key(hi), range = lo < hi ? top - of_key(lo) : 0.f, scale = bins_over(range);
  unsigned bin[2], slot[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float x = of_key((unsigned)(mine[e] >> 32));
    bin[e] = (unsigned)fminf((x == top ? 0.f : top - x) * scale, (float)(SF_BINS - 1));
    if (mine[e]) slot[e] = atomicAdd(&held[bin[e]], 1u);
  }
  __syncthreads();
  const unsigned c0 = held[2 * tid], c1 = held[2 * tid + 1];
  if (max(c0, c1) > SF_CROWD) S.found = 1;
  const unsigned first = scan_before<unsigned>(c0 + c1, S.redu[2]);
  start[2 * tid] = first;
  start[2 * tid + 1] = first + c0;
  __syncthreads();
  if (S.found) {
    for (unsigned i = count + tid; i < n2; i += 1024) S.list[i] = 0;
    for (unsigned size = 2; size <= n2; size *= 2)
      for (unsigned step = size / 2; step > 0; step /= 2) {
        __syncthreads();
        for (unsigned i = tid; i < n2 / 2; i += 1024) {
          const unsigned x = 2 * i - (i & (step - 1)), y = x + step;
          const u64 q = S.list[x], r = S.list[y];
          if ((q < r) == ((x & size) == 0)) { S.list[x] = r; S.list[y] = q; }
        }
      }
    __syncthreads();
    return;
  }
  unsigned at[2], n[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    at[e] = start[bin[e]];
    n[e] = mine[e] && at[e] < want ? held[bin[e]] : 0;
    if (n[e]) S.list[at[e] + slot[e]] = mine[e];
  }
  __syncthreads();
  unsigned rank[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e)
    for (unsigned i = 0, j = slot[e]; i < n[e]; ++i) {  // from its own place on: the bins' starts may share a bank
      rank[e] += S.list[at[e] + j] > mine[e];
      j = j + 1 == n[e] ? 0 : j + 1;
    }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (n[e]) S.list[at[e] + rank[e]] = mine[e];
  __syncthreads();
}

// A row's entries in their order up to a border: the last one's (key, ~index), their mass in units
struct Border { u64 last; double mass; };
enum { BY_COUNT, BY_MASS, OVER_MASS };
struct Goal {
  int by;
  unsigned count;
  double mass;
  __device__ bool reached(unsigned c, double m) const { return by == BY_COUNT ? c >= count : by == BY_MASS ? m >= mass : m > mass; }
};

// The entries of a row that are counted, and their bins: of equal width from the top (scale: bins a unit of logit), or (shift >= 0) of
// 2^shift keys from hi
struct Bins {
  float top, scale;
  double it;
  unsigned lo, hi;  // other keys do not count
  int shift;

  __device__ unsigned of_width(float x) const {  // of equal width
    const float d = x == top ? 0.f : top - x;
    return (unsigned)fminf(d * scale, (float)(SF_BINS - 1));
  }
  __device__ unsigned of(float x) const { return shift >= 0 ? (hi - key_of(x)) >> shift : of_width(x); }
  __device__ double weight_of(float x) const { return weight(x, top, it); }
  __device__ double weight_of(unsigned key) const { return weight_of(of_key(key)); }
  __device__ static u64 units(double w) {  // rint(w 2^45): the low bits of the sum with 2^52
    return (u64)__double_as_longlong(fma(w, SF_UNIT, 4503599627370496.0)) & 0xfffffffffffffull;
  }
  __device__ void split() {  // the keys lo .. hi into 2048 bins or fewer
    const unsigned range = hi - lo;
    shift = range < SF_BINS ? 0 : 21 - __builtin_clz(range);
  }
};

// A weight is e^(-its bin's middle) e^r, |r| <= 1 / 120 in narrow bins: those of e^r are summed (to r^5 / 120: 5e-16 left), half of
// the whole exponential's instructions (25 -> 16 us of 33 flat rows of 50257), and the bins' factors applied behind it
template <typename L>
__device__ __forceinline__ void fill_bins(const L* row, int V, PickLds& S, const Bins& r) {
  __syncthreads();
  for (int i = threadIdx.x; i < SF_BINS; i += 1024) { S.mass[i] = 0; S.count[i] = 0; }
  __syncthreads();
  const float from = of_key(r.lo), to = of_last(r.hi);
  const double step = r.it / r.scale;  // of the exponent, a bin
  if (r.shift < 0 && step <= 1.0 / 60) {
    const double top = r.top, half = 0.5 * step;
    each_entry(row, V, S, [&](float x, int) {
      if (__builtin_amdgcn_fmed3f(x, from, to) != x) return;
      const unsigned at = r.of_width(x);
      const double e = fma(fmin((double)x - top, 0.0), r.it, fma((double)at, step, half));  // (0 of infinite ones)
      double q = 1.0 / 120;
      q = fma(q, e, 1.0 / 24);
      q = fma(q, e, 1.0 / 6);
      q = fma(q, e, 0.5);
      q = fma(q, e, 1.0);
      q = fma(q, e, 1.0);
      atomicAdd(&S.count[at], 1u);
      atomicAdd(&S.mass[at], Bins::units(q));
    });
    __syncthreads();
    for (int i = threadIdx.x; i < SF_BINS; i += 1024)
      if (S.mass[i]) S.mass[i] = (u64)rint((double)S.mass[i] * exp_neg(-fma((double)i, step, half)));
  } else {
    each_entry(row, V, S, [&](float x, int) {
      if (__builtin_amdgcn_fmed3f(x, from, to) != x) return;
      const unsigned at = r.of(x);
      atomicAdd(&S.count[at], 1u);
      atomicAdd(&S.mass[at], Bins::units(r.weight_of(x)));
    });
  }
  __syncthreads();
}

// The first bin by which the goal is reached, from `above` entries of mass `m_above` on (the last that holds something, if none is):
// S.bin, what is before it, and what it holds
__device__ __forceinline__ void find_bin(PickLds& S, const Goal& goal, unsigned above, u64 m_above) {
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const unsigned c0 = S.count[2 * tid], c1 = S.count[2 * tid + 1];
  const u64 m0 = S.mass[2 * tid], m1 = S.mass[2 * tid + 1];
  const unsigned cs = wave_scan(c0 + c1);
  const u64 ms = wave_scan(m0 + m1);
  __syncthreads();
  if (lane == 63) { S.redu[0][wv] = cs; S.redm[wv] = ms; }
  if (tid == 0) S.found = 0;
  __syncthreads();
  unsigned all = above, cb = above + cs - (c0 + c1);
  u64 mb = m_above + ms - (m0 + m1);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    all += S.redu[0][i];
    cb += i < wv ? S.redu[0][i] : 0;
    mb += i < wv ? S.redm[i] : 0;
  }
  auto take = [&](unsigned i, unsigned c_above, unsigned c_at, u64 mass) { S.bin = i; S.c_above = c_above; S.c_at = c_at; S.m_above = mass; };
  const bool r0 = goal.reached(cb, (double)mb), r1 = goal.reached(cb + c0, (double)(mb + m0)), r2 = goal.reached(cb + c0 + c1, (double)(mb + m0 + m1));
  if (c0 && !r0 && r1) take(2 * tid, cb, c0, mb), S.found = 1;
  if (c1 && !r1 && r2) take(2 * tid + 1, cb + c0, c1, mb + m0), S.found = 1;
  __syncthreads();
  if (!S.found) {
    if (c0 && cb + c0 == all) take(2 * tid, cb, c0, mb);
    if (c1 && cb + c0 + c1 == all) take(2 * tid + 1, cb + c0, c1, mb + m0);
  }
  __syncthreads();
}

// The smallest key of lo .. hi for which f holds, as it does for the larger ones (and for hi); whole waves: 64 keys of a range at a time
template <typename F>
__device__ __forceinline__ unsigned first_key(unsigned lo, unsigned hi, F f) {
  const unsigned lane = threadIdx.x & 63;
  while (lo < hi) {
    const unsigned step = (hi - lo) / 64 + 1, k = lo + lane * step;
    const u64 in = __ballot(k >= lo && k < hi && f(k));
    if (!in) {  // behind the last key tried
      lo += (hi - 1 - lo) / step * step + 1;
      continue;
    }
    const unsigned i = __builtin_ctzll(in);
    hi = lo + i * step;
    lo = i ? hi - step + 1 : lo;
  }
  return lo;
}

// The border in the bin that was found (of equal width, up to CAP entries): its entries sorted
template <typename L>
__device__ __forceinline__ Border sorted_border(const L* row, int V, PickLds& S, const Bins& r, const Goal& goal) {
  const int tid = threadIdx.x;
  const unsigned bin = S.bin, above = S.c_above;
  const double m_above = (double)S.m_above;
  if (tid == 0) S.n_list = 0;
  // the bin's keys, from the first of it to before the first of the bin above
  if (tid < 128) {
    const unsigned upto = tid < 64 ? bin : bin - 1;  // (hi is in bin 0)
    const unsigned a = upto < SF_BINS ? first_key(r.lo, r.hi, [&](unsigned k) { return r.of_width(of_key(k)) <= upto; }) : r.hi + 1;
    if ((tid & 63) == 0) S.range[tid >> 6] = tid < 64 ? a : a - 1;
  }
  __syncthreads();
  const unsigned from = uniform(S.range[0]), to = uniform(S.range[1]);
  collect(row, V, S, from, to, false);
  __syncthreads();
  const unsigned n = min(S.n_list, (unsigned)SF_CAP);
  sort_list(S, n, n);
  double w[2], sum = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const unsigned i = 2 * tid + e;
    sum += w[e] = i < n ? (double)Bins::units(r.weight_of((unsigned)(S.list[i] >> 32))) : 0.0;
  }
  double C = m_above + scan_before<double>(sum, S.redd[0]);
  unsigned before = 0;  // entries that do not reach the goal
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const unsigned i = 2 * tid + e;
    C += w[e];
    if (i < n) {
      S.C[i] = C;
      before += !goal.reached(above + i + 1, C);
    }
  }
  const unsigned at = min(block_sum_u(before, S.redu[2]), n - 1);
  const Border b{S.list[at], S.C[at]};
  __syncthreads();
  return b;
}

// The border among the entries of one value, r.hi, which the bins of one key each have found: the last one's index by counting
template <typename L>
__device__ __forceinline__ Border equal_border(const L* row, int V, PickLds& S, const Bins& r, const Goal& goal) {
  const int tid = threadIdx.x, lane = tid & 63;
  const unsigned key = r.hi, above = S.c_above, at = S.c_at;
  const double m_above = (double)S.m_above, w = (double)Bins::units(r.weight_of(key));
  double n = at;  // of that value
  if (S.found && goal.by == BY_COUNT) n = goal.count - above;
  else if (S.found && w > 0) n = goal.by == BY_MASS ? ceil((goal.mass - m_above) / w) : floor((goal.mass - m_above) / w) + 1;
  const unsigned nth = (unsigned)fmin(fmax(n, 1.0), (double)at);
  __syncthreads();
  for (int g = tid; g < SF_MAX_GROUPS; g += 1024) S.match[g] = 0;
  __syncthreads();
  const float value = of_key(key);
  each_entry(row, V, S, [&](float x, int v) {
    if (x == value) atomicAdd(&S.match[v / SF_GROUP], 1u);
  });
  __syncthreads();
  unsigned c[4], sum = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) sum += c[e] = S.match[4 * tid + e];
  unsigned before = scan_before<unsigned>(sum, S.redu[0]);
  if (before < nth && before + sum >= nth) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (before < nth && before + c[e] >= nth) {
        S.bin = 4 * tid + e;
        S.c_at = nth - before;  // of its matches
      }
      before += c[e];
    }
  }
  __syncthreads();
  const int v = S.bin * SF_GROUP + lane;  // (each wave for itself)
  const u64 hit = __ballot(v < V && key_of(entry(logit_f(row[min(v, V - 1)]))) == key);
  const u64 me = __ballot((hit >> lane & 1) && __popcll(hit & ((2ull << lane) - 1)) == S.c_at);
  const unsigned index = S.bin * SF_GROUP + __builtin_ctzll(me | (1ull << 63));
  __syncthreads();
  return {((u64)key << 32) | (unsigned)~index, m_above + nth * w};
}

// Rows of more entries than the list holds: the borders of top-k and of top-p, then u's. A function of its own, with the LDS as such:
// inside the kernel its registers were the other rows' too (23 of them went to memory, a row of 32064 took a quarter longer), and
// through generic pointers it took 95 us for 68. One for
// each kernel: it knows where the LDS is (66 us for 61).
typedef __attribute__((address_space(3))) PickLds* lds_pick_t;
template <typename L, bool JOINED>
__device__ __attribute__((noinline)) u64 pick_counted(const __attribute__((address_space(1))) L* global, int V, lds_pick_t lds, RowOpts o,
                                                  Bins all, double zt, double u) {
  const L* row = (const L*)uniform(global);
  PickLds& S = *(PickLds*)lds;
  const int tid = threadIdx.x;
  V = uniform(V);
  o = {uniform(o.T), uniform(o.p), uniform(o.m), uniform(o.k)};
  all = {uniform(all.top), uniform(all.scale), uniform(all.it), uniform(all.lo), uniform(all.hi), -1};
  zt = uniform(zt);
  u = uniform(u);
  Border end{0, 0};  // of what is kept (last 0: all that counts)
  const bool mass_of_k = o.k && o.p < 1;  // the mass of the top k counts, whatever min-p leaves of them
  auto from_min_p = [&] {  // the keys of too small a weight for it
    if (tid < 64) S.range[0] = first_key(all.lo, all.hi, [&](unsigned k) { return all.weight_of(k) >= o.m; });
    __syncthreads();
    all.lo = uniform(S.range[0]);
    __syncthreads();
  };
  if (o.m > 0 && !mass_of_k) from_min_p();
  Bins r = all;
  bool filled = false, cut = !mass_of_k;
  int border = o.k ? 0 : o.p < 1 ? 1 : 2;
  unsigned above = 0;
  u64 m_above = 0;
  for (;;) {
    if (border == 2 && r.shift < 0 && o.m > 0 && !cut && r.weight_of((unsigned)(end.last >> 32)) < o.m) {
      cut = true;
      from_min_p();
      r.lo = all.lo;
      filled = false;
      end.last = 0;
    }
    if (!filled) fill_bins(row, V, S, r);
    filled = true;
    if (border == 2 && r.shift < 0 && end.last == 0) {
      const u64 mine = S.mass[2 * tid] + S.mass[2 * tid + 1], before = scan_before<u64>(mine, S.redm);
      if (tid == 1023) S.m_above = before + mine;
      __syncthreads();
      end.mass = (double)S.m_above;
    }
    const Goal goal = border == 0 ? Goal{BY_COUNT, (unsigned)o.k, 0.0}
                      : border == 1 ? Goal{BY_MASS, 0, fmax(o.p * (o.k ? end.mass : zt * SF_UNIT), 1.0)}  // (the first entry at least)
                                    : Goal{OVER_MASS, 0, u * end.mass};
    find_bin(S, goal, above, m_above);
    Border b;
    if (r.shift < 0 && uniform(S.c_at) <= SF_CAP) {
      b = sorted_border(row, V, S, r, goal);
    } else {
      // too many in one bin: all the keys into bins of keys, and again the bin that is found, until it is one key
      if (r.shift >= 0) {
        above = uniform(S.c_above);
        m_above = uniform(S.m_above);
        r.hi -= uniform(S.bin) << r.shift;
        const unsigned low = r.hi - ((1u << r.shift) - 1);
        if (low > r.lo && low <= r.hi) r.lo = low;
      }
      filled = false;
      if (r.shift != 0) {
        r.split();
        continue;
      }
      b = equal_border(row, V, S, r, goal);
      above = 0;
      m_above = 0;
      r.lo = all.lo;
      r.hi = all.hi;
      r.shift = -1;
    }
    if (b.last > end.last) end = {b.last, border == 2 ? end.mass : b.mass};  // (an earlier entry is larger; u's is no later than the end)
    if (border == 2) return end.last;
    border = border == 0 && o.p < 1 ? 1 : 2;
  }
}

// Rows of which more entries than the list holds pass the bound, but top-k keeps fewer: all that pass it into 2048 bins of equal width,
// and those down to the k-th's bin into the list. Returns how many they are (or too many, as before)
template <typename L, bool JOINED>
__device__ __attribute__((noinline)) unsigned collect_k(const __attribute__((address_space(1))) L* global, int V, lds_pick_t lds, unsigned k,
                                                        unsigned kappa, unsigned hi) {
  const L* row = (const L*)uniform(global);
  PickLds& S = *(PickLds*)lds;
  const int tid = threadIdx.x;
  V = uniform(V);
  k = uniform(k);
  kappa = uniform(kappa);
  hi = uniform(hi);
  const float top = of_key(hi), from = of_key(kappa), range = top - from, scale = bins_over(range);
  if (!(range > 0.f && range < INFINITY)) return SF_CAP + 1;
  S.count[2 * tid] = S.count[2 * tid + 1] = 0;
  __syncthreads();
  each_entry(row, V, S, [&](float x, int) {
    if (x >= from) atomicAdd(&S.count[(unsigned)fminf((top - x) * scale, (float)(SF_BINS - 1))], 1u);
  });
  __syncthreads();
  const unsigned c0 = S.count[2 * tid], c1 = S.count[2 * tid + 1], before = scan_before<unsigned>(c0 + c1, S.redu[0]);
  if (before < k && before + c0 + c1 >= k) {
    const bool second = before + c0 < k;
    S.bin = 2 * tid + second;
    S.c_at = before + c0 + (second ? c1 : 0);
  }
  if (tid == 0) S.n_list = 0;
  __syncthreads();
  if (S.c_at > SF_CAP) return SF_CAP + 1;
  // the bin's lower end, below what rounding could do
  const float edge = (S.bin + 1) / scale, low = top - edge - 1e-6f * (fabsf(top) + edge);
  collect(row, V, S, max(kappa, key_of(low)), hi, true);
  __syncthreads();
  return S.n_list;
}

// Up to 64 NW entries: NW waves (the others have ended), an entry a thread
template <int NW>
__device__ __forceinline__ u64 pick_few(PickLds& S, unsigned count, const RowOpts& o, float top, double it, double zt, double u) {
  const unsigned tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  // (a lone wave's lanes run together and its LDS accesses are in order: only the compiler has to keep them so)
  auto sync = [] {
    if constexpr (NW > 1) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  };
  auto votes = [&](bool v, unsigned* red) {  // threads of the NW waves for which v
    const unsigned n = __popcll(__ballot(v));
    if constexpr (NW == 1) return n;
    if (lane == 0) red[wv] = n;
    __syncthreads();
    unsigned all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) all += red[i];
    return all;
  };
  const u64 mine = tid < count ? S.list[tid] : 0;
  unsigned rank = 0;
#pragma unroll 4
  for (unsigned j = 0; j < count; ++j) rank += S.list[j] > mine;
  sync();
  if (tid < count) S.list[rank] = mine;
  sync();
  const u64 at = tid < count ? S.list[tid] : 0;
  const double w = tid < count ? weight(of_key((unsigned)(at >> 32)), top, it) : 0.0;
  double C = wave_scan(w);
  if constexpr (NW > 1) {
    if (lane == 63) S.redd[0][wv] = C;
    __syncthreads();
    double off = 0;
#pragma unroll
    for (int i = 0; i < NW - 1; ++i) off += i < (int)wv ? S.redd[0][i] : 0.0;
    C += off;
  }
  S.C[tid] = C;
  sync();
  unsigned n = min(o.k ? (unsigned)o.k : count, count);
  if (o.p < 1) n = min(n, votes(tid < count && C < o.p * (o.k ? S.C[n - 1] : zt), S.redu[0]) + 1);
  if (o.m > 0) n = min(n, max(1u, votes(tid < count && w >= o.m, S.redu[1])));
  const double t = u * S.C[n - 1];
  return S.list[min(votes(tid < n && C <= t, S.redu[2]), n - 1)];
}

__device__ __forceinline__ u64 pick_sorted(PickLds& S, unsigned count, const RowOpts& o, float top, double it, double zt, double u) {
  const int tid = threadIdx.x;
  const unsigned want = o.k ? min((unsigned)o.k, count) : count;
  sort_list(S, count, want);
  count = want;
  double w[2], sum = 0;
  unsigned over = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const unsigned i = 2 * tid + e;
    sum += w[e] = i < count ? weight(of_key((unsigned)(S.list[i] >> 32)), top, it) : 0.0;
    over += i < count && w[e] >= o.m;
  }
  double C = scan_before<double>(sum, S.redd[0]);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    C += w[e];
    S.C[2 * tid + e] = C;
  }
  __syncthreads();
  unsigned n = min(o.k ? (unsigned)o.k : count, count);
  if (o.p < 1) {
    const double t = o.p * (o.k ? S.C[n - 1] : zt);
    unsigned c = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) c += (unsigned)(2 * tid + e) < count && S.C[2 * tid + e] < t;
    n = min(n, block_sum_u(c, S.redu[0]) + 1);
  }
  if (o.m > 0) n = min(n, max(1u, block_sum_u(over, S.redu[1])));
  const double t = u * S.C[n - 1];
  unsigned c = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e) c += (unsigned)(2 * tid + e) < n && S.C[2 * tid + e] <= t;
  return S.list[min(block_sum_u(c, S.redu[2]), n - 1)];
}

// JOINED: the statistics in the same launch, of which the last of a row's workgroups to have its own goes on
template <typename L, bool JOINED>
__global__ void __launch_bounds__(1024) filter_pick_kernel(FilterArgs a) {
  __shared__ __attribute__((aligned(16))) PickLds S;
  const int b = JOINED ? blockIdx.y : blockIdx.x;
  if constexpr (JOINED) {
    chunk_stats<L, true>(a, b, blockIdx.x * SF_WG + (threadIdx.x >> 6));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (gridDim.x > 1) {
      if (threadIdx.x == 0) {
        S.found = __hip_atomic_fetch_add(a.tickets + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
        if (S.found) put<true>(a.tickets + b, 0);
      }
      __syncthreads();
      if (!S.found) return;
    }
  }
  const int V = a.s.V, tid = threadIdx.x, lane = tid & 63;
  const L* row = (const L*)a.s.logits + (long)b * a.s.ld;
  const int lead = lead_of(row, V), NG = groups_of(V + lead), NC = chunks_of(V + lead);
  a.gmax += (long)b * groups_of(V + SF_LEAD);
  ChunkSum cs{0, 0.f, -INFINITY, 0, 0};
  if (tid < NC) {
    const u64* p = (const u64*)(a.sums + (long)b * chunks_of(V + SF_LEAD) + tid);
    const u64 q0 = get<JOINED>(p), q1 = get<JOINED>(p + 1), q2 = get<JOINED>(p + 2);
    cs = {__builtin_bit_cast(double, q0), __uint_as_float((unsigned)q1), __uint_as_float((unsigned)(q1 >> 32)), (int)q2, 0};
  }
  unsigned gm[4];
  unsigned least = ~0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    gm[e] = tid + 1024 * e < NG ? get<JOINED>(a.gmax + tid + 1024 * e) : 0;
    if (tid + 1024 * e < NG) least = min(least, gm[e]);
  }
  const RowOpts o = row_opts(a, b);
  const double it = 1.0 / o.T;
  double u;
  if (a.u) u = a.u[b];
  else u = u01(a.s.seed, (a.s.ctr ? (unsigned)a.s.ctr[b] : a.s.step) * 131071u + (unsigned)b, 0u);
  u = fmin(fmax(u, 0.0), 1.0);
  if (tid == 0) S.kappa = 0, S.n_group = 0, S.n_list = 0, S.lead = lead;
  S.count[tid] = 0;
  const float tops = max_8_64(max8(cs.m));
  least = wave_min(least);
  if (lane == 63) { S.topw[tid >> 6] = tops; S.redu[1][tid >> 6] = least; }
  __syncthreads();
  float top = S.topw[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, S.topw[i]);  // (chunks there are up to 512 of)
  if (top == -INFINITY) {
    if (tid == 0) sample_bookkeep(a.s, b, 0, -INFINITY);
    return;
  }
  double z1 = 0, zt = 0;  // of exp(x - top) without the entries of `top`, and how many these are
  int tops_n = 0;
  if (cs.m != -INFINITY) {
    z1 = ((double)cs.rest + (cs.m == top ? 0 : cs.n)) * weight(cs.m, top, 1.0);
    tops_n = cs.m == top ? cs.n : 0;
    if (o.p < 1 && o.k == 0) zt = cs.zt * weight(cs.m, top, it);
  }
  if (tid < 512) {
    z1 = wave_scan(z1);
    zt = wave_scan(zt);
    tops_n = wave_scan(tops_n);
    if (lane == 63) { S.redd[0][tid >> 6] = z1; S.redd[1][tid >> 6] = zt; S.redt[tid >> 6] = tops_n; }
  }
  const unsigned hi = key_of(top);
  // ---- the bound ----
  unsigned kappa = key_of(-INFINITY);
  if (o.k && o.k <= NG) {
    // the k-th largest group's bin of 1024 between the smallest and the largest
#pragma unroll
    for (int i = 0; i < 16; ++i) least = min(least, S.redu[1][i]);
    const unsigned range = hi - least;
    const int shift = range < 1024 ? 0 : 22 - __builtin_clz(range);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (tid + 1024 * e < NG) atomicAdd(&S.count[(hi - gm[e]) >> shift], 1u);
    __syncthreads();
    const unsigned mine = S.count[tid], before = scan_before<unsigned>(mine, S.redu[0]);
    if (before < (unsigned)o.k && before + mine >= (unsigned)o.k) {
      const unsigned up = ((unsigned)tid << shift) + ((1u << shift) - 1);
      S.kappa = up >= hi ? 0 : hi - up;
    }
    __syncthreads();
    kappa = max(kappa, S.kappa);
  }
  __syncthreads();
  z1 = zt = 0;
  tops_n = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    z1 += S.redd[0][i];
    tops_n += S.redt[i];
    zt += S.redd[1][i];
  }
  // entries 44 T below the top: 262144 of them hold 2e-14, a tenth of the rounding of a weight
  kappa = max(kappa, key_of(fmaxf(top - (float)(44.0 * o.T), -INFINITY)));
  if (!(o.k && o.p < 1)) {  // (with both, the mass of the top k is needed)
    double least_w = o.m;
    if (o.p < 1) least_w = fmax(least_w, (1.0 - o.p) * zt / V);
    if (least_w > 0) {
      const float below = fminf((float)o.T * __logf((float)least_w), 0.f);
      const float f = top + below - 1e-5f * (fabsf(top) + fabsf(below) + (float)o.T);  // (safely below what rounding could do)
      if (f == f) kappa = max(kappa, key_of(f));
    }
    kappa = min(kappa, hi);
  }
  // ---- the groups that pass it, in any order, and their entries ----
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool hit = tid + 1024 * e < NG && gm[e] >= kappa;
    const u64 all = __ballot(hit);
    if (!all) continue;
    unsigned at = 0;
    if (lane == 0) at = atomicAdd(&S.n_group, __popcll(all));
    at = __builtin_amdgcn_readfirstlane(at) + __popcll(all & ((1ull << lane) - 1));
    if (hit) S.group[at] = (unsigned short)(tid + 1024 * e);
  }
  __syncthreads();
  collect(row, V, S, kappa, hi, true);  // (too many to sort: the counted way, whatever their number)
  __syncthreads();
  unsigned count = S.n_list;
  if (count > SF_CAP && o.k && o.k < SF_CAP)
    count = collect_k<L, JOINED>((const __attribute__((address_space(1))) L*)row, V, (lds_pick_t)&S, (unsigned)o.k, kappa, hi);
  u64 at;
  if (count <= 64) {
    if (tid >= 64) return;
    at = pick_few<1>(S, count, o, top, it, zt, u);
  } else if (count <= 64 * SF_FEW) {
    if (tid >= 64 * SF_FEW) return;
    at = pick_few<SF_FEW>(S, count, o, top, it, zt, u);
  } else if (count <= SF_CAP) {
    at = pick_sorted(S, count, o, top, it, zt, u);
  } else {
    // weights below a unit's half do not count: 32 T below the top
    kappa = max(kappa, key_of(fmaxf(top - (float)(32.0 * o.T), -INFINITY)));
    const float range = top - of_key(kappa);
    at = pick_counted<L, JOINED>((const __attribute__((address_space(1))) L*)row, V, (lds_pick_t)&S, o, Bins{top, bins_over(range), it, kappa, hi, -1}, zt, u);
  }
  if (tid == 0) {
    const float x = of_key((unsigned)(at >> 32));
    const double d = x == top ? 0.0 : (double)x - (double)top;
    const double y = z1 + (tops_n - 1);  // what the others are beside the first: log(1 + y) to y's own precision
    double log_z = y * (1.0 - y * (0.5 - y * (1.0 / 3)));
    if (y > 1e-4) {  // (and a step of Newton's method)
      log_z = log1pf((float)y);
      log_z += (1.0 + y) * exp_neg(-log_z) - 1.0;
    }
    sample_bookkeep(a.s, b, (int)~(unsigned)at, (float)(d - log_z));
  }
}

DA_EXPORT size_t da_sample_filtered_ws(int B, int V) {
  return B * (chunks_of(V + SF_LEAD) * sizeof(ChunkSum) + groups_of(V + SF_LEAD) * (size_t)4);
}

static int workgroups_of(int V) { return (chunks_of(V + SF_LEAD) + SF_WG - 1) / SF_WG; }  // of a row, in one launch

// Whether B rows go in one launch, and how many tickets (ints, 0) that takes: none where a workgroup has a whole row
static bool one_launch(int B, int V) {
  const int wgs = workgroups_of(V);
  return wgs == 1 ? B <= SF_JOINED_ROWS : B * (long)wgs <= SF_JOINED;
}
DA_EXPORT int da_sample_filtered_tickets(int B, int V) { return workgroups_of(V) > 1 && one_launch(B, V) ? B : 0; }

DA_EXPORT int da_sample_filtered(const void* logits, int f32, int B, int V, int ld, double T, double p, double m, int k,
                                 const void* Ts, const void* ps, const void* ms, const void* ks, const void* u, unsigned seed,
                                 unsigned step, const void* ctr, void* ws, void* tickets, void* out_tok, void* out_lp, void* conf, void* active,
                                 void* pos, void* lens, void* hist, const void* start, int hist_ld, int eos0, int eos1, int eos2,
                                 int eos3, void* stream) {
  if (V < 1 || V > SF_MAX_V || B > 65535 || (hist && (!pos || !start))) return (int)hipErrorInvalidValue;
  if (B == 0) return 0;
  const int NC = chunks_of(V + SF_LEAD);
  SampleArgs s{logits, V, ld, 0.f, seed, step, (const int*)ctr, (int*)out_tok, (float*)out_lp, (float*)conf, (int*)active,
               (int*)pos, (int*)lens, (int*)hist, (const int*)start, hist_ld, eos0, eos1, eos2, eos3};
  FilterArgs a{T, p, m, (const float*)Ts, (const float*)ps, (const float*)ms, k, (const int*)ks, (const float*)u,
               (unsigned*)((char*)ws + (size_t)B * NC * sizeof(ChunkSum)), (ChunkSum*)ws, (int*)tickets, s};
  hipStream_t st = (hipStream_t)stream;
  const int wgs = workgroups_of(V);
  if (one_launch(B, V)) {
    if (wgs > 1 && !tickets) return (int)hipErrorInvalidValue;
    if (f32) filter_pick_kernel<float, true><<<dim3(wgs, B), 1024, 0, st>>>(a);
    else filter_pick_kernel<bf16_t, true><<<dim3(wgs, B), 1024, 0, st>>>(a);
    DA_LAUNCH_CHECK();
  }
  if (f32) filter_stats_kernel<float><<<dim3((NC + 3) / 4, B), 256, 0, st>>>(a);
  else filter_stats_kernel<bf16_t><<<dim3((NC + 3) / 4, B), 256, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (f32) filter_pick_kernel<float, false><<<B, 1024, 0, st>>>(a);
  else filter_pick_kernel<bf16_t, false><<<B, 1024, 0, st>>>(a);
  DA_LAUNCH_CHECK();
}
