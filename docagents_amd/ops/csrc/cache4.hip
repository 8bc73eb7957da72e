// A key / value cache held in 4 bits: its write (RoPE inside or not), its read, attention of one new token a sequence over
// it, and the eviction of the keys of least weight.
//
// Format: codes [slots, Hkv, max_seq, D / 2] (element 2 j in the low half of byte j), a code a sign and one of the magnitudes
// 0, .5, 1, 1.5, 2, 3, 4, 6 (e2m1), and a scale for 32 elements along the head: 2^(byte - 127), [slots, Hkv, max_seq, 4] bytes
// of which D / 32 are used; 255: the block held an inf or a NaN and reads as NaN. Power-of-two scales: a value is exact in
// bf16, one conversion instruction makes two of them, and both products run on bf16 MFMA. Rows are whole and in order, so that
// a token is written, read and moved by itself. 136 bytes a key and KV head of 128 for 512 in bf16.
// Scale of a block with largest magnitude a = m 2^e (1 <= m < 2): 2^(e - 2) for m < 1.75 and 2^(e - 1) above it (6 stands for
// up to 7 then): root mean square error 11.2 % of normal values, 11.5 % if the step is at m = 2 or 1.5. The smallest scale is 2^-126
// (codes of it may be subnormal); an element of 1.75 2^127 or more is 2^128, which reads as inf.
#include "common.h"

typedef __attribute__((ext_vector_type(2))) __bf16 bf2_t;

struct Cache4 {
  uint8_t *k, *ks, *v, *vs;
  int slots, Hkv, max_seq;
};

template <int B>  // byte of w
__device__ __forceinline__ unsigned bf2_of4(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}

// Byte `at` as the scale of a conversion: turned to where an exponent is; what else is in the word does not count
__device__ __forceinline__ float scale_of(unsigned bytes, int at) {
  return __uint_as_float(__builtin_amdgcn_alignbit(bytes, bytes, (8 * at + 9) & 31));  // (the conversion takes bits 23 - 30; 255: NaN)
}

__device__ __forceinline__ long row_of(const Cache4& c, int slot, int h, int at) {
  return ((long)slot * c.Hkv + h) * c.max_seq + at;
}

// ------------------------------------------------------------------------------------------- write, read
// 8 consecutive elements a lane, 4 lanes a block; x as bf16 pairs. Returns the codes (the conversion's rounding: to nearest, ties to
// the even code, past 6 to 6); the block's scale byte in `sb`.
__device__ __forceinline__ unsigned encode8(const u32x4_t& x, unsigned& sb) {
  unsigned a = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) a = max(a, max((x[e] << 16) & 0x7fffffffu, x[e] & 0x7fff0000u));
  a = max(a, (unsigned)__builtin_amdgcn_mov_dpp((int)a, 0xB1, 0xf, 0xf, true));  // lanes 1 and 2 away
  a = max(a, (unsigned)__builtin_amdgcn_mov_dpp((int)a, 0x4E, 0xf, 0xf, true));
  sb = (unsigned)max(1, (int)((a + 0x200000u) >> 23) - 2);
  const float scale = __uint_as_float(sb << 23);
  const unsigned x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];  // (a bit_cast of a vector's element itself is one of its first)
  unsigned r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(bf2_t, x0), scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf2_t, x1), scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf2_t, x2), scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf2_t, x3), scale, 3);
  if ((a >> 23) >= 255) { sb = 255; r = 0; }
  return r;
}

struct Write4 {
  bf16_t *q, *k, *v;  // rows of T tokens; q only with cs
  int ldk, ldv, T, H, D, npos;  // npos: rows of cs
  const int *slot, *at, *pos;
  const float* cs;
  float* weight;
  Cache4 c;
};

// A lane per 8 elements, 8 (heads of 64) or 16 lanes a row, W4_T tokens a thread, one behind the other in the cache as a rule: their
// rows share lines. With cs the heads of q and k are rotated in place first (rope_cache's arithmetic, its bits).
// Bound by memory: 16384 tokens of 32 heads x 96 (258 MB read and written) 107 us with a token a thread, 64-bit divisions, comparisons
// for the codes and a byte a scale; neighbouring tokens on one XCD and inputs past the caches as well -> 54.
constexpr int W4_T = 4;
__global__ void __launch_bounds__(256) cache4_write_kernel(Write4 p) {
  const int wg = xcd_remap(blockIdx.x + gridDim.x * blockIdx.y, gridDim.x * gridDim.y), tb = wg % gridDim.x;
  const int lg = p.D == 64 ? 3 : 4, r = wg / gridDim.x * 256 + threadIdx.x, hh = r >> lg, c = r & ((1 << lg) - 1);
  if (hh >= p.H + 2 * p.c.Hkv) return;  // (whole rows)
  const bool is_q = hh < p.H, is_k = !is_q && hh < p.H + p.c.Hkv, in = c < p.D / 8;
  const int h = is_q ? hh : is_k ? hh - p.H : hh - p.H - p.c.Hkv;
  bf16_t* src = (is_q ? p.q : is_k ? p.k : p.v) + h * p.D + c * 8;
  const long ld = is_q || is_k ? p.ldk : p.ldv;
  const int t0 = tb * W4_T;
  u32x4_t x[W4_T];
  int s[W4_T], at[W4_T];
#pragma unroll
  for (int i = 0; i < W4_T; ++i) {
    const int t = min(t0 + i, p.T - 1);
    x[i] = in ? __builtin_nontemporal_load((const u32x4_t*)(src + t * ld)) : u32x4_t{0, 0, 0, 0};
    s[i] = p.slot[t];
    at[i] = p.at[t];
  }
#pragma unroll
  for (int i = 0; i < W4_T; ++i) {
    const int t = t0 + i;
    if (t >= p.T) return;
    if (p.cs && (unsigned)p.pos[t] >= (unsigned)p.npos) continue;
    if (p.cs && (is_q || is_k) && in) {
      const float* f = p.cs + ((long)p.pos[t] * (p.D / 2) + c * 4) * 2;
      const f32x4_t c01 = *(const f32x4_t*)f, c23 = *(const f32x4_t*)(f + 4);
      const float cc[4] = {c01[0], c01[2], c23[0], c23[2]}, sn[4] = {c01[1], c01[3], c23[1], c23[3]};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x1 = bf2f(x[i][e] & 0xffff), x2 = bf2f(x[i][e] >> 16);
        x[i][e] = pack_bf2(fmaf(x1, cc[e], -(x2 * sn[e])), fmaf(x2, cc[e], x1 * sn[e]));
      }
      *(u32x4_t*)(src + t * ld) = x[i];
    }
    if (is_q) continue;
    unsigned sb;
    const unsigned codes = encode8(x[i], sb);
    unsigned all = (c & 3) ? 0 : sb << (8 * (c >> 2));  // the row's scales, in its first lane
    if (!in) all = 0;
    if (lg == 4) all |= (unsigned)__shfl_down((int)all, 8, 16);
    all |= (unsigned)__shfl_down((int)all, 4, 8);
    if ((unsigned)s[i] >= (unsigned)p.c.slots || (unsigned)at[i] >= (unsigned)p.c.max_seq) continue;
    const long row = row_of(p.c, s[i], h, at[i]);
    if (in) *(unsigned*)((is_k ? p.c.k : p.c.v) + row * (p.D / 2) + c * 4) = codes;
    if (c == 0) {
      *(unsigned*)((is_k ? p.c.ks : p.c.vs) + row * 4) = all;
      if (p.weight && is_k) p.weight[row] = 0.f;
    }
  }
}

__global__ void __launch_bounds__(256) cache4_read_kernel(Cache4 c, int slot, int n, int D, bf16_t* k, bf16_t* v) {
  const int ch = D / 8;
  const long item = (long)blockIdx.x * 256 + threadIdx.x, each = (long)c.Hkv * n * ch;
  if (item >= 2 * each) return;
  const bool is_v = item >= each;
  const long i = is_v ? item - each : item;
  const long hr = i / ch;
  const int e = (int)(i - hr * ch), h = (int)(hr / n), at = (int)(hr - (long)h * n);
  const long row = row_of(c, slot, h, at);
  const unsigned w = *(const unsigned*)((is_v ? c.v : c.k) + row * (D / 2) + e * 4);
  const float s = scale_of(*(const unsigned*)((is_v ? c.vs : c.ks) + row * 4), e >> 2);
  *(u32x4_t*)((is_v ? v : k) + i * 8) = u32x4_t{bf2_of4<0>(w, s), bf2_of4<1>(w, s), bf2_of4<2>(w, s), bf2_of4<3>(w, s)};
}

DA_EXPORT int da_cache4_write(void* q, void* k, void* v, int ldk, int ldv, const void* slot, const void* at, const void* pos,
                              const void* cs, int npos, void* ck, void* cks, void* cv, void* cvs, void* weight, int T, int H,
                              int Hkv, int D, int slots, int max_seq, void* stream) {
  if (D % 32 || D < 32 || D > 128 || (cs && (!pos || !q)) || (!cs && H)) return (int)hipErrorInvalidValue;
  if (T == 0) return 0;
  const long rows = H + 2l * Hkv, wgs = (rows * (D == 64 ? 8 : 16) + 255) / 256;
  if (wgs > 65535) return (int)hipErrorInvalidValue;
  Write4 p{(bf16_t*)q, (bf16_t*)k, (bf16_t*)v, ldk, ldv, T, H, D, npos, (const int*)slot, (const int*)at, (const int*)pos,
           (const float*)cs, (float*)weight, {(uint8_t*)ck, (uint8_t*)cks, (uint8_t*)cv, (uint8_t*)cvs, slots, Hkv, max_seq}};
  cache4_write_kernel<<<dim3((T + W4_T - 1) / W4_T, (unsigned)wgs), 256, 0, (hipStream_t)stream>>>(p);
  DA_LAUNCH_CHECK();
}

DA_EXPORT int da_cache4_read(void* ck, void* cks, void* cv, void* cvs, int Hkv, int D, int slots, int max_seq, int slot, int n,
                             void* k, void* v, void* stream) {
  if (D % 32 || D < 32 || D > 128 || slot < 0 || slot >= slots || n < 0 || n > max_seq) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  const long items = 2l * Hkv * n * (D / 8);
  if ((items + 255) / 256 > 0x7fffffffl) return (int)hipErrorInvalidValue;
  cache4_read_kernel<<<(unsigned)((items + 255) / 256), 256, 0, (hipStream_t)stream>>>(
      {(uint8_t*)ck, (uint8_t*)cks, (uint8_t*)cv, (uint8_t*)cvs, slots, Hkv, max_seq}, slot, n, D, (bf16_t*)k, (bf16_t*)v);
  DA_LAUNCH_CHECK();
}

// ------------------------------------------------------------------------------------------- attention
// One new token a sequence. The G query heads of a KV head are the columns of the products (16, zeros behind G): per 16 keys
//   S^T[key][g] = K Q^T     A: lane (c, f) has chunks f CH .. f CH + CH - 1 of 8 elements (CH = D / 32 steps) of row c, which
//                           is key 4 (c & 3) + (c >> 2)
// so that lane (g, f) has the scores of keys 4 i + f (i = 0 .. 3), and per 32 keys
//   O^T[d][g] += V^T P^T    B: P^T straight from S^T's registers; A: lane (c, f) has the D / 16 elements (D / 16) c .. of those
//                           8 keys, as bytes of two elements, and row c of tile i is element (D / 16) c + i
// The order in which a product takes its elements and keys is that of the bytes in memory: nothing is transposed, and the
// keys' order spreads a wave's reads of V over all LDS banks.
// The weights P keep 16 bits, in two pieces of 8: where there are places (G <= 8) a head has two columns, whose lanes have the same
// scores and take a piece each; with more heads the second piece has a product of its own. Pieces' outputs and sums are added in fp32.
// In 8 bits weights were off by up to 2^-8 of sum p |v|, as much as the output's own rounding; a third column leaves nothing, at one
// percent of the time more (64 x 8192 keys: 80.1 us in 8 bits, 81.8 in 16, 82.6 in 24).
// A wave walks 64 keys at a time, copied by LDS-DMA (1 KiB an instruction, rows past the end are zeros) into two places of its
// own, K's and V's: a place is filled again as soon as its codes are in registers, with counted waits and no barrier.
struct Attn4 {
  const bf16_t* q;
  int ldq;
  Cache4 c;
  const int *lens, *slot, *pre;
  int B, H, max_len, nsplit, keys, ldo;
  float scale_log2e;
  float *po, *pm, *pl;  // of the splits
  float* sc;            // scores [B, H, ld_sc] (log2; 16 keys as 4 f + i for 4 i + f), or null
  int ld_sc;
  float* weight;
  bf16_t* out;
  int* cnt;  // tickets [B, Hkv], 0 between launches: the last split of a row's KV head joins them; null: another launch does
};

// A row's keys evenly over as many splits as hold `keys` of them each: splits of one size whatever the rows' lengths
__device__ __forceinline__ int splits4(const Attn4& a, int L) { return min(a.nsplit, max(1, (L + a.keys - 1) / a.keys)); }

__device__ __forceinline__ int len4(const Attn4& a, int b) {
  const int s = a.slot[b];
  return __builtin_amdgcn_readfirstlane((unsigned)s < (unsigned)a.c.slots ? max(0, min(a.lens[b], a.max_len)) : 0);
}

// What splits hand over passes the L2s of the XCDs (agent scope): no fence, only the stores' completion
__device__ __forceinline__ void put4(float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float get4(const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// One output of a head from its splits' partials, `step` of them beside each other
template <int D>
__device__ __forceinline__ void join4(const Attn4& a, long at, int act, int d, int s0, int step, float& M, float& sum, float& acc) {
  M = -INFINITY, sum = 0.f, acc = 0.f;
  constexpr int U = 12;  // splits that are joined in the launch have one round trip
  for (int s = s0; s < act; s += U * step) {
    float ms[U], ls[U], os[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int x = min(s + j * step, act - 1);
      ms[j] = s + j * step < act ? get4(a.pm + at + x) : -INFINITY;
      ls[j] = get4(a.pl + at + x);
      os[j] = get4(a.po + (at + x) * D + d);
    }
    float mx = M;
#pragma unroll
    for (int j = 0; j < U; ++j) mx = fmaxf(mx, ms[j]);
    if (mx == -INFINITY) continue;
    const float r = exp2f(M - mx);
    sum *= r;
    acc *= r;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const float e = exp2f(ms[j] - mx);
      sum += ls[j] * e;
      acc += os[j] * e;
    }
    M = mx;
  }
}

// Reads of a place in LDS as instructions of their own: ahead of an ordinary read hipcc drains the copies that are on their way
// to the other places. Each waits for itself.
template <int D>
__device__ __forceinline__ void read_k4(unsigned at, unsigned at_s, unsigned (&k)[4][D / 32], unsigned (&s)[4]) {
  if constexpr (D == 128) {
    u32x4_t x[4];
    asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:1024\n\tds_read_b128 %2, %8 offset:2048\n\t"
                 "ds_read_b128 %3, %8 offset:%10\n\tds_read_b32 %4, %9\n\tds_read_b32 %5, %9 offset:64\n\t"
                 "ds_read_b32 %6, %9 offset:128\n\tds_read_b32 %7, %9 offset:192\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
                 : "v"(at), "v"(at_s), "n"(3 * 1024) : "memory");
#pragma unroll
    for (int e = 0; e < 16; ++e) k[e >> 2][e & 3] = x[e >> 2][e & 3];
  } else if constexpr (D == 64) {
    u32x2_t x[4];
    asm volatile("ds_read_b64 %0, %8\n\tds_read_b64 %1, %8 offset:512\n\tds_read_b64 %2, %8 offset:1024\n\t"
                 "ds_read_b64 %3, %8 offset:1536\n\tds_read_b32 %4, %9\n\tds_read_b32 %5, %9 offset:64\n\t"
                 "ds_read_b32 %6, %9 offset:128\n\tds_read_b32 %7, %9 offset:192\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
                 : "v"(at), "v"(at_s) : "memory");
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e >> 1][e & 1] = x[e >> 1][e & 1];
  } else {
    asm volatile("ds_read_b32 %0, %16\n\tds_read_b32 %1, %16 offset:4\n\tds_read_b32 %2, %16 offset:8\n\t"
                 "ds_read_b32 %3, %16 offset:768\n\tds_read_b32 %4, %16 offset:772\n\tds_read_b32 %5, %16 offset:776\n\t"
                 "ds_read_b32 %6, %16 offset:1536\n\tds_read_b32 %7, %16 offset:1540\n\tds_read_b32 %8, %16 offset:1544\n\t"
                 "ds_read_b32 %9, %16 offset:2304\n\tds_read_b32 %10, %16 offset:2308\n\tds_read_b32 %11, %16 offset:2312\n\t"
                 "ds_read_b32 %12, %17\n\tds_read_b32 %13, %17 offset:64\n\tds_read_b32 %14, %17 offset:128\n\t"
                 "ds_read_b32 %15, %17 offset:192\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(k[0][0]), "=&v"(k[0][1]), "=&v"(k[0][2]), "=&v"(k[1][0]), "=&v"(k[1][1]), "=&v"(k[1][2]), "=&v"(k[2][0]),
                   "=&v"(k[2][1]), "=&v"(k[2][2]), "=&v"(k[3][0]), "=&v"(k[3][1]), "=&v"(k[3][2]), "=&v"(s[0]), "=&v"(s[1]),
                   "=&v"(s[2]), "=&v"(s[3])
                 : "v"(at), "v"(at_s) : "memory");
  }
  __builtin_amdgcn_sched_barrier(0);
}

#define A4_READ8(op, x, at, o, st)                                                                                          \
  asm volatile(op " %0, %8 offset:%9\n\t" op " %1, %8 offset:%10\n\t" op " %2, %8 offset:%11\n\t" op " %3, %8 offset:%12\n\t" \
               op " %4, %8 offset:%13\n\t" op " %5, %8 offset:%14\n\t" op " %6, %8 offset:%15\n\t" op " %7, %8 offset:%16\n\t" \
               "s_waitcnt lgkmcnt(0)"                                                                                       \
               : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])      \
               : "v"(at), "n"(o), "n"(o + 4 * st), "n"(o + 8 * st), "n"(o + 12 * st), "n"(o + 16 * st), "n"(o + 20 * st),   \
                 "n"(o + 24 * st), "n"(o + 28 * st)                                                                         \
               : "memory")

// Rows 32 HF + 4 j (+ the lane's f, in the address): slot j is key 16 (j >> 2) + 4 (j & 3) + f
template <int D, int HF>
__device__ __forceinline__ void read_v4(unsigned at, unsigned at_s, unsigned (&v)[8], unsigned (&s)[8]) {
  constexpr int RB = D / 2, O = 32 * HF * RB;
  if constexpr (D == 64) A4_READ8("ds_read_u16", v, at, O, RB);
  else A4_READ8("ds_read_b32", v, at, O, RB);
  A4_READ8("ds_read_b32", s, at_s, 128 * HF, 4);
  __builtin_amdgcn_sched_barrier(0);
}

// The upper halves of two words: floats cut off to bf16
__device__ __forceinline__ unsigned upper(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }

template <int D, bool W, bool TWO>  // TWO: two columns a head
__global__ void __launch_bounds__(256, 4) decode_attn4_kernel(Attn4 a) {
  constexpr int CH = D / 32, VB = D / 32, NT = D / 16, RB = D / 2, KT = 64;
  constexpr int ND = KT * RB / 1024, PH = ND + 1, HALF = KT * RB + KT * 4;  // DMA instructions, bytes of K or V
  typedef __attribute__((address_space(3))) void* lds_t;
  constexpr int SO = 4 * 16 * (D + 1) * 4, RING = 4 * 2 * HALF;
  __shared__ __attribute__((aligned(16))) char ring[(SO > RING ? SO : RING) + 16];
  __shared__ float sm[4][16], sl[4][16];
  __shared__ int last;
  const int hk = blockIdx.x, b = blockIdx.y, split = blockIdx.z, G = a.H / a.c.Hkv;
  const int L = len4(a, b), act = splits4(a, L);
  if (split >= act) return;
  const int chunk = ((L + act - 1) / act + KT - 1) & ~(KT - 1);
  const int kstart = split * chunk, kend = min(L, kstart + chunk);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, f = lane >> 4;
  const long own = L ? row_of(a.c, __builtin_amdgcn_readfirstlane(a.slot[b]), hk, 0) : 0;
  int P = a.pre && L ? __builtin_amdgcn_readfirstlane(a.pre[2 * b]) : 0;
  long head = own;
  if (P > 0) {
    const int s = __builtin_amdgcn_readfirstlane(a.pre[2 * b + 1]);
    if ((unsigned)s < (unsigned)a.c.slots) head = row_of(a.c, s, hk, 0);
    else P = 0;
  }
  char *const kt = ring + w * 2 * HALF, *const vt = kt + HALF;

  const bool second = TWO && c >= G;  // the column's piece of its head's weights
  const int cg = second ? c - G : c;
  const unsigned cut = second || !TWO ? 0xffff0000u : 0u;
  bf16x8_t qf[CH];
#pragma unroll
  for (int t = 0; t < CH; ++t)
    qf[t] = cg < G && a.scale_log2e != 0.f ? *(const bf16x8_t*)(a.q + (long)b * a.ldq + (hk * G + cg) * D + (f * CH + t) * 8) : bf16x8_t{0, 0, 0, 0, 0, 0, 0, 0};
  // the scale is applied behind the largest score's choice: a positive one (q takes the sign, and the 0)
  const float scale = a.scale_log2e != 0.f ? fabsf(a.scale_log2e) : 1.f;
  const short flip = a.scale_log2e < 0.f ? (short)0x8000 : (short)0;

  // K rows of 64 bytes: the 16-byte pieces of a row are exchanged by its number, so that 16 rows' pieces are in all banks
  unsigned ko[4];  // (ND of them)
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const unsigned p = i * 64 + lane;
    ko[i & 3] = D == 128 ? (p & ~3u) * 16 + (((p & 3) ^ ((p >> 4) & 3)) << 4) : p * 16;
  }
  auto issue = [&](const uint8_t* codes, const uint8_t* scales, bool swizzled, int t0, char* dst) __attribute__((always_inline)) {
    const int n = __builtin_amdgcn_readfirstlane(max(0, min(KT, kend - t0)));  // rows (none past kend)
    const long at = (t0 < P ? head : own) + t0;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(codes + at * RB), (short)0, n * RB, 0x00020000);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(scales + at * 4), (short)0, n * 4, 0x00020000);
#pragma unroll
    for (int i = 0; i < ND; ++i)  // aux 2: read once a step
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_t)(dst + i * 1024), 16, swizzled ? ko[i & 3] : (i * 64 + lane) * 16, 0, 0, 2);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_t)(dst + KT * RB), 4, lane * 4, 0, 0, 2);
  };
  // the older of K and V; the other one's copies may be on their way. What else is (scores that are stored) makes it wait for more:
  // never for less
  auto landed = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PH) : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x4_t o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  f32x4_t ol = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY;  // of the scores before their scale
  const int kr = 4 * (c & 3) + (c >> 2);  // the lane's key of 16

  issue(a.c.k, a.c.ks, true, kstart + w * KT, kt);
  issue(a.c.v, a.c.vs, false, kstart + w * KT, vt);
#pragma unroll
  for (int t = 0; t < CH; ++t) {
    qf[t] ^= bf16x8_t{flip, flip, flip, flip, flip, flip, flip, flip};
    asm volatile("" : "+v"(qf[t]));
  }
  for (int t0 = kstart + w * KT; t0 < kend; t0 += 4 * KT) {
    landed();
    unsigned kw[4][CH], ks[4];
    const unsigned kt_at = (unsigned)(size_t)(lds_t)kt;
    read_k4<D>(kt_at + kr * RB + (D == 128 ? ((f ^ (c & 3)) << 4) : f * CH * 4), kt_at + KT * RB + kr * 4, kw, ks);
    issue(a.c.k, a.c.ks, true, t0 + 4 * KT, kt);
    f32x4_t s[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      s[tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < CH; ++t) {
        const float sc = scale_of(ks[tt], (f * CH + t) >> 2);
        const u32x4_t kk = {bf2_of4<0>(kw[tt][t], sc), bf2_of4<1>(kw[tt][t], sc), bf2_of4<2>(kw[tt][t], sc), bf2_of4<3>(kw[tt][t], sc)};
        s[tt] = mfma16(__builtin_bit_cast(bf16x8_t, kk), qf[t], s[tt]);
      }
    }
    float mx = -INFINITY;
    const bool whole = t0 + KT <= kend;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!whole && t0 + 16 * tt + 4 * i + f >= kend) s[tt][i] = -INFINITY;
        mx = fmaxf(mx, s[tt][i]);
      }
    if (W && c < G) {
      float* to = a.sc + ((long)b * a.H + hk * G + c) * a.ld_sc + t0 + 4 * f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) *(f32x4_t*)(to + 16 * tt) = s[tt] * scale;
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = max_xhalf(mx);
    if (__ballot(mx > m)) {  // (a new maximum is rare after the first tiles)
      const float mn = fmaxf(m, mx), alpha = exp2f((m - (mn == -INFINITY ? 0.f : mn)) * scale);
      m = mn;
      ol *= alpha;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= alpha;
    }
    const float use = m == -INFINITY ? 0.f : m * scale;
    unsigned pw[8], rest[TWO ? 1 : 8];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[tt][i] = __builtin_amdgcn_exp2f(fmaf(s[tt][i], scale, -use));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned first = upper(s[tt][2 * h], s[tt][2 * h + 1]);
        const float r0 = s[tt][2 * h] - __uint_as_float((first << 16) & cut), r1 = s[tt][2 * h + 1] - __uint_as_float(first & cut);
        pw[2 * tt + h] = TWO ? upper(r0, r1) : first;
        if constexpr (!TWO) rest[2 * tt + h] = upper(r0, r1);
      }
    }
    landed();
    const unsigned vt_at = (unsigned)(size_t)(lds_t)vt;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      unsigned word[8], vs[8];
      const unsigned v_at = vt_at + f * RB + c * VB, s_at = vt_at + KT * RB + f * 4;
      if (hf) {
        read_v4<D, 1>(v_at, s_at, word, vs);
        issue(a.c.v, a.c.vs, false, t0 + 4 * KT, vt);
      } else {
        read_v4<D, 0>(v_at, s_at, word, vs);
      }
      unsigned vv[8][VB];  // pairs of elements of 8 keys
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        vv[j][0] = bf2_of4<0>(word[j], scale_of(vs[j], (c * NT) >> 5));
        vv[j][1] = bf2_of4<1>(word[j], scale_of(vs[j], (c * NT + 2) >> 5));
        if constexpr (VB > 2) vv[j][2] = bf2_of4<2>(word[j], scale_of(vs[j], (c * NT + 4) >> 5));
        if constexpr (VB > 3) vv[j][3] = bf2_of4<3>(word[j], scale_of(vs[j], (c * NT + 6) >> 5));
      }
      const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, u32x4_t{pw[4 * hf], pw[4 * hf + 1], pw[4 * hf + 2], pw[4 * hf + 3]});
      // the weights' sum as a product with ones: of the pieces that V meets
      constexpr bf16x8_t ones = {0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80};
      ol = mfma16(ones, pb, ol);
      bf16x8_t pr;
      if constexpr (!TWO) {
        pr = __builtin_bit_cast(bf16x8_t, u32x4_t{rest[4 * hf], rest[4 * hf + 1], rest[4 * hf + 2], rest[4 * hf + 3]});
        ol = mfma16(ones, pr, ol);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        u32x4_t va;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          va[e] = __builtin_amdgcn_perm(vv[2 * e + 1][i >> 1], vv[2 * e][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
        o[i] = mfma16(__builtin_bit_cast(bf16x8_t, va), pb, o[i]);
        if constexpr (!TWO) o[i] = mfma16(__builtin_bit_cast(bf16x8_t, va), pr, o[i]);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (pieces past the end write zeros)
  if (f == 0) {
    sm[w][c] = m * scale;
    sl[w][c] = ol[0];
  }
  __syncthreads();  // every wave is done with its places
  float* so = (float*)ring;  // [4][16][D + 1]
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) so[(w * 16 + c) * (D + 1) + NT * (4 * f + r) + i] = o[i][r];
  __syncthreads();
  for (int i = tid; i < G * D; i += 256) {
    const int g = i / D, d = i - g * D;
    const float M = fmaxf(fmaxf(sm[0][g], sm[1][g]), fmaxf(sm[2][g], sm[3][g])), use = M == -INFINITY ? 0.f : M;
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int ww = 0; ww < 4; ++ww) {
      const float e = exp2f(sm[ww][g] - use);
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int j = TWO; j >= 0; --j) {
        x += so[(ww * 16 + g + j * G) * (D + 1) + d];
        y += sl[ww][g + j * G];
      }
      acc += x * e;
      sum += y * e;
    }
    const long at = ((long)b * a.H + hk * G + g) * a.nsplit + split;
    if (act == 1) a.out[(long)b * a.ldo + (hk * G + g) * D + d] = f2bf(L ? acc / sum : 0.f);
    else put4(a.po + at * D + d, acc);
    if (d == 0) {
      put4(a.pm + at, M);
      put4(a.pl + at, sum);
    }
  }
  if (act == 1 || !a.cnt) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    int* t = a.cnt + b * a.c.Hkv + hk;
    last = __hip_atomic_fetch_add(t, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == act - 1;
    if (last) __hip_atomic_store(t, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last) return;
  for (int i = tid; i < G * D; i += 256) {
    const int g = i / D, d = i - g * D;
    float M, sum, acc;
    join4<D>(a, ((long)b * a.H + hk * G + g) * a.nsplit, act, d, 0, 1, M, sum, acc);
    a.out[(long)b * a.ldo + (hk * G + g) * D + d] = f2bf(acc / sum);
  }
}

// The second launch of many splits or of weights: workgroup x < G of a row's KV head joins the splits of its head x, the others
// add the weights of 1024 keys each.
template <int D>
__global__ void __launch_bounds__(256) decode_attn4_join_kernel(Attn4 a) {
  __shared__ float sM[16], sR[16], part[3][4][D];
  const int hk = blockIdx.y, b = blockIdx.z, G = a.H / a.c.Hkv, tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int L = len4(a, b), act = splits4(a, L);
  const long first = ((long)b * a.H + hk * G) * a.nsplit;
  if ((int)blockIdx.x < G) {
    if (act == 1) return;
    const int g = blockIdx.x;
    for (int d = lane; d < D; d += 64) join4<D>(a, first + (long)g * a.nsplit, act, d, w, 4, part[0][w][d], part[1][w][d], part[2][w][d]);
    __syncthreads();
    if (tid < D) {
      const float M = fmaxf(fmaxf(part[0][0][tid], part[0][1][tid]), fmaxf(part[0][2][tid], part[0][3][tid]));
      float sum = 0.f, acc = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = exp2f(part[0][i][tid] - M);
        sum += part[1][i][tid] * e;
        acc += part[2][i][tid] * e;
      }
      a.out[(long)b * a.ldo + (hk * G + g) * D + tid] = f2bf(acc / sum);
    }
    return;
  }
  const int k0 = ((int)blockIdx.x - G) * 1024;
  if (k0 >= L) return;
  // 4 keys a thread: places 4 f + i of 16 are keys 4 i + f. The scores of 4 heads are on their way beside the sums of the splits
  const int at = k0 + 4 * tid, key = (at & ~15) + ((at >> 2) & 3);
  const bool in = key < L;
  const float* sc = a.sc + ((long)b * a.H + hk * G) * a.ld_sc + at;
  f32x4_t s[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) s[g] = in ? *(const f32x4_t*)(sc + (long)min(g, G - 1) * a.ld_sc) : f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int g = tid >> 4; g < G; g += 16) {  // 16 lanes a head
    float M = -INFINITY, sum = 0.f;
    for (int x = tid & 15; x < act; x += 16) {
      const float m = a.pm[first + (long)g * a.nsplit + x], l = a.pl[first + (long)g * a.nsplit + x], mx = fmaxf(M, m);
      sum = sum * exp2f(M - mx) + l * exp2f(m - mx);
      M = mx;
    }
    const float mine = M;
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 16));
    sum *= exp2f(mine - M);
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 16);
    if ((tid & 15) == 0) { sM[g] = M; sR[g] = 1.f / sum; }
  }
  __syncthreads();
  if (!in) return;
  f32x4_t p = {0.f, 0.f, 0.f, 0.f};
  for (int g0 = 0; g0 < G; g0 += 4) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (g0) s[g] = *(const f32x4_t*)(sc + (long)min(g0 + g, G - 1) * a.ld_sc);
      if (g0 + g < G)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] += exp2f(s[g][i] - sM[g0 + g]) * sR[g0 + g];
    }
  }
  float* wt = a.weight + row_of(a.c, a.slot[b], hk, key);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (key + 4 * i < L) wt[4 * i] += p[i];
}

DA_EXPORT size_t da_decode_attn4_ws(int B, int H, int D, int max_len, int nsplit, int weight) {
  return 4 * ((size_t)B * H * ((nsplit * (D + 2) + 3) / 4 * 4) + (weight ? (size_t)B * H * ((max_len + 63) / 64 * 64) : 0));
}

template <int D>
static int attn4(Attn4& a, hipStream_t st) {
  const dim3 grid(a.c.Hkv, a.B, a.nsplit);
  const bool two = a.H / a.c.Hkv <= 8;
  if (a.weight) {
    if (two) decode_attn4_kernel<D, true, true><<<grid, 256, 0, st>>>(a);
    else decode_attn4_kernel<D, true, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (two) decode_attn4_kernel<D, false, true><<<grid, 256, 0, st>>>(a);
    else decode_attn4_kernel<D, false, false><<<grid, 256, 0, st>>>(a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (a.weight || (a.nsplit > 1 && !a.cnt))
    decode_attn4_join_kernel<D><<<dim3(a.H / a.c.Hkv + (a.weight ? (a.max_len + 1023) / 1024 : 0), a.c.Hkv, a.B), 256, 0, st>>>(a);
  DA_LAUNCH_CHECK();
}

// counters (ints, B * Hkv of them, 0): the splits are joined in the launch; null (always with weights): in a second one
DA_EXPORT int da_decode_attn4(const void* q, int ldq, void* ck, void* cks, void* cv, void* cvs, const void* lens, const void* slot,
                              const void* pre, int B, int H, int Hkv, int D, int slots, int max_seq, int max_len, int nsplit,
                              int keys, float scale, void* ws, void* weight, void* out, int ldo, void* counters, void* stream) {
  if (Hkv < 1 || H % Hkv || H / Hkv > 16 || max_len < 1 || max_len > max_seq || nsplit < 1 || nsplit > 65535 || keys < 1 || B > 65535) return (int)hipErrorInvalidValue;
  if (B == 0) return 0;
  const size_t n = (size_t)B * H * nsplit, all = (size_t)B * H * ((nsplit * (D + 2) + 3) / 4 * 4);
  Attn4 a{(const bf16_t*)q, ldq, {(uint8_t*)ck, (uint8_t*)cks, (uint8_t*)cv, (uint8_t*)cvs, slots, Hkv, max_seq},
          (const int*)lens, (const int*)slot, (const int*)pre, B, H, max_len, nsplit, keys, ldo, scale * 1.44269504f,
          (float*)ws, (float*)ws + n * D, (float*)ws + n * (D + 1), weight ? (float*)ws + all : nullptr,
          (max_len + 63) / 64 * 64, (float*)weight, (bf16_t*)out, weight ? nullptr : (int*)counters};
  hipStream_t st = (hipStream_t)stream;
  return D == 64 ? attn4<64>(a, st) : D == 96 ? attn4<96>(a, st) : D == 128 ? attn4<128>(a, st) : (int)hipErrorInvalidValue;
}

// ------------------------------------------------------------------------------------------- eviction
// Of the n keys of a sequence that is too long a KV head keeps the `recent` last ones and of the others the keep - recent of largest weight
// (equal ones: the earlier), in their order, at the front of its slot or of another. A workgroup per (KV head, row, layer):
//   select  the smallest kept weight as a 32-bit key whose order is the weight's, 11 bits a pass, counted in LDS
//   list    of 4096 keys at a time the kept ones', by votes of 64 and two sums over the workgroup's waves
//   move    their rows, 512 or so at a time, in pieces of 16 bytes. A row moves to the front of where it was or stays: what a step
//           writes, no later step reads, so the next step's rows are on their way while a step's are written, with one barrier.
// Bound by memory: 12 sequences of 8192 keys to 4096, 8 heads x 128, four layers (452 MB read and written) 110 us, of which 14 go
// by before the first row is moved (its weights asked for ahead of the selection: the same); 700 keys to 500, 8 heads x 64, two
// layers 9 us, latencies of the four steps one after the other.
struct Evict4 {
  Cache4 c;
  float* weight;
  const int *lens, *slot, *to;
  int* out;
  int keep, recent, above;  // sequences of more than `above` keys are shortened to `keep`
  long layer;  // rows of a layer
};

__device__ __forceinline__ unsigned order_key(float x) {  // NaN lowest, -0 as +0
  const unsigned u = __float_as_uint(x + 0.f);
  return x != x ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

typedef unsigned long long u64;
constexpr int EV_T = 512, EV_LIST = 8 * EV_T;

// before the thread's own, over the workgroup's 8 waves; `all` of them
__device__ __forceinline__ int scan8(int x, int* red, int& all) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int y = wave_scan(x);
  __syncthreads();
  if (lane == 63) red[wv] = y;
  __syncthreads();
  int off = 0;
  all = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    off += q < wv ? red[q] : 0;
    all += red[q];
  }
  return off + y - x;
}

struct Small { unsigned ks, vs, w; };  // a row's scales and weight
__device__ __forceinline__ void arrived(u32x4_t& x) { asm volatile("" : "+v"(x)); }  // (waits for its load)
__device__ __forceinline__ void arrived(Small& x) { asm volatile("" : "+v"(x.ks), "+v"(x.vs), "+v"(x.w)); }

// Items 0 .. items - 1 from load(i, x) to store(i, x), EV_T U of them a step
template <int U, typename T, typename Load, typename Store>
__device__ __forceinline__ void move_rows(int items, Load load, Store store) {
  T now[U] = {}, next[U] = {};
#pragma unroll
  for (int e = 0; e < U; ++e) load((int)threadIdx.x + EV_T * e, now[e]);
  for (int i0 = 0; i0 < items; i0 += EV_T * U) {
#pragma unroll
    for (int e = 0; e < U; ++e) load(i0 + EV_T * U + (int)threadIdx.x + EV_T * e, next[e]);
#pragma unroll
    for (int e = 0; e < U; ++e) arrived(now[e]);
    __syncthreads();  // the whole step is in registers
#pragma unroll
    for (int e = 0; e < U; ++e) {
      store(i0 + (int)threadIdx.x + EV_T * e, now[e]);
      now[e] = next[e];
    }
  }
}

template <int D>
__global__ void __launch_bounds__(EV_T) cache4_evict_kernel(Evict4 p) {
  constexpr int NP = D / 32, RP = 2 * NP;  // 16-byte pieces of a row's codes, of keys and values
  __shared__ int hist[2048], red[2][8], sel[2];
  __shared__ unsigned short list[EV_LIST];
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int s = p.slot[b], d = p.to[b];
  const int n = (unsigned)s < (unsigned)p.c.slots && (unsigned)d < (unsigned)p.c.slots ? max(0, min(p.lens[b], p.c.max_seq)) : 0;
  const int keep = n > p.above ? min(n, p.keep) : n;
  if (blockIdx.z == 0 && hk == 0 && tid == 0) p.out[b] = keep;
  if (keep == 0 || (keep == n && s == d)) return;
  const long from = blockIdx.z * p.layer + row_of(p.c, s, hk, 0), to = blockIdx.z * p.layer + row_of(p.c, d, hk, 0);
  const float* wt = p.weight + from;
  const int m = n > keep ? n - p.recent : 0;  // keys that have to earn their place (0: all are kept)
  const int lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned cut = 0xffffffffu;
  int ties = 0;
  if (m && keep > p.recent) {
    int need = keep - p.recent;
    cut = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int sh = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11, bins = 1 << bits;
      for (int i = tid; i < 2048; i += EV_T) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < m; i += EV_T * 4) {  // loads on their way together
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = wt[min(i + EV_T * e, m - 1)];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned k = order_key(y[e]);
          if (i + EV_T * e < m && (pass == 0 || (k >> (sh + bits)) == (cut >> (sh + bits)))) atomicAdd(&hist[(k >> sh) & (bins - 1)], 1);
        }
      }
      __syncthreads();
      int v[4], mine = 0, all;  // from the largest down: 4 bins a thread
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += v[e] = hist[2047 - 4 * tid - e];
      int before = scan8(mine, red[0], all);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (before < need && before + v[e] >= need) {
          sel[0] = 2047 - 4 * tid - e;
          sel[1] = need - before;
        }
        before += v[e];
      }
      __syncthreads();
      cut |= (unsigned)sel[0] << sh;
      need = sel[1];
    }
    ties = need;
  }
  int done = 0, tied = 0;  // keys kept, keys equal to the cut so far
  const u64 lower = (1ull << lane) - 1;
  for (int t0 = 0; t0 < n; t0 += EV_LIST) {
    const int i0 = t0 + 512 * wv + lane;  // a wave's 8 times 64 keys
    unsigned k[8];
    u64 equal[8], kept[8];
    int ties_of = 0, kept_of = 0, cnt = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] = i0 + 64 * e < m ? order_key(wt[i0 + 64 * e]) : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      equal[e] = __ballot(i0 + 64 * e < m && k[e] == cut);
      ties_of += __popcll(equal[e]);
    }
    if (lane == 0) red[0][wv] = ties_of;
    __syncthreads();
    int before = tied;  // ties before the wave's
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      before += q < wv ? red[0][q] : 0;
      tied += red[0][q];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = i0 + 64 * e;
      kept[e] = __ballot(i < n && (i >= m || k[e] > cut || (k[e] == cut && before + __popcll(equal[e] & lower) < ties)));
      before += __popcll(equal[e]);
      kept_of += __popcll(kept[e]);
    }
    if (lane == 0) red[1][wv] = kept_of;
    __syncthreads();
    int at = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      at += q < wv ? red[1][q] : 0;
      cnt += red[1][q];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (kept[e] >> lane & 1) list[at + __popcll(kept[e] & lower)] = (unsigned short)(i0 - t0 + 64 * e);
      at += __popcll(kept[e]);
    }
    __syncthreads();
    const long src = from + t0, dst = to + done;
    auto codes = [&](int i, long row) {
      const int q = i % RP;
      return (u32x4_t*)((q < NP ? p.c.k : p.c.v) + row * (D / 2) + (q < NP ? q : q - NP) * 16);
    };
    move_rows<4, u32x4_t>(
        cnt * RP, [&](int i, u32x4_t& x) { if (i < cnt * RP) x = __builtin_nontemporal_load(codes(i, src + list[i / RP])); },
        [&](int i, const u32x4_t& x) { if (i < cnt * RP) __builtin_nontemporal_store(x, codes(i, dst + i / RP)); });
    move_rows<1, Small>(
        cnt,
        [&](int i, Small& x) {
          if (i >= cnt) return;
          const long row = src + list[i];
          x = {*(const unsigned*)(p.c.ks + row * 4), *(const unsigned*)(p.c.vs + row * 4), __float_as_uint(p.weight[row])};
        },
        [&](int i, const Small& x) {
          if (i >= cnt) return;
          *(unsigned*)(p.c.ks + (dst + i) * 4) = x.ks;
          *(unsigned*)(p.c.vs + (dst + i) * 4) = x.vs;
          p.weight[dst + i] = __uint_as_float(x.w);
        });
    done += cnt;
    __syncthreads();  // the list is written again
  }
}

DA_EXPORT int da_cache4_evict(void* ck, void* cks, void* cv, void* cvs, void* weight, const void* lens, const void* slot,
                              const void* to, void* out, int layers, int B, int Hkv, int D, int slots, int max_seq, int keep,
                              int recent, int above, void* stream) {
  if (D % 32 || D < 64 || D > 128 || keep < 0 || recent < 0 || recent > keep || above < keep || B > 65535 || layers > 65535) return (int)hipErrorInvalidValue;
  if (B == 0 || layers == 0) return 0;
  Evict4 p{{(uint8_t*)ck, (uint8_t*)cks, (uint8_t*)cv, (uint8_t*)cvs, slots, Hkv, max_seq}, (float*)weight, (const int*)lens,
           (const int*)slot, (const int*)to, (int*)out, keep, recent, above, (long)slots * Hkv * max_seq};
  const dim3 grid(Hkv, B, layers);
  hipStream_t st = (hipStream_t)stream;
  if (D == 64) cache4_evict_kernel<64><<<grid, EV_T, 0, st>>>(p);
  else if (D == 96) cache4_evict_kernel<96><<<grid, EV_T, 0, st>>>(p);
  else cache4_evict_kernel<128><<<grid, EV_T, 0, st>>>(p);
  DA_LAUNCH_CHECK();
}
