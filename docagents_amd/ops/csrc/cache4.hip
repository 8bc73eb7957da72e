// A key / value cache held in 4 bits: its write (RoPE inside or not), its read, attention of one new token a sequence over
// it, and the eviction of the keys of least weight.
//
// Format: codes [slots, Hkv, max_seq, D / 2] (element 2 j in the low half of byte j), a code a sign and one of the magnitudes
// 0, .5, 1, 1.5, 2, 3, 4, 6 (e2m1), and a scale for 32 elements along the head: 2^(byte - 127), [slots, Hkv, max_seq, 4] bytes
// of which D / 32 are used; 255: the block held an inf or a NaN and reads as NaN. Power-of-two scales: a value is exact in
// bf16, one conversion instruction makes two of them, and both products run on bf16 MFMA. Rows are whole and in order, so that
// a token is written, read and moved by itself. 136 bytes a key and KV head of 128 for 512 in bf16.
// Scale of a block with largest magnitude a = m 2^e (1 <= m < 2): 2^(e - 2) for m < 1.75 and 2^(e - 1) above it (6 stands for
// up to 7 then): root mean square error 11.2 % of normal values, 11.5 % if the step is at m = 2 or 1.5.
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

__device__ __forceinline__ float scale_of(unsigned bytes, int at) {
  const unsigned s = (bytes >> (8 * at)) & 255;
  return __uint_as_float(s == 255 ? 0x7fc00000u : s << 23);
}

__device__ __forceinline__ long row_of(const Cache4& c, int slot, int h, int at) {
  return ((long)slot * c.Hkv + h) * c.max_seq + at;
}

// ------------------------------------------------------------------------------------------- write, read
// 8 consecutive elements a lane, 4 lanes a block; x as bf16 pairs. Returns the codes; the block's scale byte in `sb`.
__device__ __forceinline__ unsigned encode8(const u32x4_t& x, unsigned& sb) {
  unsigned a = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) a = max(a, max((x[e] << 16) & 0x7fffffffu, x[e] & 0x7fff0000u));
  a = max(a, (unsigned)__shfl_xor((int)a, 1, 64));
  a = max(a, (unsigned)__shfl_xor((int)a, 2, 64));
  sb = (unsigned)max(1, (int)((a + 0x200000u) >> 23) - 2);
  const bool bad = (a >> 23) >= 255;
  const float up = __uint_as_float((254u - sb) << 23);
  unsigned r = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned w = e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16;
    const float y = fabsf(__uint_as_float(w) * up);
    const unsigned code = (y > 0.25f) + (y >= 0.75f) + (y > 1.25f) + (y >= 1.75f) + (y > 2.5f) + (y >= 3.5f) + (y > 5.f);
    r |= (code | ((w >> 31) << 3)) << (4 * e);
  }
  if (bad) { sb = 255; r = 0; }
  return r;
}

struct Write4 {
  bf16_t *q, *k, *v;  // rows of T tokens; q only with cs
  int ldk, ldv, T, H, D;
  const int *slot, *at, *pos;
  const float* cs;
  float* weight;
  Cache4 c;
};

// A lane per 8 elements. With cs the heads of q and k are rotated in place first (rope_cache's arithmetic, its bits).
__global__ void __launch_bounds__(256) cache4_write_kernel(Write4 p) {
  const int ch = p.D / 8, heads = p.H + 2 * p.c.Hkv;
  const long item = (long)blockIdx.x * 256 + threadIdx.x;
  const int t = (int)(item / (heads * ch)), r = (int)(item - (long)t * heads * ch);
  if (t >= p.T) return;  // (whole blocks: a token has a multiple of 4 items)
  const int hh = r / ch, c = r - hh * ch;
  const bool is_q = hh < p.H, is_k = !is_q && hh < p.H + p.c.Hkv;
  const int h = is_q ? hh : is_k ? hh - p.H : hh - p.H - p.c.Hkv;
  bf16_t* src = (is_q ? p.q + (long)t * p.ldk : is_k ? p.k + (long)t * p.ldk : p.v + (long)t * p.ldv) + h * p.D + c * 8;
  u32x4_t x = *(const u32x4_t*)src;
  if (p.cs && (is_q || is_k)) {
    const float* f = p.cs + ((long)p.pos[t] * (p.D / 2) + c * 4) * 2;
    const f32x4_t c01 = *(const f32x4_t*)f, c23 = *(const f32x4_t*)(f + 4);
    const float cc[4] = {c01[0], c01[2], c23[0], c23[2]}, sn[4] = {c01[1], c01[3], c23[1], c23[3]};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x1 = bf2f(x[e] & 0xffff), x2 = bf2f(x[e] >> 16);
      x[e] = pack_bf2(fmaf(x1, cc[e], -(x2 * sn[e])), fmaf(x2, cc[e], x1 * sn[e]));
    }
    *(u32x4_t*)src = x;
  }
  if (is_q) return;
  unsigned sb;
  const unsigned codes = encode8(x, sb);
  const int s = p.slot[t], at = p.at[t];
  if ((unsigned)s >= (unsigned)p.c.slots || (unsigned)at >= (unsigned)p.c.max_seq) return;
  const long row = row_of(p.c, s, h, at);
  *(unsigned*)((is_k ? p.c.k : p.c.v) + row * (p.D / 2) + c * 4) = codes;
  if ((c & 3) == 0) (is_k ? p.c.ks : p.c.vs)[row * 4 + (c >> 2)] = (uint8_t)sb;
  if (p.weight && is_k && c == 0) p.weight[row] = 0.f;
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
                              const void* cs, void* ck, void* cks, void* cv, void* cvs, void* weight, int T, int H, int Hkv,
                              int D, int slots, int max_seq, void* stream) {
  if (D % 32 || D < 32 || D > 128 || (cs && (!pos || !q)) || (!cs && H)) return (int)hipErrorInvalidValue;
  if (T == 0) return 0;
  const long items = (long)T * (H + 2 * Hkv) * (D / 8);
  if ((items + 255) / 256 > 0x7fffffffl) return (int)hipErrorInvalidValue;
  Write4 p{(bf16_t*)q, (bf16_t*)k, (bf16_t*)v, ldk, ldv, T, H, D, (const int*)slot, (const int*)at, (const int*)pos,
           (const float*)cs, (float*)weight, {(uint8_t*)ck, (uint8_t*)cks, (uint8_t*)cv, (uint8_t*)cvs, slots, Hkv, max_seq}};
  cache4_write_kernel<<<(unsigned)((items + 255) / 256), 256, 0, (hipStream_t)stream>>>(p);
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
// One new token a sequence. The G query heads of a KV head are the columns of the products (16, zeros behind G): per 32 keys
//   S^T[key][g] = K Q^T     A: lane (c, f) has key c and its chunks of 8 elements f CH .. f CH + CH - 1 (CH = D / 32 steps)
//   O^T[d][g] += V^T P^T    B: P^T straight from S^T's registers (slot j of lane group f is key 16 (j >> 2) + 4 f + (j & 3));
//                           A: lane (c, f) has the D / 16 elements (D / 16) c .. of those 8 keys, as bytes of two elements,
//                           and row c of tile i is element (D / 16) c + i
// so that the order in which a product takes its elements and keys is that of the bytes in memory and nothing is transposed.
struct Attn4 {
  const bf16_t* q;
  int ldq;
  Cache4 c;
  const int *lens, *slot, *pre;
  int B, H, max_len, nsplit, ldo;
  float scale_log2e;
  float *po, *pm, *pl;  // of the splits
  float* sc;            // scores [B, H, ld_sc] (log2), or null
  int ld_sc;
  float* weight;
  bf16_t* out;
};

constexpr int A4_KEYS = 256;  // keys that a split takes at least

__device__ __forceinline__ int splits4(int L, int nsplit) { return min(nsplit, max(1, (L + A4_KEYS - 1) / A4_KEYS)); }

__device__ __forceinline__ int len4(const Attn4& a, int b) {
  const int s = a.slot[b];
  return (unsigned)s < (unsigned)a.c.slots ? max(0, min(a.lens[b], a.max_len)) : 0;
}

template <int D>
__global__ void __launch_bounds__(256, 2) decode_attn4_kernel(Attn4 a) {
  constexpr int CH = D / 32, VB = D / 32, NT = D / 16;
  __shared__ float so[4][16][D + 1], sm[4][16], sl[4][16];
  const int split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, G = a.H / a.c.Hkv;
  const int L = len4(a, b), act = splits4(L, a.nsplit);
  if (split >= act) return;
  const int chunk = ((L + act - 1) / act + 127) & ~127;
  const int kstart = split * chunk, kend = min(L, kstart + chunk);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 15, f = lane >> 4;
  const long own = L ? row_of(a.c, a.slot[b], hk, 0) : 0;
  const int P = a.pre && L ? a.pre[2 * b] : 0;
  const long head = P ? row_of(a.c, a.pre[2 * b + 1], hk, 0) : own;

  bf16x8_t qf[CH];
#pragma unroll
  for (int t = 0; t < CH; ++t)
    qf[t] = c < G ? *(const bf16x8_t*)(a.q + (long)b * a.ldq + (hk * G + c) * D + (f * CH + t) * 8) : bf16x8_t{0, 0, 0, 0, 0, 0, 0, 0};
  f32x4_t o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  for (int t0 = kstart + 32 * w; t0 < kend; t0 += 128) {
    const long base = t0 < P ? head : own;
    f32x4_t s[2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const long row = base + min(t0 + 16 * tt + c, kend - 1);
      const unsigned* kp = (const unsigned*)(a.c.k + row * (D / 2)) + f * CH;
      const unsigned sb = *(const unsigned*)(a.c.ks + row * 4);
      s[tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < CH; ++t) {
        const float sc = scale_of(sb, (f * CH + t) >> 2);
        const u32x4_t kk = {bf2_of4<0>(kp[t], sc), bf2_of4<1>(kp[t], sc), bf2_of4<2>(kp[t], sc), bf2_of4<3>(kp[t], sc)};
        s[tt] = mfma16(__builtin_bit_cast(bf16x8_t, kk), qf[t], s[tt]);
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[tt][i] = t0 + 16 * tt + 4 * f + i < kend ? s[tt][i] * a.scale_log2e : -INFINITY;
        mx = fmaxf(mx, s[tt][i]);
      }
    if (a.sc && c < G) {
      float* to = a.sc + ((long)b * a.H + hk * G + c) * a.ld_sc + t0 + 4 * f;
      *(f32x4_t*)to = s[0];
      *(f32x4_t*)(to + 16) = s[1];
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = max_xhalf(mx);
    const float mn = fmaxf(m, mx), use = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m - use);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] *= alpha;
    unsigned pw[4];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[tt][i] = __builtin_amdgcn_exp2f(s[tt][i] - use);
        l += s[tt][i];
      }
      pw[2 * tt] = pack_bf2(s[tt][0], s[tt][1]);
      pw[2 * tt + 1] = pack_bf2(s[tt][2], s[tt][3]);
    }
    const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, u32x4_t{pw[0], pw[1], pw[2], pw[3]});
    unsigned vv[8][VB];  // pairs of elements of 8 keys
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const long row = base + min(t0 + 16 * (j >> 2) + 4 * f + (j & 3), kend - 1);
      const uint8_t* vp = a.c.v + row * (D / 2) + c * VB;
      const unsigned sb = *(const unsigned*)(a.c.vs + row * 4);
      unsigned word = 0;
      __builtin_memcpy(&word, vp, VB);
      vv[j][0] = bf2_of4<0>(word, scale_of(sb, (c * NT) >> 5));
      vv[j][1] = bf2_of4<1>(word, scale_of(sb, (c * NT + 2) >> 5));
      if constexpr (VB > 2) vv[j][2] = bf2_of4<2>(word, scale_of(sb, (c * NT + 4) >> 5));
      if constexpr (VB > 3) vv[j][3] = bf2_of4<3>(word, scale_of(sb, (c * NT + 6) >> 5));
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      u32x4_t va;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        va[e] = __builtin_amdgcn_perm(vv[2 * e + 1][i >> 1], vv[2 * e][i >> 1], i & 1 ? 0x07060302u : 0x05040100u);
      o[i] = mfma16(__builtin_bit_cast(bf16x8_t, va), pb, o[i]);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l = sum_xhalf(l);
  if (f == 0) { sm[w][c] = m; sl[w][c] = l; }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) so[w][c][NT * (4 * f + r) + i] = o[i][r];
  __syncthreads();
  for (int i = tid; i < G * D; i += 256) {
    const int g = i / D, d = i - g * D;
    const float M = fmaxf(fmaxf(sm[0][g], sm[1][g]), fmaxf(sm[2][g], sm[3][g])), use = M == -INFINITY ? 0.f : M;
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int ww = 0; ww < 4; ++ww) {
      const float e = exp2f(sm[ww][g] - use);
      acc += so[ww][g][d] * e;
      sum += sl[ww][g] * e;
    }
    const long at = ((long)b * a.H + hk * G + g) * a.nsplit + split;
    if (a.nsplit == 1) a.out[(long)b * a.ldo + (hk * G + g) * D + d] = f2bf(L ? acc / sum : 0.f);
    else a.po[at * D + d] = acc;
    if (d == 0) { a.pm[at] = M; a.pl[at] = sum; }
  }
}

// The splits of a head joined, and (weight) its share of each key's weight added: a workgroup per (1024 keys, KV head, row).
template <int D>
__global__ void __launch_bounds__(256) decode_attn4_join_kernel(Attn4 a) {
  __shared__ float sM[16], sR[16];
  const int hk = blockIdx.y, b = blockIdx.z, G = a.H / a.c.Hkv, tid = threadIdx.x;
  const int L = len4(a, b), act = splits4(L, a.nsplit);
  if (blockIdx.x && (int)blockIdx.x * 1024 >= L) return;
  if (tid < G) {
    const long at = ((long)b * a.H + hk * G + tid) * a.nsplit;
    float M = -INFINITY, sum = 0.f;
    for (int s = 0; s < act; ++s) M = fmaxf(M, a.pm[at + s]);
    for (int s = 0; s < act; ++s) sum += a.pl[at + s] * exp2f(a.pm[at + s] - (M == -INFINITY ? 0.f : M));
    sM[tid] = M == -INFINITY ? 0.f : M;
    sR[tid] = 1.f / sum;
  }
  __syncthreads();
  if (blockIdx.x == 0 && a.nsplit > 1)
    for (int i = tid; i < G * D; i += 256) {
      const int g = i / D, d = i - g * D;
      const long at = ((long)b * a.H + hk * G + g) * a.nsplit;
      float acc = 0.f;
      for (int s = 0; s < act; ++s) acc += a.po[(at + s) * D + d] * exp2f(a.pm[at + s] - sM[g]);
      a.out[(long)b * a.ldo + (hk * G + g) * D + d] = f2bf(L ? acc * sR[g] : 0.f);
    }
  if (!a.weight) return;
  float* wt = a.weight + row_of(a.c, a.slot[b], hk, 0);
  for (int key = blockIdx.x * 1024 + tid; key < min(L, (int)(blockIdx.x + 1) * 1024); key += 256) {
    float p = 0.f;
    for (int g = 0; g < G; ++g) p += exp2f(a.sc[((long)b * a.H + hk * G + g) * a.ld_sc + key] - sM[g]) * sR[g];
    wt[key] += p;
  }
}

DA_EXPORT size_t da_decode_attn4_ws(int B, int H, int D, int max_len, int nsplit, int weight) {
  return 4 * ((size_t)B * H * nsplit * (D + 2) + (weight ? (size_t)B * H * ((max_len + 31) / 32 * 32) : 0));
}

template <int D>
static int attn4(Attn4& a, hipStream_t st) {
  decode_attn4_kernel<D><<<dim3(a.nsplit, a.c.Hkv, a.B), 256, 0, st>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (a.nsplit > 1 || a.weight)
    decode_attn4_join_kernel<D><<<dim3(a.weight ? (a.max_len + 1023) / 1024 : 1, a.c.Hkv, a.B), 256, 0, st>>>(a);
  DA_LAUNCH_CHECK();
}

DA_EXPORT int da_decode_attn4(const void* q, int ldq, void* ck, void* cks, void* cv, void* cvs, const void* lens, const void* slot,
                              const void* pre, int B, int H, int Hkv, int D, int slots, int max_seq, int max_len, int nsplit,
                              float scale, void* ws, void* weight, void* out, int ldo, void* stream) {
  if (Hkv < 1 || H % Hkv || H / Hkv > 16 || max_len < 1 || max_len > max_seq || nsplit < 1 || B > 65535 || Hkv > 65535) return (int)hipErrorInvalidValue;
  if (B == 0) return 0;
  const size_t n = (size_t)B * H * nsplit;
  Attn4 a{(const bf16_t*)q, ldq, {(uint8_t*)ck, (uint8_t*)cks, (uint8_t*)cv, (uint8_t*)cvs, slots, Hkv, max_seq},
          (const int*)lens, (const int*)slot, (const int*)pre, B, H, max_len, nsplit, ldo, scale * 1.44269504f,
          (float*)ws, (float*)ws + n * D, (float*)ws + n * (D + 1), weight ? (float*)ws + n * (D + 2) : nullptr,
          (max_len + 31) / 32 * 32, (float*)weight, (bf16_t*)out};
  hipStream_t st = (hipStream_t)stream;
  return D == 64 ? attn4<64>(a, st) : D == 96 ? attn4<96>(a, st) : D == 128 ? attn4<128>(a, st) : (int)hipErrorInvalidValue;
}

// ------------------------------------------------------------------------------------------- eviction
// Of a sequence's n > keep keys a KV head keeps the `recent` last ones and of the others the keep - recent of largest weight
// (equal ones: the earlier), in their order, at the front of its slot or of another. A workgroup per (KV head, row, layer):
//   select  the smallest kept weight as a 32-bit key whose order is the weight's, 8 bits a pass, counted in LDS
//   move    1024 keys at a time: ranks by a scan over the workgroup, then rows in pieces of 16 bytes, all of a step's reads
//           before its writes (a row never moves back, so later steps read what is still there)
struct Evict4 {
  Cache4 c;
  float* weight;
  const int *lens, *slot, *to;
  int* out;
  int D, keep, recent;
  long layer;  // rows of a layer
};

__device__ __forceinline__ unsigned order_key(float x) {  // NaN lowest, -0 as +0
  const unsigned u = __float_as_uint(x + 0.f);
  return x != x ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(1024) cache4_evict_kernel(Evict4 p) {
  __shared__ int hist[256], wsum[16], src[1024], sel[2];
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int s = p.slot[b], d = p.to[b];
  const int n = (unsigned)s < (unsigned)p.c.slots && (unsigned)d < (unsigned)p.c.slots ? max(0, min(p.lens[b], p.c.max_seq)) : 0;
  const int keep = min(n, p.keep);
  if (blockIdx.z == 0 && hk == 0 && tid == 0) p.out[b] = keep;
  if (keep == n && s == d) return;
  const long from = blockIdx.z * p.layer + row_of(p.c, s, hk, 0), to = blockIdx.z * p.layer + row_of(p.c, d, hk, 0);
  const float* wt = p.weight + from;
  const int m = n > keep ? n - p.recent : 0;  // keys that have to earn their place (0: all are kept)
  unsigned cut = 0;
  int ties = 0;
  if (m) {
    int need = keep - p.recent;
    for (int sh = 24; need > 0 && sh >= 0; sh -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < m; i += 1024) {
        const unsigned k = order_key(wt[i]);
        if (sh == 24 || (k >> (sh + 8)) == (cut >> (sh + 8))) atomicAdd(&hist[(k >> sh) & 255], 1);
      }
      __syncthreads();
      if (tid < 64) {  // from the largest down: lane t has the bins 255 - 4 t .. 252 - 4 t
        int v[4], mine = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) mine += v[e] = hist[255 - 4 * lane - e];
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int u = __shfl_up(upto, o, 64);
          if (lane >= o) upto += u;
        }
        int before = upto - mine;
        if (before < need && upto >= need) {
          int e = 0;
          while (before + v[e] < need) before += v[e++];
          sel[0] = 255 - 4 * lane - e;
          sel[1] = need - before;
        }
      }
      __syncthreads();
      cut |= (unsigned)sel[0] << sh;
      need = sel[1];
      __syncthreads();
    }
    ties = need;
    if (keep == p.recent) cut = 0xffffffffu, ties = 0;
  }
  const int np = p.D / 32;  // 16-byte pieces of a row's codes
  int done = 0, tied = 0;   // keys kept, keys equal to the cut so far
  for (int t0 = 0; t0 < n; t0 += 1024) {
    const int i = t0 + tid;
    const unsigned k = i < m ? order_key(wt[i]) : 0;
    const int tie = i < m && k == cut;
    auto scan = [&](int x, int& total) {  // exclusive, over the workgroup
      int y = x;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(y, o, 64);
        if (lane >= o) y += u;
      }
      if (lane == 63) wsum[wv] = y;
      __syncthreads();
      int off = 0;
      total = 0;
      for (int q = 0; q < 16; ++q) {
        off += q < wv ? wsum[q] : 0;
        total += wsum[q];
      }
      __syncthreads();
      return off + y - x;
    };
    int all_ties, cnt;
    const int before = tied + scan(tie, all_ties);
    const int kept = i < n && (i >= m || k > cut || (tie && before < ties));
    tied += all_ties;
    const int at = scan(kept, cnt);
    if (kept) src[at] = i;
    __syncthreads();
    u32x4_t piece[8];
    const int pieces = cnt * 2 * np;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int x = tid + 1024 * e;
      if (x < pieces) {
        const int row = x / (2 * np), q = x - row * 2 * np;
        piece[e] = *(const u32x4_t*)((q < np ? p.c.k : p.c.v) + (from + src[row]) * (p.D / 2) + (q < np ? q : q - np) * 16);
      }
    }
    unsigned ks = 0, vs = 0;
    float w = 0.f;
    if (tid < cnt) {
      const long row = from + src[tid];
      ks = *(const unsigned*)(p.c.ks + row * 4);
      vs = *(const unsigned*)(p.c.vs + row * 4);
      w = p.weight[row];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int x = tid + 1024 * e;
      if (x < pieces) {
        const int row = x / (2 * np), q = x - row * 2 * np;
        *(u32x4_t*)((q < np ? p.c.k : p.c.v) + (to + done + row) * (p.D / 2) + (q < np ? q : q - np) * 16) = piece[e];
      }
    }
    if (tid < cnt) {
      const long row = to + done + tid;
      *(unsigned*)(p.c.ks + row * 4) = ks;
      *(unsigned*)(p.c.vs + row * 4) = vs;
      p.weight[row] = w;
    }
    done += cnt;
    __syncthreads();
  }
}

DA_EXPORT int da_cache4_evict(void* ck, void* cks, void* cv, void* cvs, void* weight, const void* lens, const void* slot,
                              const void* to, void* out, int layers, int B, int Hkv, int D, int slots, int max_seq, int keep,
                              int recent, void* stream) {
  if (D % 32 || D < 32 || D > 128 || keep < 0 || recent < 0 || recent > keep || B > 65535 || layers > 65535) return (int)hipErrorInvalidValue;
  if (B == 0 || layers == 0) return 0;
  Evict4 p{{(uint8_t*)ck, (uint8_t*)cks, (uint8_t*)cv, (uint8_t*)cvs, slots, Hkv, max_seq}, (float*)weight, (const int*)lens,
           (const int*)slot, (const int*)to, (int*)out, D, keep, recent, (long)slots * Hkv * max_seq};
  cache4_evict_kernel<<<dim3(Hkv, B, layers), 1024, 0, (hipStream_t)stream>>>(p);
  DA_LAUNCH_CHECK();
}
