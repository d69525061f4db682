// Block-scaled 8-bit KV cache of the serving path (ops/kv8.py): append, single-token decode attention, read-back.
//
// With one scale for every (block of T tokens, KV head) the codes follow the values' own range, so int8 or e4m3 entries
// need no calibration.  A block is quantised once, when it is full, from its bf16 rows:
//   scale = max(amax / QMAX, 2^-126),   code = round(x * (1 / scale)),   QMAX = 127 (int8) / 448 (e4m3)
// and the block that is still open stays in bf16, so what the cache holds after n tokens does not depend on how they
// were grouped into appends.  A block with an entry that is not finite gets the scale NaN and reads back as NaN.
#include <algorithm>
#include <type_traits>

#include "dph_common.h"
#include "kernels.h"

namespace dph {

namespace {

constexpr float kTinyScale = 1.17549435e-38f;   // 2^-126: keeps 1 / scale finite for blocks of zeros

// fp32 -> nearest 8-bit codes of four values already divided by the scale, packed
template <bool E4M3>
__device__ __forceinline__ unsigned pack4(const float (&q)[4]) {
  if constexpr (E4M3) {
    float c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = __builtin_amdgcn_fmed3f(q[j], 448.f, -448.f);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false),
                                                     true);
  } else {
    unsigned r = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int v = (int)__builtin_amdgcn_fmed3f(rintf(q[j]), 127.f, -127.f);
      r |= ((unsigned)v & 0xffu) << (8 * j);
    }
    return r;
  }
}

// byte e, signed: shifts of 32 bits fold into a conversion that selects the byte, those of a narrower type do not
__device__ __forceinline__ int sbyte_of(unsigned v, int e) { return (int)(v << (24 - 8 * e)) >> 24; }

template <bool E4M3>
__device__ __forceinline__ void unpack4(unsigned r, float (&o)[4]) {
  if constexpr (E4M3) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)r, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)r, true);
    o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (float)sbyte_of(r, j);
  }
}

// Interleaved pairs of 8 elements (pair index 4c + j) rotated by the angles of position t.  Products of bf16 and fp32
// are exact in 64 bits and their sum is rounded there once, whether or not it is contracted to an fma, so the stored
// codes are the same bits for whoever recomputes them.  Then 64 -> 32 -> 16 bits, in two roundings as a tensor cast does
// it: round32 keeps the compiler from folding them into one (a compare and three selects more for each element).
__device__ __forceinline__ float round32(double v) {
  float f = (float)v;
  asm("" : "+v"(f));
  return f;
}
__device__ __forceinline__ bf16x8 rotate8(bf16x8 x, const float* cos_t, const float* sin_t) {
  const f32x4 co = *reinterpret_cast<const f32x4*>(cos_t), si = *reinterpret_cast<const f32x4*>(sin_t);
  bf16x8 o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double a = (double)(float)x[2 * j], b = (double)(float)x[2 * j + 1];
    const double c = (double)co[j], s = (double)si[j];
    o[2 * j] = (bf16)round32(a * c - b * s);
    o[2 * j + 1] = (bf16)round32(a * s + b * c);
  }
  return o;
}

// One workgroup per (sequence, K or V head, touched block).  The block is gathered into registers (old rows from the
// tail, new ones from qkv, keys rotated), reduced to its largest magnitude -- as integers: |bf16| compares like its
// bits, and infinities and NaN compare above every finite value -- and quantised if this append fills it.  The first
// touched block's workgroup is the only one that reads the tail, so it also stores the rows of the block left open,
// after those reads: no other workgroup has to be waited for.  The remaining workgroups rotate q.
template <bool E4M3, int NC>
__global__ __launch_bounds__(256) void kv8_append_k(KV8AppendParams p, int nblk, int quant_wgs) {
  const KV8& c = p.c;
  const int CH = c.D / 8, T = c.T, half = c.D / 2;
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= quant_wgs) {
    const int64_t i = (int64_t)(blockIdx.x - quant_wgs) * 256 + tid;
    if (i >= (int64_t)c.B * p.S * p.Hq * CH) return;
    const int ch = (int)(i % CH);
    int64_t r = i / CH;
    const int h = (int)(r % p.Hq);
    r /= p.Hq;
    const int s = (int)(r % p.S), b = (int)(r / p.S);
    const int64_t t = (int64_t)p.pos[b] + s;
    if (p.pos[b] < 0 || t >= c.Smax) return;   // the host checks capacity; the tables end with the cache
    bf16* x = (bf16*)p.qkv + (int64_t)b * p.qkv_sb + (int64_t)s * p.qkv_ss + (int64_t)h * c.D + ch * 8;
    *reinterpret_cast<bf16x8*>(x) =
        rotate8(*reinterpret_cast<const bf16x8*>(x), p.cos + t * half + ch * 4, p.sin + t * half + ch * 4);
    return;
  }
  __shared__ unsigned red[4];
  const int j = blockIdx.x % nblk;
  int r0 = blockIdx.x / nblk;
  const int hh = r0 % (2 * c.Hkv), b = r0 / (2 * c.Hkv);
  const bool is_k = hh < c.Hkv;
  const int h = is_k ? hh : hh - c.Hkv;
  const int pos = p.pos[b];
  if (pos < 0 || pos >= c.Smax) return;   // whole workgroup, before any barrier
  const int n = (int)min((int64_t)pos + p.S, (int64_t)c.Smax);
  const int blk = (pos >> c.lgT) + j, t0 = blk * T;
  if (t0 >= n) return;
  const bool full = n - t0 >= T;
  if (!full && j > 0) return;

  bf16* src = (bf16*)p.qkv + (int64_t)b * p.qkv_sb + (int64_t)(p.Hq + hh) * c.D;   // row s of this head: + s * qkv_ss
  bf16* tail = (bf16*)(is_k ? c.kt : c.vt) + (int64_t)b * c.t_sb + (int64_t)h * c.t_sh;
  auto fresh = [&](int t, int ch) -> bf16x8 {   // new row t; keys are rotated, in qkv too
    bf16* x = src + (int64_t)(t - pos) * p.qkv_ss + ch * 8;
    bf16x8 v = *reinterpret_cast<const bf16x8*>(x);
    if (is_k) {
      v = rotate8(v, p.cos + (int64_t)t * half + ch * 4, p.sin + (int64_t)t * half + ch * 4);
      *reinterpret_cast<bf16x8*>(x) = v;
    }
    return v;
  };
  if (full) {
    bf16x8 val[NC];
    unsigned mx = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int e = i * 256 + tid;
      if (e < T * CH) {
        const int row = e / CH, ch = e % CH, t = t0 + row;
        val[i] = t < pos ? *reinterpret_cast<const bf16x8*>(tail + (int64_t)row * c.t_ss + ch * 8) : fresh(t, ch);
        const u32x4 w = __builtin_bit_cast(u32x4, val[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) mx = max(mx, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = max(mx, (unsigned)__shfl_xor((int)mx, o, 64));
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    mx = max(max(red[0], red[1]), max(red[2], red[3]));
    const float amax = __uint_as_float(mx << 16);
    const bool finite = mx < 0x7f80u;
    const float sc = finite ? fmaxf(amax / (E4M3 ? 448.f : 127.f), kTinyScale) : __uint_as_float(0x7fc00000u);
    const float inv = finite ? 1.f / sc : 0.f;
    uint8_t* code = (uint8_t*)(is_k ? c.kc : c.vc) + (int64_t)b * c.c_sb + (int64_t)h * c.c_sh;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int e = i * 256 + tid;
      if (e < T * CH) {
        const int row = e / CH, ch = e % CH;
        float lo[4], hi[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          lo[k] = finite ? (float)val[i][k] * inv : 0.f;
          hi[k] = finite ? (float)val[i][4 + k] * inv : 0.f;
        }
        *reinterpret_cast<uint2*>(code + (int64_t)(t0 + row) * c.c_ss + ch * 8) =
            make_uint2(pack4<E4M3>(lo), pack4<E4M3>(hi));
      }
    }
    if (tid == 0) (is_k ? c.ks : c.vs)[(int64_t)b * c.s_sb + (int64_t)blk * c.s_sn + (int64_t)h * c.s_sh] = sc;
  }
  if (j == 0) {   // the barrier above ordered the tail's reads before these writes
    const int o0 = n >> c.lgT << c.lgT, from = max(o0, pos);
    for (int e = tid; e < (n - from) * CH; e += 256) {
      const int t = from + e / CH, ch = e % CH;
      *reinterpret_cast<bf16x8*>(tail + (int64_t)(t - o0) * c.t_ss + ch * 8) = fresh(t, ch);
    }
  }
}

// 8 elements of row t of the cache that holds n rows, in fp32
template <bool E4M3>
__device__ __forceinline__ void row8(const KV8& c, bool is_k, int b, int h, int t, int n, int ch, float (&o)[8]) {
  if (t < n >> c.lgT << c.lgT) {
    const uint2 r = *reinterpret_cast<const uint2*>((const uint8_t*)(is_k ? c.kc : c.vc) + (int64_t)b * c.c_sb +
                                                    (int64_t)t * c.c_ss + (int64_t)h * c.c_sh + ch * 8);
    const float sc = (is_k ? c.ks : c.vs)[(int64_t)b * c.s_sb + (int64_t)(t >> c.lgT) * c.s_sn + (int64_t)h * c.s_sh];
    float lo[4], hi[4];
    unpack4<E4M3>(r.x, lo);
    unpack4<E4M3>(r.y, hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k] = lo[k] * sc;
      o[4 + k] = hi[k] * sc;
    }
  } else {
    Vec8<bf16>::load((const bf16*)(is_k ? c.kt : c.vt) + (int64_t)b * c.t_sb + (int64_t)(t & (c.T - 1)) * c.t_ss +
                         (int64_t)h * c.t_sh + ch * 8, o);
  }
}

// ---- Decode attention: o = softmax(scale q K^T) V for one token of every sequence.
//
// Bound by the bytes of the codes: a key and value of one head are 2 D bytes, used by the G = Hq / Hkv query heads of
// the group.  So a wave takes 32 keys at a time and ALL heads of the group (up to 16, the width of the matrix tile):
//   S[key, head] = K q^T on v_mfma_f32_16x16x32_bf16, K as the A operand.  A code is exact in bf16 (8 significant bits
//     at most), so the scales stay out of the products: S is multiplied by the block's scale in fp32.
//   O^T[d, head] = V^T P, the accumulator of S reused as the B operand: a lane of S's result holds four keys of a head,
//     which become its eight k-slots of two 16-key tiles, so P never leaves its lane.  V^T is the A operand under the same
//     order of keys: lane (c, g) loads D / 16 contiguous bytes of its eight keys and takes byte e of each for d-tile e.
//   The weights times the scale of V enter as the sum of two bf16 parts (16 significant bits) -- a second product over the
//   operand that is converted anyway.
// 8-bit -> bf16 conversion is the largest part of the arithmetic: about 1.5 instructions an element, a third of what the
// vector units can do in the time that the bytes take.  Four waves of a workgroup share a unit of `chunk` keys in turns
// of 32 and merge over LDS; where a sequence is longer than a unit, units leave unnormalised sums for kv8_combine_k.
template <int D>
struct Raw {   // a lane's share of the codes of one key (K) and of one key's part of a head (V)
  typedef typename std::conditional<D >= 64, u32x4, uint2>::type K;
  typedef typename std::conditional<D == 128, uint2, typename std::conditional<D == 64, unsigned, uint16_t>::type>::type V;
};

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// four codes -> bf16, exact
template <bool E4M3>
__device__ __forceinline__ void widen4(unsigned r, bf16x8& o, int at) {
  float f[4];
  unpack4<E4M3>(r, f);
#pragma unroll
  for (int j = 0; j < 4; ++j) o[at + j] = (bf16)f[j];
}

// byte e of eight values of 1, 2, 4 or 8 bytes
__device__ __forceinline__ unsigned byte_of(uint2 v, int e) { return (e < 4 ? v.x >> (8 * e) : v.y >> (8 * (e - 4))) & 0xff; }
__device__ __forceinline__ unsigned byte_of(unsigned v, int e) { return v >> (8 * e) & 0xff; }
__device__ __forceinline__ unsigned byte_of(uint16_t v, int e) { return (unsigned)v >> (8 * e) & 0xff; }

__device__ __forceinline__ int sbyte_of(uint2 v, int e) { return sbyte_of(e < 4 ? v.x : v.y, e & 3); }

template <bool E4M3, typename V>
__device__ __forceinline__ bf16x8 column(const V (&v)[8], int e) {
  bf16x8 o;
  if constexpr (E4M3) {
    unsigned lo = 0, hi = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo |= byte_of(v[j], e) << (8 * j);
      hi |= byte_of(v[4 + j], e) << (8 * j);
    }
    widen4<true>(lo, o, 0);
    widen4<true>(hi, o, 4);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (bf16)(float)sbyte_of(v[j], e);
  }
  return o;
}

// 2^x, zero below 2^-126: a weight that small adds nothing
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// The running softmax of one wave: lane (c, g) holds head c's maximum, its own keys' share of the sum, and rows
// (D / 16) (4 g + r) + e of O^T in acc[e][r].
template <int D>
struct Online {
  f32x4 acc[D / 16];
  float m, l;
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int e = 0; e < D / 16; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }
  // s: scores in units of log2 (-inf: no key); vs: scale of V of the two tiles; column(e): A operand of d-tile e
  template <typename F>
  __device__ __forceinline__ void step(const f32x4 (&s)[2], const float (&vs)[2], F&& vcol) {
    float mx = m;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[a][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float base = mx == -INFINITY ? 0.f : mx;   // no key so far: exp2(-inf - 0) = 0
    if (__any(mx > m)) {
      const float a = fast_exp2(m - base);
      l *= a;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) acc[e] *= a;
    }
    m = mx;
    bf16x8 hi, lo;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = fast_exp2(s[a][r] - base);   // a NaN score leaves m alone and makes l and acc NaN for good
        l += p;
        const float w = p * vs[a];
        const bf16 h = (bf16)w;
        hi[4 * a + r] = h;
        lo[4 * a + r] = (bf16)(w - (float)h);
      }
#pragma unroll
    for (int e = 0; e < D / 16; ++e) {
      const bf16x8 v = vcol(e);
      acc[e] = mfma16(v, hi, acc[e]);
      acc[e] = mfma16(v, lo, acc[e]);
    }
  }
};

template <bool E4M3, int D>
__global__ __launch_bounds__(256, 4) void kv8_decode_k(KV8DecodeParams p) {
  constexpr int NI = D / 32, NE = D / 16, NH = D >= 64 ? D / 64 : 1, LD = D + 4;   // LD: rows of heads fall on other banks
  __shared__ float so[4][16][LD];
  __shared__ float sml[4][16][2];
  const KV8& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, g = lane >> 4;
  int id = blockIdx.x;
  const int u = id % p.units;
  id /= p.units;
  const int G = p.Hq / c.Hkv, tiles = (G + 15) / 16;
  const int ct = id % tiles;
  id /= tiles;
  const int h = id % c.Hkv, b = id / c.Hkv;
  const int n = max(0, min(p.pos[b], c.Smax - 1) + 1);
  const int lo = u * p.chunk, hi = min(n, lo + p.chunk);
  const int hq0 = h * G + ct * 16, nq = min(16, G - ct * 16);
  if (lo >= n) {   // no keys; a sequence without any has a zero output
    if (n == 0 && u == 0)
      for (int i = tid; i < nq * D; i += 256) ((bf16*)p.out)[((int64_t)b * p.Hq + hq0) * D + i] = (bf16)0.f;
    return;
  }
  const int full = n >> c.lgT << c.lgT;
  const float sl2 = p.scale * 1.4426950408889634f;

  // q as the B operand: lane (head, g), chunk i holds the d that K's chunk i has in the lanes of group g
  auto dof = [&](int i) { return D >= 64 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 8 * g; };
  bf16x8 qf[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    qf[i] = bf16x8{};
    if (r16 < nq)
      qf[i] = *reinterpret_cast<const bf16x8*>((const bf16*)p.q + (int64_t)b * p.q_sb + (int64_t)(hq0 + r16) * D + dof(i));
  }
  Online<D> st;
  st.init();

  const int end = min(hi, full);   // keys lo .. end are codes; end - lo is a multiple of 16
  const int first = lo + 32 * __builtin_amdgcn_readfirstlane(wave);
  if (first < end) {
    // lane i keeps the scales of the unit's block i (chunk <= 64 T): no load of a single float inside the loop
    const int blk0 = lo >> c.lgT;
    float ksl = 0.f, vsl = 0.f;
    if (lane < (end - lo) >> c.lgT) {
      const int64_t at = (int64_t)b * c.s_sb + (int64_t)h * c.s_sh + (int64_t)(blk0 + lane) * c.s_sn;
      ksl = c.ks[at];
      vsl = c.vs[at];
    }
    auto scale_at = [&](float v, int key) {
      return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), (key >> c.lgT) - blk0));
    };
    // uniform base of a 16-key tile plus 32-bit offsets of the lane that stay the same; where the codes end with the
    // step's first tile (T = 16), the second one re-reads it and is masked
    const int64_t head = (int64_t)b * c.c_sb + (int64_t)h * c.c_sh;
    const int ss = (int)c.c_ss;
    const unsigned ko = (unsigned)(r16 * ss + (D >= 64 ? 16 : 8) * g);
    unsigned vo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vo[j] = (unsigned)((4 * g + j) * ss + r16 * NE);
    auto tile = [&](int k0, int a) { return head + (int64_t)(k0 + (a && k0 + 16 < end ? 16 : 0)) * c.c_ss; };
    typename Raw<D>::K k[2][NH];
    auto load_k = [&](int k0) {
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint8_t* base = (const uint8_t*)c.kc + tile(k0, a);
#pragma unroll
        for (int x = 0; x < NH; ++x) k[a][x] = *reinterpret_cast<const typename Raw<D>::K*>(base + ko + 64 * x);
      }
    };
    load_k(first);
    for (int k0 = first; k0 < end; k0 += 128) {
      typename Raw<D>::V v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = *reinterpret_cast<const typename Raw<D>::V*>((const uint8_t*)c.vc + tile(k0, j >> 2) + vo[j & 3]);
      f32x4 s[2];
      float vs[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        s[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          bf16x8 kb;
          if constexpr (D >= 64) {
            widen4<E4M3>(k[a][i >> 1][2 * (i & 1)], kb, 0);
            widen4<E4M3>(k[a][i >> 1][2 * (i & 1) + 1], kb, 4);
          } else {
            widen4<E4M3>(k[a][0].x, kb, 0);
            widen4<E4M3>(k[a][0].y, kb, 4);
          }
          s[a] = mfma16(kb, qf[i], s[a]);
        }
        const int key = a && k0 + 16 < end ? k0 + 16 : k0;
        const float f = sl2 * scale_at(ksl, key);
        vs[a] = scale_at(vsl, key);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[a][r] *= f;
      }
      if (k0 + 16 >= end) s[1] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      load_k(k0 + 128 < end ? k0 + 128 : k0);   // the last turn re-reads its own keys: no branch around loads
      st.step(s, vs, [&](int e) { return column<E4M3>(v, e); });
    }
  }
  // the open block's bf16 rows, 32 of them a wave
  const int t0 = 32 * wave, rows = hi - full;
  if (t0 < rows) {
    const bf16* kt = (const bf16*)c.kt + (int64_t)b * c.t_sb + (int64_t)h * c.t_sh;
    const bf16* vt = (const bf16*)c.vt + (int64_t)b * c.t_sb + (int64_t)h * c.t_sh;
    f32x4 s[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      s[a] = f32x4{0.f, 0.f, 0.f, 0.f};
      const bf16* row = kt + (int64_t)min(t0 + 16 * a + r16, rows - 1) * c.t_ss;
#pragma unroll
      for (int i = 0; i < NI; ++i) s[a] = mfma16(*reinterpret_cast<const bf16x8*>(row + dof(i)), qf[i], s[a]);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[a][r] = t0 + 16 * a + 4 * g + r < rows ? s[a][r] * sl2 : -INFINITY;
    }
    typedef __bf16 vrow __attribute__((ext_vector_type(NE)));
    vrow v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = *reinterpret_cast<const vrow*>(vt + (int64_t)min(t0 + 16 * (j >> 2) + 4 * g + (j & 3), rows - 1) * c.t_ss +
                                            r16 * NE);
    const float one[2] = {1.f, 1.f};
    st.step(s, one, [&](int e) {
      bf16x8 o;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = v[j][e];
      return o;
    });
  }

  // merge the four waves
  float l = st.l;
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (r16 < nq) {
    if (g == 0) {
      sml[wave][r16][0] = st.m;
      sml[wave][r16][1] = l;
    }
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int r = 0; r < 4; ++r) so[wave][r16][NE * (4 * g + r) + e] = st.acc[e][r];
  }
  __syncthreads();
  for (int i = tid; i < nq * D; i += 256) {
    const int q = i / D, d = i % D;
    float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sml[w][q][0]);
    const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = fast_exp2(sml[w][q][0] - base);
      L = fmaf(a, sml[w][q][1], L);
      o = fmaf(a, so[w][q][d], o);
    }
    const int64_t row = (int64_t)b * p.Hq + hq0 + q;
    if (p.units == 1) {
      ((bf16*)p.out)[row * D + d] = (bf16)(o / L);
    } else {
      const int64_t slot = row * p.units + u;
      p.opart[slot * D + d] = o;
      if (d == 0) {
        p.mlpart[2 * slot] = M;
        p.mlpart[2 * slot + 1] = L;
      }
    }
  }
}

// One workgroup per (sequence, query head): its waves take the units in turns, then merge.  D / 64 (at least 1) elements a
// lane.
template <int D>
__global__ __launch_bounds__(256) void kv8_combine_k(KV8DecodeParams p) {
  constexpr int E = D >= 64 ? D / 64 : 1;
  __shared__ float so[4][D], sl[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const int n = max(0, min(p.pos[row / p.Hq], p.c.Smax - 1) + 1), nu = min((int)cdiv(n, p.chunk), p.units);
  if (nu == 0) return;   // zeros already stored
  const float* ml = p.mlpart + row * p.units * 2;
  const float* op = p.opart + row * p.units * D;
  float M = -INFINITY;
  for (int i = lane; i < nu; i += 64) M = fmaxf(M, ml[2 * i]);
  M = wave_max(M);
  const float base = M == -INFINITY ? 0.f : M;
  const bool active = lane * E < D;
  float L = 0.f, o[E] = {};
#pragma unroll 4
  for (int i = wave; i < nu; i += 4) {
    const float a = fast_exp2(ml[2 * i] - base);
    L = fmaf(a, ml[2 * i + 1], L);
    if (active) {
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(a, op[(int64_t)i * D + lane * E + e], o[e]);
    }
  }
  if (lane == 0) sl[wave] = L;
  if (active) {
#pragma unroll
    for (int e = 0; e < E; ++e) so[wave][lane * E + e] = o[e];
  }
  __syncthreads();
  if ((int)threadIdx.x < D) {
    const int d = threadIdx.x;
    const float sum = (so[0][d] + so[1][d]) + (so[2][d] + so[3][d]), all = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    ((bf16*)p.out)[row * D + d] = (bf16)(sum / all);
  }
}

template <bool E4M3>
__global__ __launch_bounds__(256) void kv8_read_k(KV8ReadParams p) {
  const KV8& c = p.c;
  const int CH = c.D / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)c.B * p.count * c.Hkv * 2 * CH) return;
  const int ch = (int)(i % CH);
  int64_t r = i / CH;
  const int h = (int)(r % c.Hkv);
  r /= c.Hkv;
  const int s = (int)(r % p.count);
  r /= p.count;
  const int b = (int)(r % c.B);
  const bool is_k = r < c.B;
  const int n = max(0, min(p.pos[b], c.Smax)), t = n - p.count + s;
  float v[8] = {};
  if (t >= 0) row8<E4M3>(c, is_k, b, h, t, n, ch, v);
  Vec8<bf16>::store((bf16*)(is_k ? p.ko : p.vo) + (int64_t)b * p.o_sb + (int64_t)s * p.o_ss + (int64_t)h * p.o_sh + ch * 8,
                    v);
}

}  // namespace

void kv8_append(const KV8AppendParams& p, hipStream_t st) {
  const KV8& c = p.c;
  if (c.B == 0 || p.S == 0) return;
  const int CH = c.D / 8;
  const int nblk = (p.S + c.T - 2) / c.T + 1;   // blocks that S rows can touch, whatever their first position
  const int quant = c.B * 2 * c.Hkv * nblk;
  const dim3 grid((unsigned)(quant + cdiv((int64_t)c.B * p.S * p.Hq * CH, 256)));
#define DPH_KV8_APP(E_, NC_) hipLaunchKernelGGL((kv8_append_k<E_, NC_>), grid, dim3(256), 0, st, p, nblk, quant)
#define DPH_KV8_APP_E(NC_)               \
  do {                                   \
    if (c.e4m3) DPH_KV8_APP(true, NC_);  \
    else DPH_KV8_APP(false, NC_);        \
  } while (0)
  const int chunks = c.T * CH;   // 16-B chunks of one block, in registers: at most 8 a thread
  if (chunks <= 256) DPH_KV8_APP_E(1);
  else if (chunks <= 512) DPH_KV8_APP_E(2);
  else if (chunks <= 1024) DPH_KV8_APP_E(4);
  else DPH_KV8_APP_E(8);
#undef DPH_KV8_APP_E
#undef DPH_KV8_APP
}

// Keys of one unit of work: enough units to fill the card several times over whatever the batch (ragged sequences then
// even out), no fewer than a step of each wave, and a multiple of every block size, so that no open block crosses units.
int kv8_decode_chunk(int B, int Hkv, int Hq, int T, int max_len) {
  const int64_t rows = (int64_t)B * Hkv * cdiv(Hq / Hkv, 16);
  const int64_t keys = cdiv(rows * max_len, 1024);
  return (int)std::min<int64_t>(128 * std::max<int64_t>(1, cdiv(keys, 128)), 64 * T);   // a lane holds a block's scales
}

void kv8_decode_attention(const KV8DecodeParams& p, hipStream_t st) {
  const KV8& c = p.c;
  if (c.B == 0) return;
  const dim3 grid((unsigned)((int64_t)p.units * c.B * c.Hkv * cdiv(p.Hq / c.Hkv, 16)));
#define DPH_KV8_DEC(D_)                                                                          \
  do {                                                                                           \
    if (c.e4m3) hipLaunchKernelGGL((kv8_decode_k<true, D_>), grid, dim3(256), 0, st, p);         \
    else hipLaunchKernelGGL((kv8_decode_k<false, D_>), grid, dim3(256), 0, st, p);               \
    if (p.units > 1) hipLaunchKernelGGL(kv8_combine_k<D_>, dim3((unsigned)(c.B * p.Hq)), dim3(256), 0, st, p); \
  } while (0)
  if (c.D == 128) DPH_KV8_DEC(128);
  else if (c.D == 64) DPH_KV8_DEC(64);
  else DPH_KV8_DEC(32);
#undef DPH_KV8_DEC
}

void kv8_read(const KV8ReadParams& p, hipStream_t st) {
  const int64_t total = (int64_t)p.c.B * p.count * p.c.Hkv * 2 * (p.c.D / 8);
  if (total == 0) return;
  const dim3 grid((unsigned)cdiv(total, 256));
  if (p.c.e4m3) hipLaunchKernelGGL(kv8_read_k<true>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(kv8_read_k<false>, grid, dim3(256), 0, st, p);
}

}  // namespace dph
