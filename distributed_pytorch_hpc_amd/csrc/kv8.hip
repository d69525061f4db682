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

// byte e, signed: shifts of 32 bits fold into a conversion that selects the byte, those of a narrower type do not (and the
// signed bit-field-extract builtin before a conversion to float came out as an unsigned conversion: wrong codes)
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
struct Angles {   // of a chunk's four pairs
  f32x4 c, s;
};
__device__ __forceinline__ bf16x8 rotate8(bf16x8 x, const Angles& w) {
  bf16x8 o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double a = (double)(float)x[2 * j], b = (double)(float)x[2 * j + 1];
    const double c = (double)w.c[j], s = (double)w.s[j];
    o[2 * j] = (bf16)round32(a * c - b * s);
    o[2 * j + 1] = (bf16)round32(a * s + b * c);
  }
  return o;
}

// Two kinds of workgroups.  The first: one per (sequence, K or V head, touched block).  The block is gathered into
// registers (old rows from the tail, new ones from qkv, keys rotated), reduced to its largest magnitude -- as integers:
// |bf16| compares like its bits, and infinities and NaN compare above every finite value -- and quantised if this append
// fills it.  The first touched block's workgroup is the only one that reads the tail, so it also stores the rows of the
// block left open, after those reads: no other workgroup has to be waited for.  The second kind rotates q, one per new
// token: a thread keeps its angles and goes from head to head with them.
template <bool E4M3, int NC>
__global__ __launch_bounds__(256) void kv8_append_k(KV8AppendParams p, int nblk, int quant_wgs) {
  const KV8& c = p.c;
  const int T = c.T, half = c.D / 2, tid = threadIdx.x;
  auto angles = [&](int t, int ch) {
    const int64_t o = (int64_t)t * half + ch * 4;
    return Angles{*reinterpret_cast<const f32x4*>(p.cos + o), *reinterpret_cast<const f32x4*>(p.sin + o)};
  };
  if ((int)blockIdx.x >= quant_wgs) {
    const int i = blockIdx.x - quant_wgs, b = i / p.S, s = i - b * p.S;
    bf16* x = (bf16*)p.qkv + (int64_t)b * p.qkv_sb + (int64_t)s * p.qkv_ss;
    const int n = p.Hq << c.lgC;   // chunks; 256 is a multiple of a head's
    bf16x8 v[4];
    auto load = [&](int e) {
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const bf16x8*>(x + 8 * (e + 256 * u < n ? e + 256 * u : e));
    };
    if (tid >= n) return;
    load(tid);   // before the position is known: only the angles wait for it
    const int64_t t = (int64_t)p.pos[b] + s;
    if (t < s || t >= c.Smax) return;   // the host checks capacity; the tables end with the cache
    const Angles w = angles((int)t, tid & ((1 << c.lgC) - 1));
    for (int e = tid; e < n; e += 4 * 256) {
      if (e != tid) load(e);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (e + 256 * u < n) *reinterpret_cast<bf16x8*>(x + 8 * (e + 256 * u)) = rotate8(v[u], w);
    }
    return;
  }
  __shared__ unsigned red[4];
  const int j = blockIdx.x % nblk, r0 = blockIdx.x / nblk;
  const int hh = r0 % (2 * c.Hkv), b = r0 / (2 * c.Hkv);
  const bool is_k = hh < c.Hkv;
  const int h = is_k ? hh : hh - c.Hkv;
  const int pos = p.pos[b];
  if (pos < 0 || pos >= c.Smax) return;   // whole workgroup, before any barrier
  const int n = (int)min((int64_t)pos + p.S, (int64_t)c.Smax);
  const int blk = (pos >> c.lgT) + j, t0 = blk << c.lgT;
  if (t0 >= n) return;
  const bool full = n - t0 >= T;
  if (!full && j > 0) return;

  bf16* src = (bf16*)p.qkv + (int64_t)b * p.qkv_sb + (int64_t)(p.Hq + hh) * c.D;   // row s of this head: + s * qkv_ss
  bf16* tail = (bf16*)(is_k ? c.kt : c.vt) + (int64_t)b * c.t_sb + (int64_t)h * c.t_sh;
  const int chunks = T << c.lgC, mask = (1 << c.lgC) - 1;
  if (full) {
    bf16x8 val[NC];
    Angles w[NC];
    // every load at once: rows come from one of two places by address, threads past a small block take its last chunk
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int e = min(i * 256 + tid, chunks - 1), row = e >> c.lgC, ch = e & mask, t = t0 + row;
      val[i] = *reinterpret_cast<const bf16x8*>(t < pos ? tail + (int64_t)row * c.t_ss + ch * 8
                                                        : src + (int64_t)(t - pos) * p.qkv_ss + ch * 8);
    }
    if (is_k) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int e = min(i * 256 + tid, chunks - 1);
        w[i] = angles(t0 + (e >> c.lgC), e & mask);
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int e = min(i * 256 + tid, chunks - 1), t = t0 + (e >> c.lgC);
        const bf16x8 r = rotate8(val[i], w[i]);
        if (t >= pos) {
          val[i] = r;
          if (i * 256 + tid < chunks)
            *reinterpret_cast<bf16x8*>(src + (int64_t)(t - pos) * p.qkv_ss + (e & mask) * 8) = r;
        }
      }
    }
    unsigned mx = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (i * 256 + tid >= chunks) continue;   // not its chunk: the owner may have rotated it in qkv before it was read
      const u32x4 u = __builtin_bit_cast(u32x4, val[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) mx = max(mx, max(u[k] & 0x7fffu, (u[k] >> 16) & 0x7fffu));
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
      if (e < chunks) {
        float lo[4], hi[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          lo[k] = finite ? (float)val[i][k] * inv : 0.f;
          hi[k] = finite ? (float)val[i][4 + k] * inv : 0.f;
        }
        *reinterpret_cast<uint2*>(code + (int64_t)(t0 + (e >> c.lgC)) * c.c_ss + (e & mask) * 8) =
            make_uint2(pack4<E4M3>(lo), pack4<E4M3>(hi));
      }
    }
    if (tid == 0) (is_k ? c.ks : c.vs)[(int64_t)b * c.s_sb + (int64_t)blk * c.s_sn + (int64_t)h * c.s_sh] = sc;
  }
  if (j == 0) {   // the barrier above ordered the tail's reads before these writes
    const int o0 = n >> c.lgT << c.lgT, from = max(o0, pos);
    for (int e = tid; e < (n - from) << c.lgC; e += 256) {
      const int t = from + (e >> c.lgC), ch = e & mask;
      bf16* x = src + (int64_t)(t - pos) * p.qkv_ss + ch * 8;
      bf16x8 v = *reinterpret_cast<const bf16x8*>(x);
      if (is_k) {
        v = rotate8(v, angles(t, ch));
        *reinterpret_cast<bf16x8*>(x) = v;
      }
      *reinterpret_cast<bf16x8*>(tail + (int64_t)(t - o0) * c.t_ss + ch * 8) = v;
    }
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
// vector units can do in the time that the bytes take.  Four waves of a workgroup share a turn of 128 keys and merge over
// LDS; where several workgroups share a row, they leave unnormalised sums for kv8_combine_k.
// Measured (kernel trace): 16 sequences of 1000 to 4000 tokens, 32 / 32 heads, 328 MB: 63 us, 5.2 TB/s (a streaming read of
// that size: 5.8 to 6.0); 32 of 4000 to 8100 tokens, 64 / 8 heads, 398 MB: 75.5 us; one of 32 002 tokens, 64 / 8 heads:
// 15.8 us; one of 2346 tokens, 32 / 32 heads: 8.6 us.  The merge adds 3.5 to 5.7 us and a launch.  One thread per 8
// elements and key instead of matrix tiles: 399, 964, 2095 and 152 us.
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

// 2^x, zero below 2^-126: a weight that small adds nothing (and makes NaN of an infinity, as any weight of zero does)
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ bf16x8 finite_or_zero(bf16x8 v) {
  u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned x = u[k];
    u[k] = ((x & 0x7f800000u) == 0x7f800000u ? 0u : x & 0xffff0000u) | ((x & 0x7f80u) == 0x7f80u ? 0u : x & 0xffffu);
  }
  return __builtin_bit_cast(bf16x8, u);
}

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
  // s: scores in units of log2 (-inf: no key); vs: scale of V of the two tiles; column(e): A operand of d-tile e.
  // OPEN: V is bf16 and may hold infinities (codes have none, a block with one has the scale NaN).  The weight's low part
  // is zero or of either sign, so it must not meet them: their sum with the high part alone is the infinity that stands
  // there.  A sum that is finite has met none; looking at the sums takes 0.1 to 0.2 us of a call, less than looking at V.
  template <bool OPEN, typename F>
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
    if constexpr (OPEN) {
      float z = 0.f;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        acc[e] = mfma16(vcol(e), hi, acc[e]);
#pragma unroll
        for (int r = 0; r < 4; ++r) z = fmaf(acc[e][r], 0.f, z);
      }
      const bool finite = !__any(z != 0.f);
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        bf16x8 v = vcol(e);
        if (!finite) v = finite_or_zero(v);
        acc[e] = mfma16(v, lo, acc[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        const bf16x8 v = vcol(e);
        acc[e] = mfma16(v, hi, acc[e]);
        acc[e] = mfma16(v, lo, acc[e]);
      }
    }
  }
};

// The work of a call, in turns of 128 keys (32 for each wave of a workgroup): row (b, h, tile of 16 heads) has
// ceil(n_b / 128) turns, at least one, and the rows' turns stand in one line, which the workgroups divide evenly whatever
// the lengths are -- with a fixed number of keys a workgroup, sequences of 1000 to 4000 tokens left the card half idle at
// the end (16 of 7B heads: 73 us, divided evenly 66).  The lengths are only known on the device, so every workgroup adds
// them up for itself.
struct Line {
  int turns;       // of all rows
  int per, rem;    // workgroup w has per + (w < rem) of them, from share_of(w)
  int b, n, row0;  // the sequence of this workgroup's first turn, its length, and the turn at which its rows begin
};

__device__ __forceinline__ int length_of(const KV8DecodeParams& p, int b) {
  return max(0, min(p.pos[b], p.c.Smax - 1) + 1);
}
// turns that a row of n keys counts for; one, where there is no workspace for shares of it (max_len <= 128)
__device__ __forceinline__ int turns_of(const KV8DecodeParams& p, int n) { return p.opart ? max(1, (n + 127) >> 7) : 1; }
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
// workgroups past the last turn (fewer turns than workgroups) begin and end there
__device__ __forceinline__ int share_of(const Line& o, int w) { return min(w * o.per + min(w, o.rem), o.turns); }
__device__ __forceinline__ int owner_of(const Line& o, int turn) {
  const int big = o.rem * (o.per + 1);
  return turn < big ? (unsigned)turn / (unsigned)(o.per + 1) : o.rem + (unsigned)(turn - big) / (unsigned)o.per;
}

// inclusive sum over the wave's lanes: within rows of 16 lanes, then across them (DPP: no trip through LDS)
__device__ __forceinline__ int scan64(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast 15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast 31 into rows 2 and 3
  return v;
}

__device__ __forceinline__ Line line_up(const KV8DecodeParams& p, int w) {
  const int lane = threadIdx.x & 63, B = p.c.B, heads = p.c.Hkv * p.tiles;
  Line o;
  int total = 0, scan = 0, nt = 0, n = 0;
  auto sum_up = [&](int base) {
    n = base + lane < B ? length_of(p, base + lane) : 0;
    nt = base + lane < B ? turns_of(p, n) : 0;
    scan = scan64(nt);
  };
  for (int base = 0; base < B; base += 64) {
    sum_up(base);
    total += __builtin_amdgcn_readlane(scan, 63);
  }
  o.turns = total * heads;
  const int wgs = min(p.wgs, o.turns);
  o.per = uni((unsigned)o.turns / (unsigned)wgs);
  o.rem = o.turns - o.per * wgs;
  const int at = share_of(o, w);
  o.b = o.n = o.row0 = 0;
  for (int base = 0, before = 0; base < B; base += 64) {
    if (B > 64) sum_up(base);   // otherwise the sums above still stand
    const unsigned long long hit = __ballot((before + scan) * heads > at);
    if (hit) {
      const int l = uni(__ffsll(hit) - 1);
      o.b = base + l;
      o.n = __builtin_amdgcn_readlane(n, l);
      o.row0 = (before + __builtin_amdgcn_readlane(scan - nt, l)) * heads;
      break;
    }
    before += __builtin_amdgcn_readlane(scan, 63);
  }
  return o;
}

template <bool E4M3, int D>
__global__ __launch_bounds__(256, 2) void kv8_decode_k(KV8DecodeParams p) {
  constexpr int NI = D / 32, NE = D / 16, NH = D >= 64 ? D / 64 : 1, LD = D + 4;   // LD: rows of heads fall on other banks
  __shared__ float so[4][16][LD];
  __shared__ float sml[4][16][2];
  const KV8& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), r16 = lane & 15, g = lane >> 4;
  const int w = blockIdx.x, G = p.Hq / c.Hkv, heads = c.Hkv * p.tiles;
  const Line line = line_up(p, w);
  int at = share_of(line, w);
  const int stop = share_of(line, w + 1);
  if (at >= stop) return;
  int b = line.b, n = line.n, nt = turns_of(p, n);
  int row = uni((unsigned)(at - line.row0) / (unsigned)nt), t0 = at - line.row0 - row * nt;
  const float sl2 = p.scale * 1.4426950408889634f;
  // the d of chunk i of a key (and so of q) in the lanes of group g
  auto dof = [&](int i) { return D >= 64 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 8 * g; };

  // A row's share of this workgroup's turns at a time: turns t0 .. t1 of nt.  What a share begins with -- q, its first
  // keys, the scales of its first 64 blocks -- is asked for before the last share's sums are merged.
  int t1, hq0, nq, full, end, first;
  int64_t head;
  bf16x8 qf[NI];              // q as the B operand: lane (head, g)
  typename Raw<D>::K k[2][NH];
  float ksl = 0.f, vsl = 0.f;   // lane i: the scales of block blk0 + i
  int blk0 = 0, h;
  // uniform base of a 16-key tile plus 32-bit offsets of the lane that stay the same; where the codes end with a step's
  // first tile (T = 16), the second one re-reads it and is masked
  const int ss = (int)c.c_ss;
  const unsigned ko = (unsigned)(r16 * ss + (D >= 64 ? 16 : 8) * g);
  unsigned vo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) vo[j] = (unsigned)((4 * g + j) * ss + r16 * NE);
  auto tile = [&](int k0, int a) { return head + (int64_t)(k0 + (a && k0 + 16 < end ? 16 : 0)) * c.c_ss; };
  auto load_k = [&](int k0) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const uint8_t* base = (const uint8_t*)c.kc + tile(k0, a);
#pragma unroll
      for (int x = 0; x < NH; ++x) k[a][x] = *reinterpret_cast<const typename Raw<D>::K*>(base + ko + 64 * x);
    }
  };
  auto load_scales = [&](int key) {
    blk0 = key >> c.lgT;
    if (blk0 + lane < end >> c.lgT) {
      const int64_t off = (int64_t)b * c.s_sb + (int64_t)h * c.s_sh + (int64_t)(blk0 + lane) * c.s_sn;
      ksl = c.ks[off];
      vsl = c.vs[off];
    }
  };
  auto begin = [&]() {
    t1 = min(nt, t0 + stop - at);
    h = p.tiles == 1 ? row : uni((unsigned)row / (unsigned)p.tiles);
    const int ct = row - h * p.tiles;
    hq0 = h * G + ct * 16;
    nq = min(16, G - ct * 16);
    full = n >> c.lgT << c.lgT;
    end = t1 == nt ? full : 128 * t1;   // keys 128 t0 .. end are codes; a multiple of 16
    first = 128 * t0 + 32 * wave;
    head = (int64_t)b * c.c_sb + (int64_t)h * c.c_sh;
    const bf16* q = (const bf16*)p.q + (int64_t)b * p.q_sb + (int64_t)(hq0 + min(r16, nq - 1)) * D;
#pragma unroll
    for (int i = 0; i < NI; ++i) qf[i] = *reinterpret_cast<const bf16x8*>(q + dof(i));   // spare columns: the last head
    if (first < end) {
      load_scales(first);
      load_k(first);
    }
  };
  begin();
  while (true) {
    Online<D> st;
    st.init();
    if (first < end) {
      auto scale_at = [&](float v, int key) {
        return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), (key >> c.lgT) - blk0));
      };
      // spans of 64 blocks: the loop over a span has no load of a single float (nor one under a condition, for which the
      // compiler would wait with the loads of V in flight)
      for (int span = first; span < end; span += 64 << c.lgT) {
        if (span != first) load_scales(span);
        const int span_end = min(end, span + (64 << c.lgT) - 127);
        for (int k0 = span; k0 < span_end; k0 += 128) {
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
          st.template step<false>(s, vs, [&](int e) { return column<E4M3>(v, e); });
        }
      }
    }
    // the open block's bf16 rows lie in the row's last turn (T divides 128): 32 of them a wave
    const int u0 = 32 * wave, rows = t1 == nt ? n - full : 0;
    if (u0 < rows) {
      const int64_t base = (int64_t)b * c.t_sb + (int64_t)h * c.t_sh;
      const char* kt = (const char*)((const bf16*)c.kt + base);
      const char* vt = (const char*)((const bf16*)c.vt + base);
      const unsigned ts = 2u * (unsigned)c.t_ss;
      typedef __bf16 vrow __attribute__((ext_vector_type(NE)));
      bf16x8 kr[2][NI];
      vrow v[8];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const unsigned off = (unsigned)min(u0 + 16 * a + r16, rows - 1) * ts + 2u * (unsigned)dof(0);
#pragma unroll
        for (int i = 0; i < NI; ++i) kr[a][i] = *reinterpret_cast<const bf16x8*>(kt + off + 2 * (dof(i) - dof(0)));
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = *reinterpret_cast<const vrow*>(vt + (unsigned)min(u0 + 16 * (j >> 2) + 4 * g + (j & 3), rows - 1) * ts +
                                              (unsigned)(r16 * NE * 2));
      __builtin_amdgcn_sched_barrier(0);   // all sixteen loads before the first wait
      f32x4 s[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        s[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NI; ++i) s[a] = mfma16(kr[a][i], qf[i], s[a]);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[a][r] = u0 + 16 * a + 4 * g + r < rows ? s[a][r] * sl2 : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)   // rows past the last one are it again, of weight 0: no infinity may meet that
        if (u0 + 16 * (j >> 2) + 4 * g + (j & 3) >= rows) v[j] = vrow{};
      const float one[2] = {1.f, 1.f};
      st.template step<true>(s, one, [&](int e) {
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
    const bool whole = t0 == 0 && t1 == nt, none = n == 0;
    const int64_t slot = 2 * (int64_t)w + (t0 == 0 ? 1 : 0);   // one share that goes on from the last workgroup's row, one
                                                               // that the next one goes on with
    if (p.opart && t0 == 0 && tid == 0) {   // who has the row, for kv8_combine_k
      int* info = p.info + 2 * ((int64_t)b * heads + row);
      info[0] = w;
      info[1] = owner_of(line, at + nt - 1) - w + 1;
    }
    const int heads_here = nq;
    const int64_t out_row = (int64_t)b * p.Hq + hq0;
    at += t1 - t0;
    const bool more = at < stop;
    if (more) {
      t0 = 0;
      if (++row == heads) {
        row = 0;
        n = uni(length_of(p, ++b));
        nt = turns_of(p, n);
      }
      begin();
    }
    __syncthreads();
    for (int i = tid; i < heads_here * D; i += 256) {
      const int q = i / D, d = i % D;
      float M = -INFINITY, L = 0.f, o = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) M = fmaxf(M, sml[x][q][0]);
      const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float a = fast_exp2(sml[x][q][0] - base);
        L = fmaf(a, sml[x][q][1], L);
        o = fmaf(a, so[x][q][d], o);
      }
      if (whole) {   // a sequence without keys has a zero output
        ((bf16*)p.out)[(out_row + q) * D + d] = (bf16)(none ? 0.f : o / L);
      } else {
        p.opart[(slot * 16 + q) * D + d] = o;
        if (d == 0) {
          p.mlpart[(slot * 16 + q) * 2] = M;
          p.mlpart[(slot * 16 + q) * 2 + 1] = L;
        }
      }
    }
    if (!more) break;
    __syncthreads();   // before the next share's sums overwrite these
  }
}

// One workgroup per (sequence, query head) joins the shares of a row that several workgroups had: its waves take them in
// turns, then merge.  D / 64 (at least 1) elements a lane.  3.5 (32 rows) to 5.7 us (2048 rows): latency.
template <int D>
__global__ __launch_bounds__(256) void kv8_combine_k(KV8DecodeParams p) {
  constexpr int E = D >= 64 ? D / 64 : 1;
  __shared__ float so[4][D];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int hq = blockIdx.x % p.Hq, b = blockIdx.x / p.Hq, G = p.Hq / p.c.Hkv, q = hq % G % 16;
  const int* info = p.info + 2 * ((int64_t)b * p.c.Hkv * p.tiles + hq / G * p.tiles + hq % G / 16);
  const int w0 = uni(info[0]), shares = uni(info[1]);
  if (shares == 1) return;   // stored whole
  auto slot = [&](int i) { return (2 * (int64_t)(w0 + i) + (i == 0 ? 1 : 0)) * 16 + q; };
  const bool active = lane * E < D;
  // 64 shares at a time: lane i weighs share i, the wave's own ones among them are added up
  float M = -INFINITY, L = 0.f, o[E] = {};
  for (int base = 0; base < shares; base += 64) {
    float m = -INFINITY, l = 0.f;
    if (base + lane < shares) {
      const float2 ml = *reinterpret_cast<const float2*>(p.mlpart + 2 * slot(base + lane));
      m = ml.x;
      l = ml.y;
    }
    const float mx = fmaxf(M, wave_max(m)), ref = mx == -INFINITY ? 0.f : mx, old = fast_exp2(M - ref);
    const float a = fast_exp2(m - ref);
    L = L * old + wave_sum(a * l);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= old;
    M = mx;
    const int n = min(64, shares - base);
    for (int i0 = wave; i0 < n; i0 += 32) {   // eight loads in flight; past the end the last share again, not added
      float v[8][E], ai[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = min(i0 + 4 * u, n - 1);
        ai[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(a), i));
#pragma unroll
        for (int e = 0; e < E; ++e) v[u][e] = p.opart[slot(base + i) * D + (active ? lane * E + e : 0)];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e)   // a sum of 0, not a weight of 0: that would make NaN of an infinity
          o[e] = fmaf(ai[u], i0 + 4 * u < n ? v[u][e] : 0.f, o[e]);
    }
  }
  if (active) {
#pragma unroll
    for (int e = 0; e < E; ++e) so[wave][lane * E + e] = o[e];
  }
  __syncthreads();
  if ((int)threadIdx.x < D) {
    const int d = threadIdx.x;
    const float sum = (so[0][d] + so[1][d]) + (so[2][d] + so[3][d]);
    ((bf16*)p.out)[((int64_t)b * p.Hq + hq) * D + d] = (bf16)(sum / L);
  }
}

// Read-back: a workgroup per (sequence, K or V, head, 8192 / D output rows), two chunks of 16 elements a thread.  Bound by
// its 3 bytes an element; a head's rows are read next to each other, rows of an output are written D elements at a time.
// 3500 rows of 32 x 128 heads, 87 MB: 15.4 us, 5.6 TB/s (a thread per 8 elements with its own divisions: 21.4 us).
template <bool E4M3, int D>
__global__ __launch_bounds__(256) void kv8_read_k(KV8ReadParams p, int nrow) {
  constexpr int CH = D / 16, R = 8192 / D;
  const KV8& c = p.c;
  const int part = blockIdx.x % nrow;
  int id = blockIdx.x / nrow;
  const int h = id % c.Hkv;
  id /= c.Hkv;
  const bool is_k = id & 1;
  const int b = id >> 1;
  const int n = max(0, min(p.pos[b], c.Smax)), full = n >> c.lgT << c.lgT;
  const uint8_t* code = (const uint8_t*)(is_k ? c.kc : c.vc) + (int64_t)b * c.c_sb + (int64_t)h * c.c_sh;
  const float* scale = (is_k ? c.ks : c.vs) + (int64_t)b * c.s_sb + (int64_t)h * c.s_sh;
  const bf16* tail = (const bf16*)(is_k ? c.kt : c.vt) + (int64_t)b * c.t_sb + (int64_t)h * c.t_sh;
  bf16* out = (bf16*)(is_k ? p.ko : p.vo) + (int64_t)b * p.o_sb + (int64_t)h * p.o_sh;
  const int ch = threadIdx.x % CH;
  int s[2], t[2];
  u32x4 raw[2] = {};
  float sc[2] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s[i] = part * R + i * (R / 2) + (int)threadIdx.x / CH;
    t[i] = n - p.count + s[i];
  }
  if (full > 0) {   // whole workgroup: rows that are not codes read the nearest ones
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = max(0, min(t[i], full - 1));
      raw[i] = *reinterpret_cast<const u32x4*>(code + (int64_t)r * c.c_ss + ch * 16);
      sc[i] = scale[(int64_t)(r >> c.lgT) * c.s_sn];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (s[i] >= p.count) continue;
    bf16x8 o[2] = {};
    if (t[i] >= full) {
      const bf16* src = tail + (int64_t)(t[i] - full) * c.t_ss + ch * 16;
      o[0] = *reinterpret_cast<const bf16x8*>(src);
      o[1] = *reinterpret_cast<const bf16x8*>(src + 8);
    } else if (t[i] >= 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float f[4];
        unpack4<E4M3>(raw[i][k], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k >> 1][4 * (k & 1) + e] = (bf16)(f[e] * sc[i]);
      }
    }
    bf16* dst = out + (int64_t)s[i] * p.o_ss + ch * 16;
    *reinterpret_cast<bf16x8*>(dst) = o[0];
    *reinterpret_cast<bf16x8*>(dst + 8) = o[1];
  }
}

}  // namespace

void kv8_append(const KV8AppendParams& p, hipStream_t st) {
  const KV8& c = p.c;
  if (c.B == 0 || p.S == 0) return;
  const int nblk = (p.S + c.T - 2) / c.T + 1;   // blocks that S rows can touch, whatever their first position
  const int quant = c.B * 2 * c.Hkv * nblk;
  const dim3 grid((unsigned)(quant + c.B * p.S));
#define DPH_KV8_APP(E_, NC_) hipLaunchKernelGGL((kv8_append_k<E_, NC_>), grid, dim3(256), 0, st, p, nblk, quant)
#define DPH_KV8_APP_E(NC_)               \
  do {                                   \
    if (c.e4m3) DPH_KV8_APP(true, NC_);  \
    else DPH_KV8_APP(false, NC_);        \
  } while (0)
  const int chunks = c.T << c.lgC;   // 16-B chunks of one block, in registers: at most 8 a thread
  if (chunks <= 256) DPH_KV8_APP_E(1);
  else if (chunks <= 512) DPH_KV8_APP_E(2);
  else if (chunks <= 1024) DPH_KV8_APP_E(4);
  else DPH_KV8_APP_E(8);
#undef DPH_KV8_APP_E
#undef DPH_KV8_APP
}

// Workgroups of a call: two to a CU (what the registers allow at once; memory is busy with them), or one for each turn that
// the longest sequences could have.
int kv8_decode_workgroups(int64_t turns) { return (int)std::min<int64_t>(turns, 512); }

void kv8_decode_attention(const KV8DecodeParams& p, hipStream_t st) {
  const KV8& c = p.c;
  if (c.B == 0) return;
  const dim3 grid((unsigned)p.wgs);
#define DPH_KV8_DEC(D_)                                                                          \
  do {                                                                                           \
    if (c.e4m3) hipLaunchKernelGGL((kv8_decode_k<true, D_>), grid, dim3(256), 0, st, p);         \
    else hipLaunchKernelGGL((kv8_decode_k<false, D_>), grid, dim3(256), 0, st, p);               \
    if (p.opart) hipLaunchKernelGGL(kv8_combine_k<D_>, dim3((unsigned)(c.B * p.Hq)), dim3(256), 0, st, p); \
  } while (0)
  if (c.D == 128) DPH_KV8_DEC(128);
  else if (c.D == 64) DPH_KV8_DEC(64);
  else DPH_KV8_DEC(32);
#undef DPH_KV8_DEC
}

void kv8_read(const KV8ReadParams& p, hipStream_t st) {
  const KV8& c = p.c;
  if (c.B == 0 || p.count == 0) return;
  const int nrow = (int)cdiv((int64_t)p.count * c.D, 8192);
  const dim3 grid((unsigned)((int64_t)nrow * c.Hkv * 2 * c.B));
#define DPH_KV8_READ(D_)                                                                              \
  do {                                                                                                \
    if (c.e4m3) hipLaunchKernelGGL((kv8_read_k<true, D_>), grid, dim3(256), 0, st, p, nrow);          \
    else hipLaunchKernelGGL((kv8_read_k<false, D_>), grid, dim3(256), 0, st, p, nrow);                \
  } while (0)
  if (c.D == 128) DPH_KV8_READ(128);
  else if (c.D == 64) DPH_KV8_READ(64);
  else DPH_KV8_READ(32);
#undef DPH_KV8_READ
}

}  // namespace dph
