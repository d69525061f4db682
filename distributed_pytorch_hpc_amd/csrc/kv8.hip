// Block-scaled 8-bit KV cache of the serving path (ops/kv8.py): append, single-token decode attention, read-back.
//
// With one scale for every (block of T tokens, KV head) the codes follow the values' own range, so int8 or e4m3 entries
// need no calibration.  A block is quantised once, when it is full, from its bf16 rows:
//   scale = max(amax / QMAX, 2^-126),   code = round(x * (1 / scale)),   QMAX = 127 (int8) / 448 (e4m3)
// and the block that is still open stays in bf16, so what the cache holds after n tokens does not depend on how they
// were grouped into appends.  A block with an entry that is not finite gets the scale NaN and reads back as NaN.
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

template <bool E4M3>
__device__ __forceinline__ void unpack4(unsigned r, float (&o)[4]) {
  if constexpr (E4M3) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)r, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)r, true);
    o[0] = a[0]; o[1] = a[1]; o[2] = b[0]; o[3] = b[1];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (float)(int8_t)(r >> (8 * j));
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
  const int blk = pos / T + j, t0 = blk * T;
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
    const int o0 = n / T * T, from = max(o0, pos);
    for (int e = tid; e < (n - from) * CH; e += 256) {
      const int t = from + e / CH, ch = e % CH;
      *reinterpret_cast<bf16x8*>(tail + (int64_t)(t - o0) * c.t_ss + ch * 8) = fresh(t, ch);
    }
  }
}

// 8 elements of row t of the cache that holds n rows, in fp32
template <bool E4M3>
__device__ __forceinline__ void row8(const KV8& c, bool is_k, int b, int h, int t, int n, int ch, float (&o)[8]) {
  if (t < n / c.T * c.T) {
    const uint2 r = *reinterpret_cast<const uint2*>((const uint8_t*)(is_k ? c.kc : c.vc) + (int64_t)b * c.c_sb +
                                                    (int64_t)t * c.c_ss + (int64_t)h * c.c_sh + ch * 8);
    const float sc = (is_k ? c.ks : c.vs)[(int64_t)b * c.s_sb + (int64_t)(t / c.T) * c.s_sn + (int64_t)h * c.s_sh];
    float lo[4], hi[4];
    unpack4<E4M3>(r.x, lo);
    unpack4<E4M3>(r.y, hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k] = lo[k] * sc;
      o[4 + k] = hi[k] * sc;
    }
  } else {
    Vec8<bf16>::load((const bf16*)(is_k ? c.kt : c.vt) + (int64_t)b * c.t_sb + (int64_t)(t % c.T) * c.t_ss +
                         (int64_t)h * c.t_sh + ch * 8, o);
  }
}

// Decode attention, plain form: a workgroup per (sequence, query head), D / 8 lanes per key, online softmax per group
// of lanes, groups and waves merged at the end.
template <bool E4M3, int D>
__global__ __launch_bounds__(256) void kv8_decode_k(KV8DecodeParams p) {
  constexpr int CH = D / 8, GROUPS = 256 / CH;
  __shared__ float sm[GROUPS], sl[GROUPS], so[GROUPS][D];
  const KV8& c = p.c;
  const int hq = blockIdx.x, b = blockIdx.y, h = hq / (p.Hq / c.Hkv);
  const int g = threadIdx.x / CH, ch = threadIdx.x % CH;
  const int n = max(0, min(p.pos[b], c.Smax - 1) + 1);
  float q[8], acc[8] = {};
  Vec8<bf16>::load((const bf16*)p.q + (int64_t)b * p.q_sb + (int64_t)hq * D + ch * 8, q);
  float m = -INFINITY, l = 0.f;
  for (int t = g; t < n; t += GROUPS) {
    float k[8], v[8];
    row8<E4M3>(c, true, b, h, t, n, ch, k);
    row8<E4M3>(c, false, b, h, t, n, ch, v);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
    for (int o = CH / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    s *= p.scale * 1.4426950408889634f;
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
    const float a = exp2f(m - base), w = exp2f(s - base);
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * a + w * v[e];
    m = mn;   // a NaN score leaves m alone and makes l and acc NaN for good
  }
  if (ch == 0) { sm[g] = m; sl[g] = l; }
#pragma unroll
  for (int e = 0; e < 8; ++e) so[g][ch * 8 + e] = acc[e];
  __syncthreads();
  if ((int)threadIdx.x < D) {
    float M = -INFINITY;
    for (int i = 0; i < GROUPS; ++i) M = fmaxf(M, sm[i]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, o = 0.f;
    for (int i = 0; i < GROUPS; ++i) {
      const float w = exp2f(sm[i] - base);
      L += w * sl[i];
      o += w * so[i][threadIdx.x];
    }
    ((bf16*)p.out)[(int64_t)b * p.Hq * D + hq * D + threadIdx.x] = (bf16)(n > 0 ? o / L : 0.f);
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

void kv8_decode_attention(const KV8DecodeParams& p, hipStream_t st) {
  const dim3 grid((unsigned)p.Hq, (unsigned)p.c.B);
  if (p.c.B == 0) return;
#define DPH_KV8_DEC(D_)                                                                          \
  do {                                                                                           \
    if (p.c.e4m3) hipLaunchKernelGGL((kv8_decode_k<true, D_>), grid, dim3(256), 0, st, p);       \
    else hipLaunchKernelGGL((kv8_decode_k<false, D_>), grid, dim3(256), 0, st, p);               \
  } while (0)
  if (p.c.D == 128) DPH_KV8_DEC(128);
  else if (p.c.D == 64) DPH_KV8_DEC(64);
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
