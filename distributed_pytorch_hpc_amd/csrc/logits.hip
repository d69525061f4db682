// Penalties for repeated tokens, biases and masks on the logits of a decode step (ops/logits.py), in one pass:
//   x = logit;  token in the history: x = x > 0 ? x / r : x * r;  c generated copies of it: x -= f c + p;  x += bias;
//   masked: x = -inf.
// A workgroup owns a segment of one row's vocabulary and counts that segment's tokens of the history in LDS -- integer
// atomics, so the order of arrival does not matter -- between asking for its logits and using them.  No state is kept from
// call to call: reading the ids again costs 8 bytes a token of the history, a [N, V] table of counts 4 bytes a logit.
// Bound by latency (launch, ids, LDS) and then by memory: one row of 32 000 with 300 ids 3.4 us; 64 rows, bf16, 4000 ids
// each, bias and mask 7.9 us, 2.4 TB/s of its 19 MB; 64 rows of fp32 with a mask alone 6.2 us.  Loads under conditions of
// their own, each waiting for the last, took 23 us.
#include "dph_common.h"
#include "kernels.h"

namespace dph {

namespace {

constexpr unsigned kInPrompt = 1u << 31;   // a count's top bit: the token stands in the prompt (counts are below 2^31)

// CH elements as they lie in memory: conversions wait for the load, so they come after everything has been asked for
template <typename T, int CH> struct Chunk { T v[CH]; };
template <> struct Chunk<bf16, 8> { bf16x8 v; };
template <> struct Chunk<float, 8> {
  f32x4 a, b;
};
template <typename T, int CH>
__device__ __forceinline__ float get(const Chunk<T, CH>& c, int e) { return (float)c.v[e]; }
template <>
__device__ __forceinline__ float get<float, 8>(const Chunk<float, 8>& c, int e) { return e < 4 ? c.a[e] : c.b[e - 4]; }

template <typename T, int CH>
__device__ __forceinline__ void put(Chunk<T, CH>& c, int e, float v) { c.v[e] = (T)v; }
template <>
__device__ __forceinline__ void put<float, 8>(Chunk<float, 8>& c, int e, float v) {
  if (e < 4) c.a[e] = v;
  else c.b[e - 4] = v;
}

// 8 logits a thread, in one chunk where every row begins at 16 bytes (CH = 8), else one by one.  Segments of 2048: longer
// ones read the history less often but wait for their own tail (4096: 9.0, 2048: 8.4 us at 64 x 32 000, 4000 ids a row).
constexpr int kSeg = 2048;
template <typename T, int CH>
__global__ __launch_bounds__(256) void process_logits_k(LogitParams p, int nseg) {
  constexpr int NC = kSeg / 256 / CH;
  __shared__ __align__(16) unsigned cnt[kSeg];
  const int row = blockIdx.x / nseg, v0 = blockIdx.x % nseg * kSeg, nv = min(kSeg, p.V - v0);
  const int tid = threadIdx.x;
  const T* x = (const T*)p.x + (int64_t)row * p.ldx + v0;
  T* y = (T*)p.y + (int64_t)row * p.V + v0;
  // no load under a condition of its own: lanes past the row read its last chunk again (with CH = 8 the vocabulary is a
  // multiple of 8), absent operands are skipped by the whole grid
  Chunk<T, CH> xr[NC];
  Chunk<float, CH> br[NC];
  int mr[NC];
  auto at = [&](int k) { return min((k * 256 + tid) * CH, nv - CH); };
#pragma unroll
  for (int k = 0; k < NC; ++k) xr[k] = *reinterpret_cast<const Chunk<T, CH>*>(x + at(k));
  if (p.mask) {
    const int* m = p.mask + (int64_t)row * p.ldm;
#pragma unroll
    for (int k = 0; k < NC; ++k) mr[k] = m[(v0 + at(k)) >> 5];
  }
  if (p.bias) {
    const float* b = p.bias + (int64_t)row * p.ldb + v0;
#pragma unroll
    for (int k = 0; k < NC; ++k) br[k] = *reinterpret_cast<const Chunk<float, CH>*>(b + at(k));
  }
  float rep = 1.f, inv = 1.f, f = 0.f, a = 0.f;
  if (p.tokens) {
    const u32x4 zero = {0, 0, 0, 0};
    for (int i = tid; i < kSeg / 4; i += 256) *reinterpret_cast<u32x4*>(&cnt[4 * i]) = zero;
    const int len = max(0, min(p.lengths[row], p.L)), plen = p.prompt ? p.prompt[row] : 0;
    if (p.rep) {
      rep = p.rep[row];
      inv = 1.f / rep;   // x / r as x * (1 / r): one rounding more, and no division a logit
    }
    if (p.freq) f = p.freq[row];
    if (p.pres) a = p.pres[row];
    const int64_t* ids = p.tokens + (int64_t)row * p.ldt;
    __syncthreads();
    for (int i0 = tid; i0 < len; i0 += 256 * 8) {   // eight loads in flight
      int64_t id[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) id[u] = ids[min(i0 + 256 * u, len - 1)];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t o = id[u] - v0;   // ids outside the vocabulary (padding) fall into no segment
        if (i0 + 256 * u < len && o >= 0 && o < nv) {
          if (i0 + 256 * u < plen) atomicOr(&cnt[o], kInPrompt);
          else atomicAdd(&cnt[o], 1u);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int i = (k * 256 + tid) * CH;
    if (i >= nv) continue;
    const unsigned allowed = p.mask ? (unsigned)mr[k] >> ((v0 + i) & 31) : ~0u;
    Chunk<T, CH> o;
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      float w = get(xr[k], e);
      const unsigned c = p.tokens ? cnt[i + e] : 0u;
      if (c) {
        w *= w > 0.f ? inv : rep;
        const unsigned made = c & ~kInPrompt;
        if (made) w -= f * (float)made + a;
      }
      if (p.bias) w += get(br[k], e);
      put(o, e, allowed >> e & 1u ? w : -INFINITY);
    }
    *reinterpret_cast<Chunk<T, CH>*>(y + i) = o;
  }
}

}  // namespace

void process_logits(const LogitParams& p, int dtype, hipStream_t st) {
  if (p.N == 0 || p.V == 0) return;
  auto aligned = [](const void* b, int64_t ld, int bytes) {
    return reinterpret_cast<uintptr_t>(b) % 16 == 0 && ld * bytes % 16 == 0;
  };
  const int es = dtype == kBF16 ? 2 : 4;
  const bool vec = p.V % 8 == 0 && aligned(p.x, p.ldx, es) && aligned(p.bias, p.ldb, 4);
  const int nseg = (int)cdiv(p.V, kSeg);
  const dim3 grid((unsigned)((int64_t)nseg * p.N));
#define DPH_LOGITS(T_)                                                                                          \
  do {                                                                                                          \
    if (vec) hipLaunchKernelGGL((process_logits_k<T_, 8>), grid, dim3(256), 0, st, p, nseg);                    \
    else hipLaunchKernelGGL((process_logits_k<T_, 1>), grid, dim3(256), 0, st, p, nseg);                        \
  } while (0)
  if (dtype == kBF16) DPH_LOGITS(bf16);
  else DPH_LOGITS(float);
#undef DPH_LOGITS
}

}  // namespace dph
