// Penalties for repeated tokens, biases and masks on the logits of a decode step (ops/logits.py), in one pass:
//   x = logit;  token in the history: x = x > 0 ? x / r : x * r;  c generated copies of it: x -= f c + p;  x += bias;
//   masked: x = -inf.
// A workgroup owns a segment of one row's vocabulary and counts that segment's tokens of the history in LDS -- integer
// atomics, so the order of arrival does not matter -- between asking for its logits and using them.  No state is kept from
// call to call, so no [N, V] table of counts has to follow a request through its slot.  The price: every segment of a row
// reads the row's ids again, 8 bytes each, 4 (1024 threads) or 16 times (256) at V = 32 000, mostly from L2; at 4000 ids
// that is the 128 kB that a row of such a table has, or four times as much.
// Bound by latency (launch, lengths, ids, LDS and two barriers, one after the other) and then by memory: one row of 32 000
// with 300 ids 3.6 us; 64 rows, bf16, 4000 ids each, bias and mask 7.2 us, 2.6 TB/s of its 19 MB, of which the history is
// about 1 us: 64 rows of fp32 with a mask alone take 6.2 us (replays of captured calls).  Loads under conditions of
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

// 8 logits a thread, in one chunk where every row begins at 16 bytes (CH = 8), else one by one: a segment of 8 * NT.
template <typename T, int CH, int NT>
__global__ __launch_bounds__(NT) void process_logits_k(LogitParams p, int nseg) {
  constexpr int NC = 8 / CH, SEG = 8 * NT;
  __shared__ __align__(16) unsigned cnt[SEG];
  const int row = blockIdx.x / nseg, v0 = blockIdx.x % nseg * SEG, nv = min(SEG, p.V - v0);
  const int tid = threadIdx.x;
  const T* x = (const T*)p.x + (int64_t)row * p.ldx + v0;
  T* y = (T*)p.y + (int64_t)row * p.V + v0;
  // no load under a condition of its own: lanes past the row read its last chunk again (with CH = 8 the vocabulary is a
  // multiple of 8), absent operands are skipped by the whole grid
  Chunk<T, CH> xr[NC];
  Chunk<float, CH> br[NC];
  int mr[NC];
  auto at = [&](int k) { return min((k * NT + tid) * CH, nv - CH); };
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
  float rep = 1.f, inv = 1.f, unit = 1.f, f = 0.f, a = 0.f;
  if (p.tokens) {
    const u32x4 zero = {0, 0, 0, 0};
    for (int i = tid; i < SEG / 4; i += NT) *reinterpret_cast<u32x4*>(&cnt[4 * i]) = zero;
    const int len = max(0, min(p.lengths[row], p.L)), plen = p.prompt ? p.prompt[row] : 0;
    if (p.rep) {
      rep = p.rep[row];
      // x / r as x * (1 / r): one rounding more, and no division a logit; x * (1 / (r u)) * u where 1 / r could be infinite
      // or lose digits (a division there instead took 0.2 us of every call)
      unit = fabsf(rep) < 0x1p-64f ? 0x1p64f : fabsf(rep) > 0x1p64f ? 0x1p-64f : 1.f;
      inv = 1.f / (rep * unit);
    }
    if (p.freq) f = p.freq[row];
    if (p.pres) a = p.pres[row];
    const int64_t* ids = p.tokens + (int64_t)row * p.ldt;
    __syncthreads();
    for (int i0 = tid; i0 < len; i0 += NT * 8) {   // eight loads in flight
      int64_t id[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) id[u] = ids[min(i0 + NT * u, len - 1)];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t o = id[u] - v0;   // ids outside the vocabulary (padding) fall into no segment
        if (i0 + NT * u < len && o >= 0 && o < nv) {
          if (i0 + NT * u < plen) atomicOr(&cnt[o], kInPrompt);
          else atomicAdd(&cnt[o], 1u);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int i = (k * NT + tid) * CH;
    if (i >= nv) continue;
    const unsigned allowed = p.mask ? (unsigned)mr[k] >> ((v0 + i) & 31) : ~0u;
    Chunk<T, CH> o;
#pragma unroll
    for (int e = 0; e < CH; ++e) {
      float w = get(xr[k], e);
      const unsigned c = p.tokens ? cnt[i + e] : 0u;
      if (c) {
        w = w > 0.f ? w * inv * unit : w * rep;
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
  // Every segment of a row reads the whole history: with 1024 threads there are a quarter as many, but few rows fill the
  // card worse and a workgroup waits for more.  Measured (us, 256 / 1024 threads, bf16, bias and mask, V = 32 000):
  //   1 row:   300 ids 3.4 / 4.6,  4000 4.3 / 5.0,  8000 5.0 / 5.1,  32 768 10.9 / 7.8
  //   16 rows: 300 ids 3.6 / 4.6,  4000 4.6 / 5.2,  8000 6.2 / 5.3,  32 768 16.3 / 8.5
  //   64 rows: 300 ids 6.4 / 5.9,  4000 8.2 / 7.1,  8000 10.2 / 7.7, 32 768 22.6 / 14.4
  // and 64 rows without a history 6.2 / 6.4.
  // A grid holds fewer than 2^32 threads: rows too many for 1024 each (the caller bounds N for 256) take the narrow form.
  const bool wide = p.tokens && (p.L >= 6144 || (int64_t)p.N * p.V >= 3 << 19) &&
                    (int64_t)p.N * cdiv(p.V, 8 * 1024) < int64_t(1) << 22;
#define DPH_LOGITS(T_, CH_, NT_)                                                                                       \
  do {                                                                                                                 \
    const int nseg = (int)cdiv(p.V, 8 * NT_);                                                                          \
    hipLaunchKernelGGL((process_logits_k<T_, CH_, NT_>), dim3((unsigned)((int64_t)nseg * p.N)), dim3(NT_), 0, st, p,   \
                       nseg);                                                                                          \
  } while (0)
#define DPH_LOGITS_T(T_)                                      \
  do {                                                        \
    if (vec && wide) DPH_LOGITS(T_, 8, 1024);                 \
    else if (vec) DPH_LOGITS(T_, 8, 256);                     \
    else if (wide) DPH_LOGITS(T_, 1, 1024);                   \
    else DPH_LOGITS(T_, 1, 256);                              \
  } while (0)
  if (dtype == kBF16) DPH_LOGITS_T(bf16);
  else DPH_LOGITS_T(float);
#undef DPH_LOGITS_T
#undef DPH_LOGITS
}

}  // namespace dph
