// Penalties for repeated tokens, biases and masks on the logits of a decode step (ops/logits.py), in one pass:
//   x = logit;  token in the history: x = x > 0 ? x / r : x * r;  c generated copies of it: x -= f c + p;  x += bias;
//   masked: x = -inf.
// A workgroup owns a segment of one row's vocabulary and counts that segment's tokens of the history in LDS -- integer
// atomics, so the order of arrival does not matter -- before it streams its logits through.
#include "dph_common.h"
#include "kernels.h"

namespace dph {

namespace {

constexpr int kSeg = 4096;
constexpr unsigned kInPrompt = 1u << 31;   // a count's top bit: the token stands in the prompt (counts are below 2^31)

template <typename T>
__global__ __launch_bounds__(256) void process_logits_k(LogitParams p, int nseg) {
  __shared__ unsigned cnt[kSeg];
  const int row = blockIdx.x / nseg, v0 = blockIdx.x % nseg * kSeg, nv = min(kSeg, p.V - v0);
  const int tid = threadIdx.x;
  if (p.tokens) {
    for (int i = tid; i < nv; i += 256) cnt[i] = 0;
    __syncthreads();
    const int len = max(0, min(p.lengths[row], p.L)), plen = p.prompt ? p.prompt[row] : 0;
    const int64_t* ids = p.tokens + (int64_t)row * p.ldt;
    for (int i = tid; i < len; i += 256) {
      const int64_t o = ids[i] - v0;   // ids outside the vocabulary (padding) fall into no segment
      if (o >= 0 && o < nv) {
        if (i < plen) atomicOr(&cnt[o], kInPrompt);
        else atomicAdd(&cnt[o], 1u);
      }
    }
    __syncthreads();
  }
  const float r = p.rep ? p.rep[row] : 1.f, f = p.freq ? p.freq[row] : 0.f, a = p.pres ? p.pres[row] : 0.f;
  const T* x = (const T*)p.x + (int64_t)row * p.ldx + v0;
  T* y = (T*)p.y + (int64_t)row * p.V + v0;
  for (int i = tid; i < nv; i += 256) {
    float z = (float)x[i];
    if (p.tokens) {
      const unsigned c = cnt[i], made = c & ~kInPrompt;
      if (c && p.rep) z = z > 0.f ? z / r : z * r;
      if (made) z -= f * (float)made + a;
    }
    const int v = v0 + i;
    if (p.bias) z += p.bias[(int64_t)row * p.ldb + v];
    if (p.mask && !((unsigned)p.mask[(int64_t)row * p.ldm + (v >> 5)] >> (v & 31) & 1u)) z = -INFINITY;
    y[i] = (T)z;
  }
}

}  // namespace

void process_logits(const LogitParams& p, int dtype, hipStream_t st) {
  if (p.N == 0 || p.V == 0) return;
  const int nseg = (int)cdiv(p.V, kSeg);
  const dim3 grid((unsigned)((int64_t)nseg * p.N));
  DPH_DISPATCH_FLOAT(dtype, T, hipLaunchKernelGGL(process_logits_k<T>, grid, dim3(256), 0, st, p, nseg));
}

}  // namespace dph
