// Logits of one decode step under the controls of their requests: penalties
// for repeated tokens, per-token biases and grammar masks, in one pass from
// the model's logits (bf16, fp16 or fp32) to the sampler's fp32.
//
// Row b, token t, with made(t) the occurrences of t in history[prompt_len,
// history_len) and seen(t) whether it occurs in history[0, history_len):
//   x = logit
//   x = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   x = x - frequency * made - presence * (made > 0)
//   x = x + bias(t)          (of entries with the same id the last one counts)
//   x = allowed(t) ? x : -inf
//
// The floor is the logits read and the fp32 row written once; the occurrence
// counts must not cost a pass of their own over a [B, V] table in HBM. A
// cluster of up to 8 CTAs owns a row, each CTA one contiguous tile of the
// vocabulary with a 32-bit word per token in shared memory:
//   bits 0-19   made(t)
//   bit  20     t occurs in the prompt part
//   bits 21-31  index + 1 of the last bias entry for t
// The cluster's CTAs each read an equal share of the history once and add to
// the word's owner through distributed shared memory (integer adds and ors:
// any order gives the same words), then every CTA streams its tile.
#include <algorithm>

#include "tc.cuh"
#include "types16.cuh"

namespace mfb {
namespace lgt {

constexpr int THREADS = 512;
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_TILE = 49152;  // tokens per CTA: 192 KB of words
constexpr int MAX_HISTORY = (1 << 20) - 1;
constexpr int MAX_BIAS = 2047;
constexpr uint32_t kMade = (1u << 20) - 1, kPrompt = 1u << 20, kSeen = kMade | kPrompt;

struct Params {
  const void* logits;
  const int* history;
  const int* prompt_len;
  const int* history_len;
  const float* repetition;
  const float* frequency;
  const float* presence;
  const int* bias_ids;
  const float* bias_values;
  const uint32_t* mask;
  const int* mask_rows;
  float* out;
  int V, L, K, mask_count, tile;
};

template <typename T>
__device__ __forceinline__ void load8(const void* base, long long at, float* x) {
  unpack16x8<T>(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at), x);
}
template <>
__device__ __forceinline__ void load8<float>(const void* base, long long at, float* x) {
  const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
  const float4 a = p[0], b = p[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ float load1(const void* base, long long at) {
  return Num16<T>::unpack2(static_cast<const uint16_t*>(base)[at]).x;
}
template <>
__device__ __forceinline__ float load1<float>(const void* base, long long at) {
  return static_cast<const float*>(base)[at];
}

__device__ __forceinline__ void cluster_add(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;\n" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_or(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;\n" ::"r"(addr), "r"(v) : "memory");
}

struct Row {
  float rep, freq, pres;
  const float* bias;
};

__device__ __forceinline__ float control(float x, uint32_t w, const Row& r) {
  if (w == 0) return x;
  if (w & kSeen) x = x > 0.f ? __fdiv_rn(x, r.rep) : x * r.rep;
  const uint32_t made = w & kMade;
  if (made) x = fmaf(-r.freq, (float)made, x) - r.pres;
  const uint32_t slot = w >> 21;
  if (slot) x += r.bias[slot - 1];
  return x;
}

// grid (cluster, rows), cluster (gridDim.x, 1, 1) when TABLE.
template <typename T, bool TABLE>
__global__ void __launch_bounds__(THREADS) logits_kernel(Params p) {
  extern __shared__ __align__(16) uint32_t words[];
  const int b = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x;
  const long long row = (long long)b * p.V;
  const int t0 = rank * p.tile, t1 = min(p.V, t0 + p.tile);
  // Vectors of 8 start where the row's element offset is a multiple of 8, so
  // that both the logits and the output are 16-byte aligned whatever V is; the
  // words of a tile are shifted by the same amount.
  const int shift = (int)(row & 7);
  Row r{1.f, 0.f, 0.f, nullptr};
  if (TABLE) {
    for (int i = tid; i < p.tile / 4 + 2; i += THREADS) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    if (p.repetition) r.rep = p.repetition[b];
    if (p.frequency) r.freq = p.frequency[b];
    if (p.presence) r.pres = p.presence[b];
    r.bias = p.bias_values + (long long)b * p.K;
    tc::cluster_sync();
    if (p.history) {
      const int used = p.history_len ? min(max(p.history_len[b], 0), p.L) : p.L;
      const int prompt = p.prompt_len ? min(max(p.prompt_len[b], 0), used) : 0;
      const int* hist = p.history + (long long)b * p.L;
      const uint32_t base = smem_u32(words);
      for (int i = rank * THREADS + tid; i < used; i += gridDim.x * THREADS) {
        const int id = hist[i];
        if ((unsigned)id >= (unsigned)p.V) continue;
        const int owner = id / p.tile;
        const uint32_t at = tc::mapa_shared(base + 4u * (uint32_t)(id - owner * p.tile + shift), owner);
        if (i < prompt) cluster_or(at, kPrompt);
        else cluster_add(at, 1u);
      }
    }
    tc::cluster_sync();
    if (p.K) {
      const int* ids = p.bias_ids + (long long)b * p.K;
      for (int i = tid; i < p.K; i += THREADS) {
        const int id = ids[i];
        if (id < t0 || id >= t1) continue;
        uint32_t* w = words + (id - t0 + shift);
        // Only the slot field changes from here on: the largest slot wins.
        atomicMax(w, ((uint32_t)(i + 1) << 21) | (*reinterpret_cast<volatile uint32_t*>(w) & kSeen));
      }
      __syncthreads();
    }
  }
  const uint32_t* mask = nullptr;
  const int W = (p.V + 31) >> 5;
  if (p.mask) {
    const int m = p.mask_rows ? p.mask_rows[b] : b;
    if ((unsigned)m < (unsigned)p.mask_count) mask = p.mask + (long long)m * W;
  }
  auto one = [&](int c) {
    float x = load1<T>(p.logits, row + c);
    if (TABLE) x = control(x, words[c - t0 + shift], r);
    if (mask && !((mask[c >> 5] >> (c & 31)) & 1u)) x = -INFINITY;
    p.out[row + c] = x;
  };
  if (t0 >= t1) return;
  const int a0 = min(t1, t0 + ((8 - shift) & 7)), nvec = (t1 - a0) >> 3, a1 = a0 + nvec * 8;
  if (tid < a0 - t0) one(t0 + tid);
  if (tid < t1 - a1) one(a1 + tid);
  for (int i = tid; i < nvec; i += THREADS) {
    const int c = a0 + 8 * i;
    float x[8];
    load8<T>(p.logits, row + c, x);
    if (TABLE) {
      const uint4* w4 = reinterpret_cast<const uint4*>(words + (c - t0 + shift));
      const uint4 wa = w4[0], wb = w4[1];
      const uint32_t w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = control(x[e], w[e], r);
    }
    if (mask) {
      const int wi = c >> 5;
      const uint32_t bits = __funnelshift_r(mask[wi], wi + 1 < W ? mask[wi + 1] : 0u, c & 31);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (bits >> e) & 1u ? x[e] : -INFINITY;
    }
    float4* o = reinterpret_cast<float4*>(p.out + row + c);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

template <typename T>
int launch(const Params& base, int B, cudaStream_t s) {
  Params p = base;
  const bool table = p.history || p.K;
  // Tiles are whole 32-token groups; a cluster of 8 (the portable limit)
  // spreads one row's history and tile over as many SMs as a row can get.
  int c = std::min(MAX_CLUSTER, cdiv(p.V, 32));
  p.tile = cdiv(cdiv(p.V, c), 32) * 32;
  c = cdiv(p.V, p.tile);
  const size_t smem = table ? sizeof(uint32_t) * ((size_t)p.tile + 8) : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(c, B);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = table ? 1 : 0;
  if (table) {
    MFB_CUDA_TRY(cudaFuncSetAttribute(logits_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)(sizeof(uint32_t) * (MAX_TILE + 8))));
    MFB_CUDA_TRY(cudaLaunchKernelEx(&cfg, logits_kernel<T, true>, p));
  } else {
    MFB_CUDA_TRY(cudaLaunchKernelEx(&cfg, logits_kernel<T, false>, p));
  }
  return MFB_OK;
}

}  // namespace lgt
}  // namespace mfb

using namespace mfb;

extern "C" int mfb_logits_process(const void* logits, int dtype, const int32_t* history, int history_capacity,
                                  const int32_t* prompt_len, const int32_t* history_len, const float* repetition,
                                  const float* frequency, const float* presence, const int32_t* bias_ids,
                                  const float* bias_values, int bias_count, const uint32_t* mask,
                                  const int32_t* mask_rows, int mask_count, float* out, int B, int V, void* stream) {
  MFB_CHECK_ARG(B > 0 && B <= 65535 && V > 0, "logits need 1 to 65535 rows and a vocabulary (B=%d V=%d)", B, V);
  MFB_CHECK_ARG(V <= lgt::MAX_CLUSTER * lgt::MAX_TILE, "vocabulary %d above the supported %d", V,
                lgt::MAX_CLUSTER * lgt::MAX_TILE);
  MFB_CHECK_ARG(dtype == MFB_DTYPE_BF16 || dtype == MFB_DTYPE_F16 || dtype == MFB_DTYPE_F32, "bad logits dtype");
  MFB_CHECK_ARG(logits && out, "NULL logits argument");
  MFB_CHECK_ARG((((uintptr_t)logits | (uintptr_t)out) & 15) == 0, "logits and out must be 16-byte aligned");
  MFB_CHECK_ARG(history_capacity >= 0 && history_capacity <= lgt::MAX_HISTORY && (history || !history_capacity),
                "history of %d tokens unsupported (0 to %d)", history_capacity, lgt::MAX_HISTORY);
  MFB_CHECK_ARG(bias_count >= 0 && bias_count <= lgt::MAX_BIAS && (!bias_count || (bias_ids && bias_values)),
                "%d bias entries unsupported (0 to %d, with ids and values)", bias_count, lgt::MAX_BIAS);
  MFB_CHECK_ARG(!mask || mask_rows || mask_count >= B, "a mask without row indices needs one row per logits row");
  MFB_CHECK_ARG(mask_count >= 0, "negative mask_count");
  lgt::Params p{};
  p.logits = logits;
  p.history = history_capacity ? history : nullptr;
  p.prompt_len = prompt_len;
  p.history_len = history_len;
  p.repetition = repetition;
  p.frequency = frequency;
  p.presence = presence;
  p.bias_ids = bias_ids;
  p.bias_values = bias_values;
  p.mask = mask;
  p.mask_rows = mask_rows;
  p.out = out;
  p.V = V;
  p.L = history_capacity;
  p.K = bias_count;
  p.mask_count = mask_count;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == MFB_DTYPE_BF16) return lgt::launch<__nv_bfloat16>(p, B, s);
  if (dtype == MFB_DTYPE_F16) return lgt::launch<__half>(p, B, s);
  return lgt::launch<float>(p, B, s);
}
