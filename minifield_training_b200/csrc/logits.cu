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
// counts must not cost a pass of their own over a [B, V] table in HBM. A CTA
// owns one contiguous tile of a row's vocabulary with a 32-bit word per token in
// shared memory:
//   bits 0-19   made(t)
//   bit  20     t occurs in the prompt part
//   bits 21-31  index + 1 of the last bias entry for t
// Every CTA of a row reads the whole history (it stays in L2) and counts the ids
// of its tile, by integer adds and ors: any order gives the same words. Then it
// streams its tile. Sharing the history among a cluster of CTAs that add to one
// another's words through distributed shared memory measured 6 to 100 % slower
// at every length tried (64 rows of 65536: 300 ids 10.4 against 10.0 us, 4096
// 16.5 against 11.2, 65536 111 against 56): the two cluster barriers and the
// remote adds cost more than the repeated reads. What bounds 64 rows with 4096
// ids (10.35 us, floor 4.1) is one wave of CTAs whose phases -- load, clear, count,
// stream -- follow one another: the issue slots are busy 29 % of the time, 5.5 of
// the 14.7 cycles between a warp's instructions go to outstanding loads. The
// history is the smaller part: 300 ids take 10.0 us.
#include <algorithm>

#include "types16.cuh"

namespace mfb {
namespace lgt {

constexpr int THREADS = 256;
constexpr int PER_SM = 4;         // CTAs on an SM
constexpr int TILE = 8192;        // tokens per CTA at most: PER_SM x 32 KB of words
constexpr int MIN_TILE = 8 * THREADS;
constexpr int MAX_VOCABULARY = 1 << 24;
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

// Eight logits as loaded, and as FP32.
template <typename T>
struct Raw {
  uint4 v;
  __device__ __forceinline__ void load(const void* base, long long at) {
    v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
  }
  __device__ __forceinline__ void get(float* x) const { unpack16x8<T>(v, x); }
};
template <>
struct Raw<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* base, long long at) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    a = p[0];
    b = p[1];
  }
  __device__ __forceinline__ void get(float* x) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
template <typename T>
__device__ __forceinline__ float load1(const void* base, long long at) {
  return Num16<T>::unpack2(static_cast<const uint16_t*>(base)[at]).x;
}
template <>
__device__ __forceinline__ float load1<float>(const void* base, long long at) {
  return static_cast<const float*>(base)[at];
}

struct Row {
  float rep, inv_rep, freq, pres;
  const float* bias;
};

// x / repetition as a product with the row's rounded reciprocal.
__device__ __forceinline__ float control(float x, uint32_t w, const Row& r) {
  x = w & kSeen ? x * (x > 0.f ? r.inv_rep : r.rep) : x;
  const float made = (float)(w & kMade);
  // Not 0 x frequency elsewhere: an infinite penalty would make a NaN of it.
  return made > 0.f ? fmaf(-r.freq, made, x) - r.pres : x;
}

constexpr int AHEAD = 4;  // vectors per thread whose loads precede the table's work

// grid (tiles, rows). TABLE: with a history or biases. Everything that does not
// depend on the words -- logits, mask words, the first history entries -- is
// loaded before they are built: a row is a chain of latencies, not of bytes.
template <typename T, bool TABLE>
__global__ void __launch_bounds__(THREADS, PER_SM) logits_kernel(Params p) {
  extern __shared__ __align__(16) uint32_t words[];
  const int b = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x;
  const long long row = (long long)b * p.V;
  const int t0 = rank * p.tile, t1 = min(p.V, t0 + p.tile);
  // Vectors of 8 start where the row's element offset is a multiple of 8, so
  // that both the logits and the output are 16-byte aligned whatever V is; the
  // words of a tile are shifted by the same amount.
  const int shift = (int)(row & 7);
  const int a0 = max(t0, min(t1, t0 + ((8 - shift) & 7))), nvec = max(0, t1 - a0) >> 3, a1 = a0 + nvec * 8;
  const uint32_t* mask = nullptr;
  const int W = (p.V + 31) >> 5;
  if (p.mask) {
    const int m = p.mask_rows ? p.mask_rows[b] : b;
    if ((unsigned)m < (unsigned)p.mask_count) mask = p.mask + (long long)m * W;
  }
  auto mask_bits = [&](int c) {
    const int wi = c >> 5;
    return mask ? __funnelshift_r(mask[wi], wi + 1 < W ? mask[wi + 1] : 0u, c & 31) : 0xFFFFFFFFu;
  };
  Raw<T> raw[AHEAD];
  uint32_t bits[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int v = tid + i * THREADS;
    if (v < nvec) {
      raw[i].load(p.logits, row + a0 + 8 * v);
      bits[i] = mask_bits(a0 + 8 * v);
    }
  }
  Row r{1.f, 1.f, 0.f, 0.f, nullptr};
  if (TABLE) {
    const int* hist = p.history + (long long)b * p.L;
    const int used = !p.history ? 0 : p.history_len ? min(max(p.history_len[b], 0), p.L) : p.L;
    const int prompt = p.prompt_len ? min(max(p.prompt_len[b], 0), used) : 0;
    if (p.repetition) r.rep = p.repetition[b];
    r.inv_rep = __fdiv_rn(1.f, r.rep);
    if (p.frequency) r.freq = p.frequency[b];
    if (p.presence) r.pres = p.presence[b];
    r.bias = p.bias_values + (long long)b * p.K;
    for (int i = tid; i < p.tile / 4 + 2; i += THREADS) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    constexpr int N = 8;  // entries whose loads are in flight
    int id[N];
    auto read = [&](int i0) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int i = i0 + k * THREADS;
        id[k] = i < p.L ? hist[i] : -1;
      }
    };
    if (p.history) read(tid);
    __syncthreads();
    for (int i0 = tid; i0 < used; i0 += N * THREADS) {
      if (i0 != tid) read(i0);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int i = i0 + k * THREADS;
        if (i < used && id[k] >= t0 && id[k] < t1) {
          uint32_t* w = words + (id[k] - t0 + shift);
          if (i < prompt) atomicOr(w, kPrompt);
          else atomicAdd(w, 1u);
        }
      }
    }
    __syncthreads();
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
  auto biased = [&](float x, uint32_t w) { return w >> 21 ? x + r.bias[(w >> 21) - 1] : x; };
  auto one = [&](int c) {
    float x = load1<T>(p.logits, row + c);
    if (TABLE) x = biased(control(x, words[c - t0 + shift], r), words[c - t0 + shift]);
    if (mask && !((mask[c >> 5] >> (c & 31)) & 1u)) x = -INFINITY;
    p.out[row + c] = x;
  };
  auto vector = [&](int c, const Raw<T>& in, uint32_t allowed) {
    float x[8];
    in.get(x);
    if (TABLE) {
      const uint4* w4 = reinterpret_cast<const uint4*>(words + (c - t0 + shift));
      const uint4 wa = w4[0], wb = w4[1];
      const uint32_t w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
      const uint32_t any = (wa.x | wa.y | wa.z | wa.w) | (wb.x | wb.y | wb.z | wb.w);
      if (any & kSeen) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = control(x[e], w[e], r);
      }
      if (any >> 21) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = biased(x[e], w[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (allowed >> e) & 1u ? x[e] : -INFINITY;
    float4* o = reinterpret_cast<float4*>(p.out + row + c);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  };
  if (tid < a0 - t0) one(t0 + tid);
  if (tid < t1 - a1) one(a1 + tid);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (tid + i * THREADS < nvec) vector(a0 + 8 * (tid + i * THREADS), raw[i], bits[i]);
  for (int v = tid + AHEAD * THREADS; v < nvec; v += THREADS) {
    raw[0].load(p.logits, row + a0 + 8 * v);
    vector(a0 + 8 * v, raw[0], mask_bits(a0 + 8 * v));
  }
}

template <typename T>
int launch(Params p, int B, cudaStream_t s) {
  // As many tiles per row as fill the GPU once, of MIN_TILE to TILE tokens in
  // whole 32-token groups.
  int dev = 0, sms = 148;
  MFB_CUDA_TRY(cudaGetDevice(&dev));
  MFB_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const int fill = std::min(std::max(1, PER_SM * sms / B), cdiv(p.V, MIN_TILE));
  p.tile = cdiv(cdiv(p.V, std::max(cdiv(p.V, TILE), fill)), 32) * 32;
  const dim3 grid(cdiv(p.V, p.tile), B);
  if (p.L || p.K) logits_kernel<T, true><<<grid, THREADS, sizeof(uint32_t) * ((size_t)p.tile + 8), s>>>(p);
  else logits_kernel<T, false><<<grid, THREADS, 0, s>>>(p);
  MFB_LAUNCH_CHECK("logits");
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
  MFB_CHECK_ARG(V <= lgt::MAX_VOCABULARY, "vocabulary %d above the supported %d", V, lgt::MAX_VOCABULARY);
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
