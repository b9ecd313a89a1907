// Head norm and rotary position of a fused q|k|v projection, forward and
// backward, and the same pass with the keys and values appended to a paged
// cache.
//
// For one head vector x of D values at position p:
//   n = x / sqrt(mean(x^2) + eps),  u = w n   (without gains: u = x)
//   y = R(p) u: the first `rotary_dim` values are rotated in pairs by the
//   angle p * freqs[i], pair i being (i, i + rotary_dim / 2) in the half
//   layout and (2i, 2i + 1) in the interleaved one; cos and sin are scaled by
//   `amplitude`; the remaining values pass through.
// Backward: du = R(p)^T dy, dw = sum over tokens and heads of du n,
//   dx = (w du - n mean(w du n)) / sqrt(mean(x^2) + eps).
// Everything is computed in FP32 from the 16-bit inputs and rounded once, at
// the store. Angles are formed in FP64 as a fraction of a turn: at position
// 2^20 an FP32 product is off by up to 2^-4 rad, the FP64 one by less than
// 2^-20 for any int32 position.
//
// Layout: a warp owns a token (or one of `slices` interleaved shares of its
// heads, for calls with few tokens) and D/8 lanes own a head, 8 values (16
// bytes) each, so every load and store is a full 128-byte line or more. The
// warp computes each of the token's rotary_dim/2 angles once, keeps them in
// shared memory and reads back the lane's own; a half-layout partner is
// rotary_dim/16 lanes away (shuffle), an interleaved one in the same lane.
#include <algorithm>

#include "types16.cuh"

namespace mfb {
namespace rot {

constexpr int WARPS = 8;
constexpr int MAX_D = 128;
constexpr int BWD_GRID_MAX = 4 * 160;  // bounds the gain-gradient partials
constexpr double kInvTwoPi = 0.15915494309189533577;

struct Params {
  const uint16_t* qkv;
  const float* wq;
  const float* wk;
  const float* freqs;
  uint16_t* q;
  uint16_t* k;  // k [M, Hk, D], or the key pages
  uint16_t* v;
  const int* positions;
  // Paged append: tokens [cu_q[b], cu_q[b + 1]) are the last ones of sequence b.
  const int* cu_q;
  const int* seq_lens;
  const int* page_table;
  int B, max_pages, num_pages, page_shift;
  long long page_stride;
  int token_stride, head_stride;
  // Backward.
  const uint16_t* dq;
  const uint16_t* dk;
  const uint16_t* dv;
  uint16_t* dqkv;
  float* partial;  // [grid][2][D]
  int ld, M, H, Hk, rotary_dim, slices;
  float amplitude, eps;
};

// cos and sin of a position's angles: lane-parallel, one per pair, into the
// warp's table; then this lane's own into c / s (1 and 0 where not rotated).
// Half layout: values sub*8 + e use pair (sub*8 + e) mod (rotary_dim / 2).
// Interleaved: values 2j and 2j + 1 use pair sub*4 + j.
template <bool IL>
__device__ __forceinline__ void angles(const Params& p, int pos, float2* table, int lane, int sub, float* c, float* s) {
  const int half = p.rotary_dim >> 1;
  __syncwarp();
  for (int i = lane; i < half; i += 32) {
    const double t = (double)pos * (double)p.freqs[i] * kInvTwoPi;
    float sn, cs;
    sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
    table[i] = make_float2(cs * p.amplitude, sn * p.amplitude);
  }
  __syncwarp();
  if (sub * 8 < p.rotary_dim) {
    if (IL) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = table[sub * 4 + j];
        c[2 * j] = c[2 * j + 1] = f.x;
        s[2 * j] = s[2 * j + 1] = f.y;
      }
    } else {
      const int base = sub * 8 < half ? sub * 8 : sub * 8 - half;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 f = table[base + e];
        c[e] = f.x;
        s[e] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 1.f, s[e] = 0.f;
  }
}

// x <- R x, or R^T x for INV (the angles negated). `from` is the lane holding
// the half-layout partners (this lane itself where nothing is rotated), `low`
// whether this lane holds the first of each pair.
template <bool IL, bool INV>
__device__ __forceinline__ void rotate(float* x, const float* c, const float* s, int from, bool low) {
  if (IL) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = x[2 * j], b = x[2 * j + 1], sn = INV ? -s[2 * j] : s[2 * j];
      x[2 * j] = a * c[2 * j] - b * sn;
      x[2 * j + 1] = b * c[2 * j] + a * sn;
    }
  } else {
    const bool minus = low != INV;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float o = __shfl_sync(0xffffffffu, x[e], from);
      x[e] = fmaf(minus ? -o : o, s[e], x[e] * c[e]);
    }
  }
}

template <int L>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sequence of token t: the last b with cu_q[b] <= t.
__device__ __forceinline__ int sequence_of(const int* cu_q, int B, int t) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu_q[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T, int D, bool IL, bool PAGED>
__global__ void __launch_bounds__(32 * WARPS) rotary_fwd_kernel(Params p) {
  constexpr int L = D / 8, HPW = 32 / L;  // lanes per head, heads per warp
  __shared__ float2 tables[WARPS][MAX_D / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, grp = lane / L;
  const int half8 = p.rotary_dim >> 4;  // lanes of half a rotated part
  const bool turned = sub * 8 < p.rotary_dim, low = sub < half8;
  const int from = turned ? (low ? lane + half8 : lane - half8) : lane;
  const bool norm = p.wq != nullptr;
  float wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    wq[e] = norm ? p.wq[sub * 8 + e] : 1.f;
    wk[e] = norm ? p.wk[sub * 8 + e] : 1.f;
  }
  const int heads = p.H + (p.v ? 2 : 1) * p.Hk;
  const long long units = (long long)p.M * p.slices, step = (long long)gridDim.x * WARPS;
  for (long long u = (long long)blockIdx.x * WARPS + warp; u < units; u += step) {
    const int row = (int)(u / p.slices), slice = (int)(u % p.slices);
    const uint16_t* src = p.qkv + (long long)row * p.ld + sub * 8;
    // Four heads' loads in flight before the first is used.
    int h = slice * HPW + grp;
    const int hstep = p.slices * HPW;
    uint4 buf[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (h + i * hstep < heads) buf[i] = *reinterpret_cast<const uint4*>(src + (long long)(h + i * hstep) * D);
    int pos;
    long long slot = -1;  // element offset of the token's first head in the pages; -1: not stored
    if (PAGED) {
      if (row < p.cu_q[0] || row >= p.cu_q[p.B]) continue;  // padding: left as it was
      const int b = sequence_of(p.cu_q, p.B, row);
      pos = p.seq_lens[b] - (p.cu_q[b + 1] - row);
      const int pg = pos >> p.page_shift;
      if (pos >= 0 && pg < p.max_pages) {
        const int id = p.page_table[(long long)b * p.max_pages + pg];
        if ((unsigned)id < (unsigned)p.num_pages)
          slot = (long long)id * p.page_stride + (long long)(pos - (pg << p.page_shift)) * p.token_stride;
      }
    } else {
      pos = p.positions[row];
    }
    float c[8], s[8];
    angles<IL>(p, pos, tables[warp], lane, sub, c, s);
    // The warp's heads in steps; a step past the end runs on for its shuffles.
    for (int h0 = slice * HPW; h0 < heads; h0 += 4 * hstep) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (h0 + i * hstep >= heads) break;
        const int hh = h0 + i * hstep + grp;
        const bool live = hh < heads;
        const uint4 raw = live ? buf[i] : make_uint4(0, 0, 0, 0);
        const int next = hh + 4 * hstep;
        if (next < heads) buf[i] = *reinterpret_cast<const uint4*>(src + (long long)next * D);
        const bool is_q = hh < p.H, is_k = !is_q && hh < p.H + p.Hk;
        float x[8];
        unpack16x8<T>(raw, x);
        if (norm) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
          const float r = rsqrtf(head_sum<L>(ss) * (1.f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= r * (is_q ? wq[e] : wk[e]);
        }
        rotate<IL, false>(x, c, s, from, low);
        if (!live) continue;
        if (is_q) {
          *reinterpret_cast<uint4*>(p.q + ((long long)row * p.H + hh) * D + sub * 8) = pack16x8<T>(x);
        } else {
          const int kh = is_k ? hh - p.H : hh - p.H - p.Hk;
          uint16_t* dst = is_k ? p.k : p.v;
          const uint4 out = is_k ? pack16x8<T>(x) : raw;
          if (!PAGED) *reinterpret_cast<uint4*>(dst + ((long long)row * p.Hk + kh) * D + sub * 8) = out;
          else if (slot >= 0) *reinterpret_cast<uint4*>(dst + slot + (long long)kh * p.head_stride + sub * 8) = out;
        }
      }
    }
  }
}

template <typename T, int D, bool IL>
__global__ void __launch_bounds__(32 * WARPS) rotary_bwd_kernel(Params p) {
  constexpr int L = D / 8, HPW = 32 / L;
  __shared__ float2 tables[WARPS][MAX_D / 2];
  __shared__ float sums[WARPS][2 * D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, grp = lane / L;
  const int half8 = p.rotary_dim >> 4;
  const bool turned = sub * 8 < p.rotary_dim, low = sub < half8;
  const int from = turned ? (low ? lane + half8 : lane - half8) : lane;
  const bool norm = p.wq != nullptr;
  float wq[8], wk[8], accq[8], acck[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    wq[e] = norm ? p.wq[sub * 8 + e] : 1.f;
    wk[e] = norm ? p.wk[sub * 8 + e] : 1.f;
    accq[e] = acck[e] = 0.f;
  }
  const int heads = p.H + 2 * p.Hk;
  const long long units = (long long)p.M * p.slices, step = (long long)gridDim.x * WARPS;
  for (long long u = (long long)blockIdx.x * WARPS + warp; u < units; u += step) {
    const int row = (int)(u / p.slices), slice = (int)(u % p.slices);
    const long long base = (long long)row * p.ld + sub * 8;
    const int hstep = p.slices * HPW;
    auto upstream = [&](int hh) {
      const uint16_t* g = hh < p.H ? p.dq + ((long long)row * p.H + hh) * D
                                   : (hh < p.H + p.Hk ? p.dk + ((long long)row * p.Hk + hh - p.H) * D
                                                      : p.dv + ((long long)row * p.Hk + hh - p.H - p.Hk) * D);
      return *reinterpret_cast<const uint4*>(g + sub * 8);
    };
    uint4 bg[2], bx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int hh = slice * HPW + grp + i * hstep;
      bg[i] = bx[i] = make_uint4(0, 0, 0, 0);
      if (hh < heads) bg[i] = upstream(hh);
      if (norm && hh < p.H + p.Hk) bx[i] = *reinterpret_cast<const uint4*>(p.qkv + base + (long long)hh * D);
    }
    float c[8], s[8];
    angles<IL>(p, p.positions[row], tables[warp], lane, sub, c, s);
    for (int h0 = slice * HPW; h0 < heads; h0 += 2 * hstep) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (h0 + i * hstep >= heads) break;
        const int hh = h0 + i * hstep + grp;
        const bool live = hh < heads;
        const uint4 graw = bg[i], xraw = bx[i];
        const int next = hh + 2 * hstep;
        if (next < heads) bg[i] = upstream(next);
        if (norm && next < p.H + p.Hk) bx[i] = *reinterpret_cast<const uint4*>(p.qkv + base + (long long)next * D);
        const bool is_q = hh < p.H, is_v = hh >= p.H + p.Hk;
        float g[8];
        unpack16x8<T>(graw, g);
        rotate<IL, true>(g, c, s, from, low);
        if (norm) {
          float x[8], ss = 0.f, dot = 0.f;
          unpack16x8<T>(xraw, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
          const float r = rsqrtf(head_sum<L>(ss) * (1.f / D) + p.eps);
          const bool add_q = live && is_q, add_k = live && !is_q && !is_v;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] *= r;
            const float gn = g[e] * x[e];
            accq[e] += add_q ? gn : 0.f;
            acck[e] += add_k ? gn : 0.f;
            g[e] *= is_q ? wq[e] : wk[e];
            dot = fmaf(g[e], x[e], dot);
          }
          const float mean = head_sum<L>(dot) * (1.f / D);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = r * fmaf(-x[e], mean, g[e]);
        }
        if (live) *reinterpret_cast<uint4*>(p.dqkv + base + (long long)hh * D) = is_v ? graw : pack16x8<T>(g);
      }
    }
  }
  if (p.partial == nullptr) return;
  // Gain gradients: heads of the warp, warps of the block, then one row of
  // partials per block for the column sum below -- all in a fixed order.
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int o = L; o < 32; o <<= 1) {
      accq[e] += __shfl_xor_sync(0xffffffffu, accq[e], o);
      acck[e] += __shfl_xor_sync(0xffffffffu, acck[e], o);
    }
    if (grp == 0) {
      sums[warp][sub * 8 + e] = accq[e];
      sums[warp][D + sub * 8 + e] = acck[e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += 32 * WARPS) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) t += sums[w][i];
    p.partial[(long long)blockIdx.x * 2 * D + i] = t;
  }
}

// dw[col] (+)= sum over `rows` partial rows; 32 columns per block, 32 row
// lanes, combined in a fixed tree. Columns [0, D) are wq's, [D, 2D) wk's.
__global__ void __launch_bounds__(1024) gain_sum_kernel(const float* __restrict__ partial, int rows, int D,
                                                        float* __restrict__ dwq, float* __restrict__ dwk,
                                                        int accumulate) {
  __shared__ float part[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  float t = 0.f;
  for (int r = y; r < rows; r += 32) t += partial[(long long)r * 2 * D + col];
  part[y][lane] = t;
  __syncthreads();
  t = warp_sum(part[lane][y]);  // row lane `lane` of column blockIdx.x * 32 + y
  if (lane == 0) {
    const int c = blockIdx.x * 32 + y;
    float* dst = c < D ? dwq + c : dwk + (c - D);
    *dst = accumulate ? *dst + t : t;
  }
}

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Shares of a token's heads: more than one where whole tokens would leave the
// GPU short of warps (each share computes the token's angles again).
int slices_for(int M, int groups, int sms) {
  int s = 1;
  while (s < 8 && s * 2 <= groups && (long long)M * s * 2 <= (long long)sms * 16) s *= 2;
  return s;
}

int check_common(const void* qkv, const float* wq, const float* wk, const float* freqs, int ld, int M, int H, int Hk,
                 int D, int rotary_dim, int dtype) {
  MFB_CHECK_ARG(M > 0 && H > 0 && Hk > 0, "rotary needs tokens and heads (M=%d H=%d Hk=%d)", M, H, Hk);
  MFB_CHECK_ARG(D == 64 || D == 128, "rotary head_dim %d unsupported (64 or 128)", D);
  MFB_CHECK_ARG((long long)(H + 2LL * Hk) * D <= 1 << 24, "too many heads (H=%d Hk=%d)", H, Hk);
  MFB_CHECK_ARG(ld >= (H + 2 * Hk) * D && ld % 8 == 0, "qkv rows need a stride of at least %d, a multiple of 8 (ld=%d)",
                (H + 2 * Hk) * D, ld);
  MFB_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 16 == 0,
                "rotary_dim %d must be a multiple of 16 up to head_dim", rotary_dim);
  MFB_CHECK_ARG(dtype == MFB_DTYPE_BF16 || dtype == MFB_DTYPE_F16, "rotary dtype must be bf16 or fp16");
  MFB_CHECK_ARG(qkv && (freqs || rotary_dim == 0), "NULL rotary argument");
  MFB_CHECK_ARG((wq == nullptr) == (wk == nullptr), "q and k gains must both be given or both be NULL");
  return MFB_OK;
}

template <typename T, int D, bool PAGED>
int launch_fwd(const Params& p, bool interleaved, int sms, cudaStream_t s) {
  const long long units = (long long)p.M * p.slices;
  const int grid = (int)std::min<long long>((units + WARPS - 1) / WARPS, 8LL * sms);
  if (interleaved) rotary_fwd_kernel<T, D, true, PAGED><<<grid, 32 * WARPS, 0, s>>>(p);
  else rotary_fwd_kernel<T, D, false, PAGED><<<grid, 32 * WARPS, 0, s>>>(p);
  MFB_LAUNCH_CHECK(PAGED ? "paged append" : "rotary fwd");
  return MFB_OK;
}

template <bool PAGED>
int dispatch_fwd(const Params& p, int D, bool interleaved, int dtype, int sms, cudaStream_t s) {
  if (dtype == MFB_DTYPE_BF16)
    return D == 64 ? launch_fwd<__nv_bfloat16, 64, PAGED>(p, interleaved, sms, s)
                   : launch_fwd<__nv_bfloat16, 128, PAGED>(p, interleaved, sms, s);
  return D == 64 ? launch_fwd<__half, 64, PAGED>(p, interleaved, sms, s)
                 : launch_fwd<__half, 128, PAGED>(p, interleaved, sms, s);
}

template <typename T, int D>
void launch_bwd(const Params& p, bool interleaved, int grid, cudaStream_t s) {
  if (interleaved) rotary_bwd_kernel<T, D, true><<<grid, 32 * WARPS, 0, s>>>(p);
  else rotary_bwd_kernel<T, D, false><<<grid, 32 * WARPS, 0, s>>>(p);
}

bool aligned16(std::initializer_list<const void*> ptrs) {
  uintptr_t a = 0;
  for (const void* x : ptrs) a |= (uintptr_t)x;
  return (a & 15) == 0;
}

}  // namespace rot
}  // namespace mfb

using namespace mfb;

extern "C" int mfb_qk_rotary_fwd(const void* qkv, int ld_qkv, const float* wq, const float* wk,
                                 const int32_t* positions, const float* freqs, void* q, void* k, void* v, int M, int H,
                                 int Hk, int D, int rotary_dim, int interleaved, int dtype, float amplitude, float eps,
                                 void* stream) {
  int st = rot::check_common(qkv, wq, wk, freqs, ld_qkv, M, H, Hk, D, rotary_dim, dtype);
  if (st) return st;
  MFB_CHECK_ARG(positions && q && k, "NULL rotary argument");
  MFB_CHECK_ARG(rot::aligned16({qkv, q, k, v}), "qkv, q, k and v must be 16-byte aligned");
  const int sms = rot::sm_count();
  rot::Params p{};
  p.qkv = (const uint16_t*)qkv;
  p.wq = wq;
  p.wk = wk;
  p.freqs = freqs;
  p.positions = positions;
  p.q = (uint16_t*)q;
  p.k = (uint16_t*)k;
  p.v = (uint16_t*)v;
  p.ld = ld_qkv;
  p.M = M;
  p.H = H;
  p.Hk = Hk;
  p.rotary_dim = rotary_dim;
  p.amplitude = amplitude;
  p.eps = eps;
  p.slices = rot::slices_for(M, cdiv(H + 2 * Hk, 256 / D), sms);
  return rot::dispatch_fwd<false>(p, D, interleaved != 0, dtype, sms, (cudaStream_t)stream);
}

extern "C" size_t mfb_qk_rotary_workspace_size(int D) { return sizeof(float) * 2 * (size_t)D * rot::BWD_GRID_MAX; }

extern "C" int mfb_qk_rotary_bwd(const void* qkv, int ld_qkv, const float* wq, const float* wk,
                                 const int32_t* positions, const float* freqs, const void* dq, const void* dk,
                                 const void* dv, void* dqkv, float* dwq, float* dwk, int accumulate, int M, int H,
                                 int Hk, int D, int rotary_dim, int interleaved, int dtype, float amplitude, float eps,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  int st = rot::check_common(qkv, wq, wk, freqs, ld_qkv, M, H, Hk, D, rotary_dim, dtype);
  if (st) return st;
  MFB_CHECK_ARG(positions && dq && dk && dv && dqkv, "NULL rotary argument");
  MFB_CHECK_ARG((dwq == nullptr) == (dwk == nullptr), "dwq and dwk must both be given or both be NULL");
  MFB_CHECK_ARG(!dwq || wq, "gain gradients need the gains");
  MFB_CHECK_ARG(rot::aligned16({qkv, dq, dk, dv, dqkv}), "qkv, dq, dk, dv and dqkv must be 16-byte aligned");
  if (dwq && (!workspace || workspace_bytes < mfb_qk_rotary_workspace_size(D)))
    return set_error(MFB_ERR_WORKSPACE, "rotary bwd workspace needs %zu bytes", mfb_qk_rotary_workspace_size(D));
  const int sms = rot::sm_count();
  rot::Params p{};
  p.qkv = (const uint16_t*)qkv;
  p.wq = wq;
  p.wk = wk;
  p.freqs = freqs;
  p.positions = positions;
  p.dq = (const uint16_t*)dq;
  p.dk = (const uint16_t*)dk;
  p.dv = (const uint16_t*)dv;
  p.dqkv = (uint16_t*)dqkv;
  p.partial = dwq ? (float*)workspace : nullptr;
  p.ld = ld_qkv;
  p.M = M;
  p.H = H;
  p.Hk = Hk;
  p.rotary_dim = rotary_dim;
  p.amplitude = amplitude;
  p.eps = eps;
  p.slices = rot::slices_for(M, cdiv(H + 2 * Hk, 256 / D), sms);
  const long long units = (long long)M * p.slices;
  const int grid = (int)std::min<long long>((units + rot::WARPS - 1) / rot::WARPS,
                                            std::min<long long>(4LL * sms, rot::BWD_GRID_MAX));
  cudaStream_t s = (cudaStream_t)stream;
  const bool il = interleaved != 0;
  if (dtype == MFB_DTYPE_BF16) {
    if (D == 64) rot::launch_bwd<__nv_bfloat16, 64>(p, il, grid, s);
    else rot::launch_bwd<__nv_bfloat16, 128>(p, il, grid, s);
  } else {
    if (D == 64) rot::launch_bwd<__half, 64>(p, il, grid, s);
    else rot::launch_bwd<__half, 128>(p, il, grid, s);
  }
  MFB_LAUNCH_CHECK("rotary bwd");
  if (dwq) {
    rot::gain_sum_kernel<<<2 * D / 32, 1024, 0, s>>>(p.partial, grid, D, dwq, dwk, accumulate);
    MFB_LAUNCH_CHECK("rotary gain gradients");
  }
  return MFB_OK;
}

extern "C" int mfb_paged_append(const void* qkv, int ld_qkv, const float* wq, const float* wk, const float* freqs,
                                const int32_t* cu_q, const int32_t* seq_lens, const int32_t* page_table, void* q,
                                void* k_pages, void* v_pages, int N, int B, int max_pages, int num_pages,
                                int page_size, int H, int Hk, int D, int rotary_dim, int interleaved, int head_major,
                                int dtype, float amplitude, float eps, void* stream) {
  int st = rot::check_common(qkv, wq, wk, freqs, ld_qkv, N, H, Hk, D, rotary_dim, dtype);
  if (st) return st;
  MFB_CHECK_ARG(cu_q && seq_lens && page_table && q && k_pages && v_pages, "NULL paged append argument");
  MFB_CHECK_ARG(B > 0 && max_pages > 0 && num_pages > 0, "paged append needs sequences and pages (B=%d, %d, %d)", B,
                max_pages, num_pages);
  MFB_CHECK_ARG(page_size >= 8 && (page_size & (page_size - 1)) == 0,
                "page_size %d must be a power of two of at least 8", page_size);
  MFB_CHECK_ARG((long long)page_size * Hk * D <= 1 << 30, "page of %d tokens too large", page_size);
  MFB_CHECK_ARG(rot::aligned16({qkv, q, k_pages, v_pages}), "qkv, q and the pages must be 16-byte aligned");
  const int sms = rot::sm_count();
  rot::Params p{};
  p.qkv = (const uint16_t*)qkv;
  p.wq = wq;
  p.wk = wk;
  p.freqs = freqs;
  p.cu_q = cu_q;
  p.seq_lens = seq_lens;
  p.page_table = page_table;
  p.q = (uint16_t*)q;
  p.k = (uint16_t*)k_pages;
  p.v = (uint16_t*)v_pages;
  p.B = B;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.page_stride = (long long)page_size * Hk * D;
  p.token_stride = head_major ? D : Hk * D;
  p.head_stride = head_major ? page_size * D : D;
  p.ld = ld_qkv;
  p.M = N;
  p.H = H;
  p.Hk = Hk;
  p.rotary_dim = rotary_dim;
  p.amplitude = amplitude;
  p.eps = eps;
  p.slices = rot::slices_for(N, cdiv(H + 2 * Hk, 256 / D), sms);
  return rot::dispatch_fwd<true>(p, D, interleaved != 0, dtype, sms, (cudaStream_t)stream);
}
