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
// warp computes each of the token's rotary_dim/2 angles once and passes them
// through shared memory. With cw = cos * w and sw = -+sin * w_partner per lane,
//   y = r (x cw + x_partner sw),
// and the partners are exchanged as the raw 16-bit words: rotary_dim/16 lanes
// away in the half layout, in the same lane in the interleaved one. The pass is
// bandwidth-bound; registers are held down so that enough warps have loads in
// flight (q, k and v heads run in loops of their own, one set of gains live).
#include <algorithm>

#include "types16.cuh"

namespace mfb {
namespace rot {

constexpr int WARPS = 8;
constexpr int MAX_D = 128;
constexpr int BWD_GRID_MAX = 3 * 160;  // bounds the gain-gradient partials
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

// The angles of a position into the warp's table: (cos, sin) times amplitude.
__device__ __forceinline__ void angles(const Params& p, int pos, float2* table, int lane) {
  __syncwarp();
  for (int i = lane; i < p.rotary_dim >> 1; i += 32) {
    const double t = (double)pos * (double)p.freqs[i] * kInvTwoPi;
    float sn, cs;
    sincospif(2.f * (float)(t - rint(t)), &sn, &cs);
    table[i] = make_float2(cs * p.amplitude, sn * p.amplitude);
  }
  __syncwarp();
}

// This lane's coefficients: value e becomes x cw + partner sw. Half layout:
// values sub*8 + e use pair (sub*8 + e) mod (rotary_dim / 2); interleaved:
// values 2j and 2j + 1 use pair sub*4 + j. INV rotates back (R^T); w (and the
// partner's wp) multiply the inputs.
template <bool IL, bool INV>
__device__ __forceinline__ void coefficients(const Params& p, const float2* table, int sub, bool turned, bool low,
                                             const float* gains, float* cw, float* sw) {
  const int half = p.rotary_dim >> 1;
  float w[8], wp[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = wp[e] = 1.f;
  if (gains) {
    const int mine = sub * 8, other = !turned || IL ? mine : (low ? mine + half : mine - half);
    const float4 a = reinterpret_cast<const float4*>(gains + mine)[0], b = reinterpret_cast<const float4*>(gains + mine)[1];
    const float4 c = reinterpret_cast<const float4*>(gains + other)[0], d = reinterpret_cast<const float4*>(gains + other)[1];
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    wp[0] = c.x, wp[1] = c.y, wp[2] = c.z, wp[3] = c.w, wp[4] = d.x, wp[5] = d.y, wp[6] = d.z, wp[7] = d.w;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float2 f = make_float2(1.f, 0.f);
    if (turned) f = table[IL ? sub * 4 + e / 2 : (low ? sub * 8 + e : sub * 8 + e - half)];
    const bool minus = (IL ? (e & 1) == 0 : low) != INV;  // y_first = x_first c - x_second s
    cw[e] = f.x * w[e];
    sw[e] = (minus ? -f.y : f.y) * (IL ? wp[e ^ 1] : wp[e]);
  }
}

// The partners' raw words (zeros where nothing is rotated).
template <bool IL>
__device__ __forceinline__ uint4 partners(const uint4& v, int from, bool turned) {
  if (IL) {
    return make_uint4(__byte_perm(v.x, 0, 0x1032), __byte_perm(v.y, 0, 0x1032), __byte_perm(v.z, 0, 0x1032),
                      __byte_perm(v.w, 0, 0x1032));
  }
  uint4 o;
  o.x = __shfl_sync(0xffffffffu, v.x, from);
  o.y = __shfl_sync(0xffffffffu, v.y, from);
  o.z = __shfl_sync(0xffffffffu, v.z, from);
  o.w = __shfl_sync(0xffffffffu, v.w, from);
  return turned ? o : make_uint4(0, 0, 0, 0);
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

__device__ __forceinline__ uint4 ld16(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void st16(uint16_t* p, const uint4& v) { *reinterpret_cast<uint4*>(p) = v; }

// Runs body(i, h, live) over this warp's heads [0, n) in steps of `step`, four
// steps' loads ahead of their use: load(h) -> uint4. All lanes take part in
// every step (shuffles); heads past the end are not live.
template <int AHEAD, typename Load, typename Body>
__device__ __forceinline__ void over_heads(int first, int grp, int step, int n, Load load, Body body) {
  for (int h0 = first; h0 < n; h0 += AHEAD * step) {
    uint4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int h = h0 + i * step + grp;
      v[i] = h < n ? load(h) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (h0 + i * step < n) body(h0 + i * step + grp, h0 + i * step + grp < n, v[i]);
  }
}

template <typename T, int D, bool IL, bool PAGED>
__global__ void __launch_bounds__(32 * WARPS, 4) rotary_fwd_kernel(Params p) {
  constexpr int L = D / 8, HPW = 32 / L;  // lanes per head, heads per warp
  __shared__ float2 tables[WARPS][MAX_D / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, grp = lane / L;
  const int half8 = p.rotary_dim >> 4;  // lanes of half a rotated part
  const bool turned = sub * 8 < p.rotary_dim, low = sub < half8;
  const int from = turned ? (low ? lane + half8 : lane - half8) : lane;
  const bool norm = p.wq != nullptr;
  const long long units = (long long)p.M * p.slices, step = (long long)gridDim.x * WARPS;
  for (long long u = (long long)blockIdx.x * WARPS + warp; u < units; u += step) {
    const int row = (int)(u / p.slices), first = (int)(u % p.slices) * HPW, hstep = p.slices * HPW;
    const uint16_t* src = p.qkv + (long long)row * p.ld + sub * 8;
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
      slot = (long long)row * p.Hk * D;
    }
    // Values: copied. Their loads are under way while the angles are computed.
    if (p.v && slot >= 0)
      over_heads<4>(first, grp, hstep, p.Hk, [&](int h) { return ld16(src + (long long)(p.H + p.Hk + h) * D); },
                    [&](int h, bool live, const uint4& v) {
                      if (live) st16(p.v + slot + (long long)h * p.head_stride + sub * 8, v);
                    });
    angles(p, pos, tables[warp], lane);
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      float cw[8], sw[8];
      coefficients<IL, false>(p, tables[warp], sub, turned, low, which ? p.wk : p.wq, cw, sw);
      const uint16_t* in = src + (which ? (long long)p.H * D : 0);
      uint16_t* out = which ? p.k + slot : p.q + (long long)row * p.H * D;
      const long long hs = which ? p.head_stride : D;
      const bool stored = !which || slot >= 0;
      over_heads<4>(first, grp, hstep, which ? p.Hk : p.H, [&](int h) { return ld16(in + (long long)h * D); },
                    [&](int h, bool live, const uint4& v) {
                      float x[8], y[8], r = 1.f;
                      unpack16x8<T>(v, x);
                      unpack16x8<T>(partners<IL>(v, from, turned), y);
                      if (norm) {
                        float ss = 0.f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
                        r = rsqrtf(head_sum<L>(ss) * (1.f / D) + p.eps);
                      }
#pragma unroll
                      for (int e = 0; e < 8; ++e) x[e] = fmaf(y[e], sw[e], x[e] * cw[e]) * r;
                      if (live && stored) st16(out + h * hs + sub * 8, pack16x8<T>(x));
                    });
    }
  }
}

template <typename T, int D, bool IL>
__global__ void __launch_bounds__(32 * WARPS, 3) rotary_bwd_kernel(Params p) {
  constexpr int L = D / 8, HPW = 32 / L;
  __shared__ float2 tables[WARPS][MAX_D / 2];
  __shared__ float sums[WARPS][2 * D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, grp = lane / L;
  const int half8 = p.rotary_dim >> 4;
  const bool turned = sub * 8 < p.rotary_dim, low = sub < half8;
  const int from = turned ? (low ? lane + half8 : lane - half8) : lane;
  const bool norm = p.wq != nullptr;
  float acc[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[0][e] = acc[1][e] = 0.f;
  const long long units = (long long)p.M * p.slices, step = (long long)gridDim.x * WARPS;
  for (long long u = (long long)blockIdx.x * WARPS + warp; u < units; u += step) {
    const int row = (int)(u / p.slices), first = (int)(u % p.slices) * HPW, hstep = p.slices * HPW;
    const long long base = (long long)row * p.ld + sub * 8;
    over_heads<4>(first, grp, hstep, p.Hk, [&](int h) { return ld16(p.dv + ((long long)row * p.Hk + h) * D + sub * 8); },
                  [&](int h, bool live, const uint4& v) {
                    if (live) st16(p.dqkv + base + (long long)(p.H + p.Hk + h) * D, v);
                  });
    angles(p, p.positions[row], tables[warp], lane);
    float c[8], s[8];
    coefficients<IL, true>(p, tables[warp], sub, turned, low, nullptr, c, s);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int heads = which ? p.Hk : p.H;
      const long long in = base + (which ? (long long)p.H * D : 0);
      const uint16_t* up = (which ? p.dk : p.dq) + (long long)row * heads * D + sub * 8;
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = norm ? (which ? p.wk : p.wq)[sub * 8 + e] : 1.f;
      for (int h0 = first; h0 < heads; h0 += 2 * hstep) {
        uint4 bg[2], bx[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int h = h0 + i * hstep + grp;
          bg[i] = bx[i] = make_uint4(0, 0, 0, 0);
          if (h < heads) {
            bg[i] = ld16(up + (long long)h * D);
            if (norm) bx[i] = ld16(p.qkv + in + (long long)h * D);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (h0 + i * hstep >= heads) break;
          const int h = h0 + i * hstep + grp;
          float g[8], y[8];
          unpack16x8<T>(bg[i], g);
          unpack16x8<T>(partners<IL>(bg[i], from, turned), y);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] = fmaf(y[e], s[e], g[e] * c[e]);
          if (norm) {
            float x[8], ss = 0.f, dot = 0.f;
            unpack16x8<T>(bx[i], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
            const float r = rsqrtf(head_sum<L>(ss) * (1.f / D) + p.eps);
            // Heads past the end are zeros and add nothing.
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              x[e] *= r;
              acc[which][e] = fmaf(g[e], x[e], acc[which][e]);
              g[e] *= w[e];
              dot = fmaf(g[e], x[e], dot);
            }
            const float mean = head_sum<L>(dot) * (1.f / D);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = r * fmaf(-x[e], mean, g[e]);
          }
          if (h < heads) st16(p.dqkv + in + (long long)h * D, pack16x8<T>(g));
        }
      }
    }
  }
  if (p.partial == nullptr) return;
  allow_dependents();
  // Gain gradients: heads of the warp, warps of the block, then one row of
  // partials per block for the column sum below -- all in a fixed order.
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float t = acc[which][e];
#pragma unroll
      for (int o = L; o < 32; o <<= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
      if (grp == 0) sums[warp][which * D + sub * 8 + e] = t;
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

// dw[col] (+)= sum over `rows` partial rows; 8 columns per block (a 32-byte
// sector of each row), 128 row lanes, combined in a fixed tree. Columns [0, D)
// are wq's, [D, 2D) wk's.
__global__ void __launch_bounds__(1024) gain_sum_kernel(const float* __restrict__ partial, int rows, int D,
                                                        float* __restrict__ dwq, float* __restrict__ dwk,
                                                        int accumulate) {
  __shared__ float part[8][128];
  const int x = threadIdx.x & 7, y = threadIdx.x >> 3, col = blockIdx.x * 8 + x;
  wait_prerequisites();
  float t = 0.f;
#pragma unroll 5
  for (int r = y; r < rows; r += 128) t += partial[(long long)r * 2 * D + col];
  part[x][y] = t;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp < 8) {  // warp w sums column blockIdx.x * 8 + w
    t = warp_sum((part[warp][lane] + part[warp][lane + 32]) + (part[warp][lane + 64] + part[warp][lane + 96]));
    if (lane == 0) {
      const int c = blockIdx.x * 8 + warp;
      float* dst = c < D ? dwq + c : dwk + (c - D);
      *dst = accumulate ? *dst + t : t;
    }
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
  MFB_CHECK_ARG((((uintptr_t)wq | (uintptr_t)wk) & 15) == 0, "gains must be 16-byte aligned");
  return MFB_OK;
}

template <typename T, int D, bool PAGED>
int launch_fwd(const Params& p, bool interleaved, int sms, cudaStream_t s) {
  const long long units = (long long)p.M * p.slices;
  const int grid = (int)std::min<long long>((units + WARPS - 1) / WARPS, 4LL * sms);
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
  p.head_stride = D;
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
                                            std::min<long long>(3LL * sms, rot::BWD_GRID_MAX));
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
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * D / 8);
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MFB_CUDA_TRY(cudaLaunchKernelEx(&cfg, rot::gain_sum_kernel, (const float*)p.partial, grid, D, dwq, dwk, accumulate));
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
