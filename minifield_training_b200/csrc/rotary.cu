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
// Layout: a thread keeps its place in the heads -- one head, two chunks of four
// values that are each other's partners (4s.. and rotary_dim/2 + 4s.. in the
// half layout; the 8 values from 8s in the interleaved one and in the part
// that is not rotated) -- and walks a run of tokens, so that gains, addresses
// and the kind of head are settled once and the rotation needs no exchange
// between lanes. Every 32-byte sector is still read and written whole. A block
// takes a few tokens at a time: their heads' loads are under way while the
// block computes the tokens' rotary_dim/2 angles each into shared memory; their
// positions and cache rows, a chain of dependent loads, are looked up for 32
// tokens at a time. The floor is the bytes. With a warp per token that loops
// over the heads, the same arithmetic took three times the instructions and 84 to
// 111 us where this takes 70 us (16384 tokens of 32 heads, forward and backward).
// In those the issue slots are now busy 65 and 63 % of the cycles and the ALUs 44,
// and of the 11 to 12 cycles between a warp's instructions 3 to 4 pass at a pass's
// barrier, where the heads' threads wait for the angles: more than anywhere else.
// Head counts that do not fill a block (32 heads of 64, 16 of 128, or a multiple)
// leave threads that load the last head and store nothing.
#include <algorithm>

#include "types16.cuh"

namespace mfb {
namespace rot {

constexpr int THREADS = 256;
constexpr int MAX_D = 128;
// Tokens of a block's pass, and blocks per SM. Measured together on 16384 tokens
// forward and backward: 8 tokens forward and 4 backward at 3 blocks 73.8, 4 and
// 2 at 4 blocks 69.7, at 3 77.6, at 5 81.6, 2 and 1 at 6 88.0 us.
constexpr int FWD_TOKENS = 4, BWD_TOKENS = 2, BLOCKS_PER_SM = 4;
// Tokens whose positions (and cache rows) a block looks up at once.
constexpr int LOOKUP = 32;
constexpr int MAX_SMS = 160;
constexpr int BWD_GRID_MAX = BLOCKS_PER_SM * MAX_SMS;  // blocks of a backward pass: rows of gain-gradient partials
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
  int ld, M, H, Hk, rotary_dim, heads;  // heads: q, k and (when written) v
  float amplitude, eps;
};

// cos and sin (times amplitude) of a block's tokens, position of token t in
// pos[t]; a warp per token. The turn is reduced in FP64, so the hardware's
// sine and cosine see at most half a turn, where they are off by 2^-20.5 at most.
template <int TOKENS>
struct Angles {
  float c[TOKENS][MAX_D / 2], s[TOKENS][MAX_D / 2];
  __device__ __forceinline__ void fill(const Params& p, const int* pos, int tokens) {
    const int half = p.rotary_dim >> 1;
    for (int t = threadIdx.x >> 5; t < tokens; t += THREADS / 32) {
      const double at = (double)pos[t] * kInvTwoPi;
      for (int k = threadIdx.x & 31; k < half; k += 32) {
        const double turns = at * (double)p.freqs[k];
        const float x = 6.283185307f * (float)(turns - rint(turns));
        c[t][k] = __cosf(x) * p.amplitude;
        s[t][k] = __sinf(x) * p.amplitude;
      }
    }
  }
};

// Runs body(t) for t < tokens: unrolled without tests where the pass is full.
template <int TOKENS, typename Body>
__device__ __forceinline__ void over_tokens(int tokens, Body body) {
  if (tokens == TOKENS) {
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) body(t);
  } else {
#pragma unroll
    for (int t = 0; t < TOKENS; ++t)
      if (t < tokens) body(t);
  }
}

// A thread's place: head `head` of the row (kind 0 q, 1 k, 2 v; head `in_kind`
// of its kind), values oa.. and ob... Threads past the last head take the last
// head's place (shuffles need them) and store nothing.
template <int D, bool IL>
struct Place {
  static constexpr int L = D / 8;  // lanes per head
  int head, kind, in_kind, sub, oa, ob;
  bool live, turned, copies;  // copies: all of this warp's heads are v's
  __device__ __forceinline__ explicit Place(const Params& p) {
    const int h = blockIdx.y * (THREADS / L) + threadIdx.x / L;
    sub = threadIdx.x % L;
    live = h < p.heads;
    head = min(h, p.heads - 1);
    kind = head < p.H ? 0 : head < p.H + p.Hk ? 1 : 2;
    in_kind = head - (kind == 0 ? 0 : kind == 1 ? p.H : p.H + p.Hk);
    turned = sub * 8 < p.rotary_dim;
    copies = __all_sync(0xffffffffu, kind == 2);
    oa = turned && !IL ? sub * 4 : sub * 8;
    ob = turned && !IL ? sub * 4 + (p.rotary_dim >> 1) : sub * 8 + 4;
  }
  __device__ __forceinline__ void gains(const Params& p, uint64_t* w) const {
    const float* g = kind == 0 ? p.wq : kind == 1 ? p.wk : nullptr;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 a = g ? reinterpret_cast<const float2*>(g + oa)[i] : make_float2(1.f, 1.f);
      const float2 b = g ? reinterpret_cast<const float2*>(g + ob)[i] : make_float2(1.f, 1.f);
      w[i] = pair(a.x, a.y);
      w[2 + i] = pair(b.x, b.y);
    }
  }
  // Rotates x (chunk a in x[0..1], b in x[2..3]) by one token's angles; INV back.
  template <bool INV>
  __device__ __forceinline__ void rotate(const float* cs, const float* sn, uint64_t* x) const {
    if (!turned) return;
    const float4 c = *reinterpret_cast<const float4*>(cs + sub * 4), s = *reinterpret_cast<const float4*>(sn + sub * 4);
    if (IL) {
      const float ca[4] = {c.x, c.y, c.z, c.w}, sa[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpair(x[i]);
        const float sg = INV ? -sa[i] : sa[i];
        x[i] = pair(f.x * ca[i] - f.y * sg, f.y * ca[i] + f.x * sg);
      }
    } else {
      const uint64_t ca[2] = {pair(c.x, c.y), pair(c.z, c.w)}, sa[2] = {pair(s.x, s.y), pair(s.z, s.w)};
      const uint64_t na[2] = {pair(-s.x, -s.y), pair(-s.z, -s.w)};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint64_t a = x[i], b = x[2 + i];
        x[i] = fma2(b, INV ? sa[i] : na[i], mul2(a, ca[i]));
        x[2 + i] = fma2(a, INV ? na[i] : sa[i], mul2(b, ca[i]));
      }
    }
  }
};

template <int L>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int D>
__device__ __forceinline__ float head_rnorm(const uint64_t* x, float eps) {
  uint64_t ss = mul2(x[0], x[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) ss = fma2(x[i], x[i], ss);
  const float2 f = unpair(ss);
  return rsqrtf(head_sum<D / 8>(f.x + f.y) * (1.f / D) + eps);
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

__device__ __forceinline__ uint2 ld8(const uint16_t* p) { return *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ void st8(uint16_t* p, const uint2& v) { *reinterpret_cast<uint2*>(p) = v; }

// A block's run of tokens.
__device__ __forceinline__ int run_begin(const Params& p, int i) { return (int)((long long)p.M * i / gridDim.x); }

template <typename T, int D, bool IL, bool PAGED>
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM) rotary_fwd_kernel(Params p) {
  __shared__ __align__(16) Angles<FWD_TOKENS> tables[2];  // by turns: a pass needs one barrier
  __shared__ int s_pos[LOOKUP];
  __shared__ long long s_place[LOOKUP];  // element offset of a token's first head in k and v; -1: not stored
  const Place<D, IL> w(p);
  uint64_t gain[4];
  w.gains(p, gain);
  const uint16_t* in = p.qkv + w.head * D;
  uint16_t* out = w.kind == 0 ? p.q + w.in_kind * D : (w.kind == 1 ? p.k : p.v) + (long long)w.in_kind * p.head_stride;
  const int begin = run_begin(p, blockIdx.x), end = run_begin(p, blockIdx.x + 1);
  for (int row0 = begin; row0 < end; row0 += FWD_TOKENS) {
    const int tokens = min(FWD_TOKENS, end - row0);
    uint2 va[FWD_TOKENS], vb[FWD_TOKENS];
    const uint16_t* src = in + (long long)row0 * p.ld;
    over_tokens<FWD_TOKENS>(tokens, [&](int t) {
      va[t] = ld8(src + w.oa);
      vb[t] = ld8(src + w.ob);
      src += p.ld;
    });
    const int at = (row0 - begin) % LOOKUP;
    if (at == 0) {
      __syncthreads();  // the last pass is done with the places
      const int row = row0 + threadIdx.x;
      if (threadIdx.x < LOOKUP && row < end) {
        int pos = 0;
        long long place = -1;
        if (PAGED) {
          if (row < p.cu_q[0] || row >= p.cu_q[p.B]) {
            place = -2;  // padding: nothing is stored
          } else {
            const int b = sequence_of(p.cu_q, p.B, row);
            pos = p.seq_lens[b] - (p.cu_q[b + 1] - row);
            const int pg = pos >> p.page_shift;
            if (pos >= 0 && pg < p.max_pages) {
              const int id = p.page_table[(long long)b * p.max_pages + pg];
              if ((unsigned)id < (unsigned)p.num_pages)
                place = (long long)id * p.page_stride + (long long)(pos - (pg << p.page_shift)) * p.token_stride;
            }
          }
        } else {
          pos = p.positions[row];
          place = (long long)row * p.Hk * D;
        }
        s_pos[threadIdx.x] = pos;
        s_place[threadIdx.x] = place;
      }
      __syncthreads();
    }
    Angles<FWD_TOKENS>& angles = tables[(row0 - begin) / FWD_TOKENS & 1];
    angles.fill(p, s_pos + at, tokens);
    __syncthreads();
    long long q_to = (long long)row0 * p.H * D;
    over_tokens<FWD_TOKENS>(tokens, [&](int t) {
      uint2 a = va[t], b = vb[t];
      if (!w.copies) {
        uint64_t x[4];
        unpack16x4<T>(a, x);
        unpack16x4<T>(b, x + 2);
        if (p.wq) {
          const float r = head_rnorm<D>(x, p.eps);
          const uint64_t r2 = pair(r, r);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = mul2(x[i], mul2(r2, gain[i]));
        }
        w.template rotate<false>(angles.c[t], angles.s[t], x);
        if (w.kind < 2) {
          a = pack16x4<T>(x);
          b = pack16x4<T>(x + 2);
        }
      }
      long long to = s_place[at + t];
      const bool stored = w.live && to >= (w.kind ? 0 : -1);
      if (w.kind == 0) to = q_to;
      q_to += p.H * D;
      if (stored) {
        st8(out + to + w.oa, a);
        st8(out + to + w.ob, b);
      }
    });
  }
}

template <typename T, int D, bool IL>
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM) rotary_bwd_kernel(Params p) {
  using W = Place<D, IL>;
  __shared__ __align__(16) Angles<BWD_TOKENS> tables[2];
  __shared__ int s_pos[LOOKUP];
  __shared__ float sums[THREADS / W::L][D];
  const W w(p);
  uint64_t gain[4], acc[4];
  w.gains(p, gain);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = pair(0.f, 0.f);
  const int kind_heads = w.kind ? p.Hk : p.H;
  const uint16_t* up = (w.kind == 0 ? p.dq : w.kind == 1 ? p.dk : p.dv) + w.in_kind * D;
  const long long up_row = (long long)kind_heads * D;
  const int begin = run_begin(p, blockIdx.x), end = run_begin(p, blockIdx.x + 1);
  for (int row0 = begin; row0 < end; row0 += BWD_TOKENS) {
    const int tokens = min(BWD_TOKENS, end - row0);
    uint2 ga[BWD_TOKENS], gb[BWD_TOKENS], xa[BWD_TOKENS], xb[BWD_TOKENS];
    const uint16_t* src = up + row0 * up_row;
    const uint16_t* row = p.qkv + (long long)row0 * p.ld + w.head * D;
    over_tokens<BWD_TOKENS>(tokens, [&](int t) {
      ga[t] = ld8(src + w.oa);
      gb[t] = ld8(src + w.ob);
      src += up_row;
      if (p.wq && !w.copies) {
        xa[t] = ld8(row + w.oa);
        xb[t] = ld8(row + w.ob);
      }
      row += p.ld;
    });
    const int at = (row0 - begin) % LOOKUP;
    if (at == 0) {
      __syncthreads();
      if (threadIdx.x < LOOKUP && row0 + threadIdx.x < end) s_pos[threadIdx.x] = p.positions[row0 + threadIdx.x];
      __syncthreads();
    }
    Angles<BWD_TOKENS>& angles = tables[(row0 - begin) / BWD_TOKENS & 1];
    angles.fill(p, s_pos + at, tokens);
    __syncthreads();
    uint16_t* out = p.dqkv + (long long)row0 * p.ld + w.head * D;
    over_tokens<BWD_TOKENS>(tokens, [&](int t) {
      uint2 a = ga[t], b = gb[t];
      if (!w.copies) {
        uint64_t g[4];
        unpack16x4<T>(a, g);
        unpack16x4<T>(b, g + 2);
        w.template rotate<true>(angles.c[t], angles.s[t], g);
        if (p.wq) {
          uint64_t x[4], dot = pair(0.f, 0.f);
          unpack16x4<T>(xa[t], x);
          unpack16x4<T>(xb[t], x + 2);
          const float r = head_rnorm<D>(x, p.eps);
          const uint64_t r2 = pair(r, r);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = mul2(x[i], r2);
            acc[i] = fma2(g[i], x[i], acc[i]);
            g[i] = mul2(g[i], gain[i]);
            dot = fma2(g[i], x[i], dot);
          }
          const float2 d2 = unpair(dot);
          const float mean = head_sum<W::L>(d2.x + d2.y) * (-1.f / D);
          const uint64_t m2 = pair(mean, mean);
#pragma unroll
          for (int i = 0; i < 4; ++i) g[i] = mul2(r2, fma2(x[i], m2, g[i]));
        }
        if (w.kind < 2) {
          a = pack16x4<T>(g);
          b = pack16x4<T>(g + 2);
        }
      }
      if (w.live) {
        st8(out + w.oa, a);
        st8(out + w.ob, b);
      }
      out += p.ld;
    });
  }
  if (p.partial == nullptr) return;
  allow_dependents();
  // Gain gradients: the block's q heads and its k heads, each in head order,
  // then one row of partials per block for the column sum below.
  float* mine = sums[threadIdx.x / W::L];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpair(acc[i]);
    float* at = mine + (i < 2 ? w.oa + 2 * i : w.ob + 2 * (i - 2));
    at[0] = w.live ? f.x : 0.f;
    at[1] = w.live ? f.y : 0.f;
  }
  __syncthreads();
  const int h0 = blockIdx.y * (THREADS / W::L);
  for (int i = threadIdx.x; i < 2 * D; i += THREADS) {
    const int lo = i < D ? 0 : p.H, hi = i < D ? p.H : p.H + p.Hk;
    float t = 0.f;
    for (int k = max(lo - h0, 0); k < min(hi - h0, THREADS / W::L); ++k) t += sums[k][i % D];
    p.partial[(long long)(blockIdx.y * gridDim.x + blockIdx.x) * 2 * D + i] = t;
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
  return std::min(sms, MAX_SMS);
}

// Blocks: `chunks` in y cover a row's heads, x cuts the tokens into runs, as
// many as are resident, one token each at least.
dim3 grid_for(const Params& p, int D, int sms) {
  const int chunks = cdiv(p.heads, THREADS / (D / 8));
  return dim3((unsigned)std::max(1, std::min(p.M, BLOCKS_PER_SM * sms / chunks)), (unsigned)chunks);
}

int check_common(const void* qkv, const float* wq, const float* wk, const float* freqs, int ld, int M, int H, int Hk,
                 int D, int rotary_dim, int dtype) {
  MFB_CHECK_ARG(M > 0 && H > 0 && Hk > 0, "rotary needs tokens and heads (M=%d H=%d Hk=%d)", M, H, Hk);
  MFB_CHECK_ARG(D == 64 || D == 128, "rotary head_dim %d unsupported (64 or 128)", D);
  MFB_CHECK_ARG(H + 2LL * Hk <= 1024, "rotary supports up to 1024 heads in a row (H=%d Hk=%d)", H, Hk);
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
  const dim3 grid = grid_for(p, D, sms);
  if (interleaved) rotary_fwd_kernel<T, D, true, PAGED><<<grid, THREADS, 0, s>>>(p);
  else rotary_fwd_kernel<T, D, false, PAGED><<<grid, THREADS, 0, s>>>(p);
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
void launch_bwd(const Params& p, bool interleaved, dim3 grid, cudaStream_t s) {
  if (interleaved) rotary_bwd_kernel<T, D, true><<<grid, THREADS, 0, s>>>(p);
  else rotary_bwd_kernel<T, D, false><<<grid, THREADS, 0, s>>>(p);
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
  p.heads = H + 2 * Hk;
  p.rotary_dim = rotary_dim;
  p.amplitude = amplitude;
  p.eps = eps;
  if (!v) p.heads = H + Hk;
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
  p.heads = H + 2 * Hk;
  p.rotary_dim = rotary_dim;
  p.amplitude = amplitude;
  p.eps = eps;
  const dim3 grid = rot::grid_for(p, D, sms);
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
    MFB_CUDA_TRY(cudaLaunchKernelEx(&cfg, rot::gain_sum_kernel, (const float*)p.partial, (int)(grid.x * grid.y), D, dwq, dwk, accumulate));
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
  p.heads = H + 2 * Hk;
  p.rotary_dim = rotary_dim;
  p.amplitude = amplitude;
  p.eps = eps;
  return rot::dispatch_fwd<true>(p, D, interleaved != 0, dtype, sms, (cudaStream_t)stream);
}
