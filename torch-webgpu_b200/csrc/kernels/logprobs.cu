// Log probabilities of given tokens under softmax(scale * logits), with the entropy of every row and
// its largest alternatives, and the gradient.
//
//   z = scale x,  lse = log sum_j e^{z_j},  logp_m = z[token_m] - lse,  H = lse - sum_j p_j z_j
//   dz_j = sum_m dlogp_m ([j = token_m] - p_j) - dH p_j (z_j - lse + H) + dlse p_j,   dx = scale dz
//
// One pass over the logits: every thread keeps the running maximum m of what it has seen, the sum
// s of e = 2^u with u = (x - m) scale log2(e), and t = sum e u; at the end H = ln s - ln2 t / s.
// The difference is taken before the scaling, so that a row of the type's lowest value is still a
// uniform distribution, and u is held at -150 or above, where 2^u is 0 and the product with u is
// not 0 * inf.  NaN passes that clamp and makes the row's numbers NaN, as +inf does.
//
// The forward pass reads 2 or 4 bytes an element and spends one exponential on it: at the rate of
// the copy bandwidth a 16-bit row takes three quarters of the special-function units' rate, so
// everything else has to stay at a few instructions an element.  A row belongs to a cluster of 1
// to 8 CTAs which combine their numbers through distributed shared memory: few long rows still
// fill the GPU, nothing passes through a workspace and there is one launch.
//
// 4096 rows of 131072 bfloat16 logits: forward 185 us (5.8 TB/s), 221 us under a load of seconds (power
// limit), gradient 319 us (6.7 TB/s, the copy bandwidth).  2047 rows of 50257 float32 logits with five
// alternatives 70 us, 79 us under that load.  Measured and dropped: loads held in registers (207 us, and
// 247 with 512 threads a row), CTAs that stay for several rows (226 us), stages of four vectors (181 us,
// but 73 us for the float32 rows).
#include <cooperative_groups.h>

#include <cfloat>

#include "twg_float.cuh"

namespace twg {

namespace cg = cooperative_groups;

constexpr int kLpMaxThreads = 256;
constexpr int kLpMaxWarps = kLpMaxThreads / 32;
constexpr int kLpUnroll = 2;       // 16-byte vectors of a thread in one stage of the forward kernel's loads
constexpr int kLpStages = 4;       // stages on their way (a power of two)
constexpr int kLpCtas = 5;         // CTAs of that size an SM holds
constexpr int kLpGradUnroll = 8;   // vectors a thread of the gradient has on their way
constexpr int kLpGradRounds = 2;   // rounds of its loads in a CTA
constexpr int kLpMaxCluster = 8;
constexpr int kLpMaxTop = 32;
constexpr int kLpCandidates = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogprobArgs {
  const void* x;
  const void* tokens;
  float *logp, *entropy, *lse, *top_logp;
  i64* top_ids;
  i64 row_stride, ts0, ts1;
  int vocab, m, top;
  float scale;
  bool tok64;
};

__device__ __forceinline__ float ex2(float u) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(u));
  return r;
}
// The larger of u and -150; NaN stays NaN.
__device__ __forceinline__ float hold(float u) {
  float r;
  asm("max.NaN.f32 %0, %1, 0fC3160000;" : "=f"(r) : "f"(u));
  return r;
}

// Running softmax numbers of a set of elements, relative to its maximum.
struct Soft {
  float m, s, t;
  __device__ __forceinline__ void rebase(float to, float c) {
    const float d = hold((m - to) * c), r = ex2(d);
    t = r * fmaf(d, s, t);
    s *= r;
    m = to;
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N], float largest, float c) {
    rebase(fmaxf(m, largest), c);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float u = hold((f[j] - m) * c), e = ex2(u);
      s += e;
      t = fmaf(e, u, t);
    }
  }
  __device__ __forceinline__ void warp_sum(float c) {
    float M = m;
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    rebase(M, c);
    for (int o = 16; o; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      t += __shfl_xor_sync(0xffffffffu, t, o);
    }
  }
};

// The same while a thread collects them, in two halves that one instruction works on.
struct SoftPair {
  float m;
  Two s, t;
  __device__ __forceinline__ SoftPair() : m(-FLT_MAX), s(0.0f, 0.0f), t(0.0f, 0.0f) {}
  template <int N>
  __device__ __forceinline__ void add_all(const float (&f)[N], float largest, float c) {
    const float to = fmaxf(m, largest), d = hold((m - to) * c), r = ex2(d);
    const Two rr(r, r), cc(c, c), base(-to, -to);
    t = mul(rr, fma(Two(d, d), s, t));
    s = mul(rr, s);
    m = to;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float u0, u1;
      mul(add(Two(f[j], f[j + 1]), base), cc).get(u0, u1);
      u0 = hold(u0);
      u1 = hold(u1);
      const Two e(ex2(u0), ex2(u1));
      s = add(s, e);
      t = fma(e, Two(u0, u1), t);
    }
  }
  __device__ __forceinline__ Soft sum() const {
    float s0, s1, t0, t1;
    s.get(s0, s1);
    t.get(t0, t1);
    return Soft{m, s0 + s1, t0 + t1};
  }
};

__device__ __forceinline__ Soft no_soft() { return Soft{-FLT_MAX, 0.0f, 0.0f}; }

// Whole number that orders floats: NaN above everything, -0 equal to 0; 0 stands for no element.
__device__ __forceinline__ u32 order_of(float x) {
  const u32 b = as_u(x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(u32 order) {
  if (order == 0xffffffffu) return as_f(0x7fffffffu);
  return as_f(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu));
}
// Larger value first, then the lower index.
__device__ __forceinline__ u64 rank_key(float x, u32 index) { return ((u64)order_of(x) << 32) | (0xffffffffu - index); }

struct LpShared {
  Soft warp[kLpMaxWarps];
  Soft part[kLpMaxCluster];              // of the cluster's CTAs, in CTA 0
  u64 found[kLpCandidates];
  u64 best[kLpMaxTop];
  u64 merge[kLpMaxCluster * kLpMaxTop];  // the CTAs' alternatives, in CTA 0
  int count;
};

// Where a row's 16-byte vectors lie: `head` elements in front of the first aligned one, nvec
// vectors, the rest behind them.
template <class T>
struct RowSplit {
  int head, nvec, tail;
  __device__ __forceinline__ RowSplit(const T* row, int n) {
    const int off = (int)((reinterpret_cast<u64>(row) & 15u) / sizeof(T));
    head = min(off ? kVecOf<T> - off : 0, n);
    nvec = (n - head) / kVecOf<T>;
    tail = n - head - nvec * kVecOf<T>;
  }
};
template <class T>
__device__ __forceinline__ uint4 minus_inf() {
  const u32 w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(w, w, w, w);
}

// Alternatives the slow way, for rows whose quick bound lets too many elements through (long runs
// of equal logits, rising logits) or that hold a NaN: every warp keeps a sorted list in its lanes.
template <class T>
__device__ __noinline__ void slow_top(const T* row, const RowSplit<T> rs, int v0, int v1, bool extra, float x_extra, int i_extra,
                                      int top, LpShared& sh) {
  constexpr int V = kVecOf<T>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 mine = 0, limit = 0;
  auto offer = [&](u64 key) {
    unsigned b = __ballot_sync(0xffffffffu, key > limit);
    while (b) {
      const u64 k = __shfl_sync(0xffffffffu, key, __ffs(b) - 1);
      b &= b - 1;
      if (k <= limit) continue;
      const int pos = __popc(__ballot_sync(0xffffffffu, mine > k));
      const u64 up = __shfl_up_sync(0xffffffffu, mine, 1);
      if (lane == pos) mine = k;
      else if (lane > pos) mine = up;
      limit = __shfl_sync(0xffffffffu, mine, top - 1);
    }
  };
  offer(extra ? rank_key(x_extra, (u32)i_extra) : 0);
  for (int v = v0 + warp * 32; v < v1; v += (int)blockDim.x) {
    float f[V];
    const bool on = v + lane < v1;
    uint4 raw = minus_inf<T>();
    if (on) raw = *reinterpret_cast<const uint4*>(row + rs.head + (i64)(v + lane) * V);
    unpack(raw, f, static_cast<const T*>(nullptr));
#pragma unroll
    for (int j = 0; j < V; ++j) offer(on ? rank_key(f[j], (u32)(rs.head + (v + lane) * V + j)) : 0);
  }
  __syncthreads();
  if (lane < top) sh.found[warp * top + lane] = mine;
  if (threadIdx.x == 0) sh.count = (int)(blockDim.x >> 5) * top;
}

// The `top` largest of the n keys in `keys` to sh.best, in order (keys are distinct except for 0).
__device__ __forceinline__ void rank_keys(const u64* keys, int n, int top, u64* best) {
  for (int i = threadIdx.x; i < n; i += (int)blockDim.x) {
    const u64 k = keys[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += keys[j] > k;
    if (k != 0 && r < top) best[r] = k;
  }
}

template <class T, bool TOP, int NT>
__global__ void __launch_bounds__(NT, kLpCtas * (kLpMaxThreads / NT)) logprobs_kernel(const __grid_constant__ LogprobArgs a) {
  constexpr int V = kVecOf<T>;
  __shared__ LpShared sh;
  extern __shared__ uint4 ring[];  // [kLpStages][kLpUnroll][threads]
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const i64 r = blockIdx.x / (unsigned)parts;
  const T* row = static_cast<const T*>(a.x) + r * a.row_stride;
  const RowSplit<T> rs(row, a.vocab);
  const int per = (rs.nvec + parts - 1) / parts;
  const int v0 = min(part * per, rs.nvec), v1 = min(v0 + per, rs.nvec);
  constexpr int nt = NT;
  const int tid = threadIdx.x;
  const float c = a.scale * kLog2e;
  if constexpr (TOP) {
    if (tid == 0) sh.count = 0;
    if (tid < kLpMaxTop) sh.best[tid] = 0;
  }

  // the elements in front of and behind the vectors belong to CTA 0
  const bool extra = part == 0 && tid < rs.head + rs.tail;
  const int i_extra = tid < rs.head ? tid : a.vocab - rs.tail + tid - rs.head;
  float fx[1] = {extra ? to_f32(row[i_extra]) : -INFINITY};

  // the given tokens' logits, asked for before anything else is waited for
  auto token = [&](int j) {
    const i64 at = r * a.ts0 + j * a.ts1;
    return a.tok64 ? static_cast<const i64*>(a.tokens)[at] : (i64) static_cast<const int*>(a.tokens)[at];
  };
  i64 tok = -1;
  float x_tok = 0.0f;
  if (part == 0 && tid < a.m) {
    tok = token(tid);
    if (tok >= 0 && tok < a.vocab) x_tok = to_f32(row[tok]);
  }

  SoftPair mine;
  float limit = INFINITY;  // only elements that reach it can be among the alternatives
  auto push = [&](float x, int index) {
    if (x >= limit) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kLpCandidates) sh.found[at] = rank_key(x, (u32)index);
    }
  };
  // Every thread copies its own vectors to its own places in shared memory and reads them back, so a
  // stage needs no barrier, and what is on its way takes no registers.
  // (`whole`: a stage of which every thread has all its vectors, which is every one but a row's last.)
  constexpr int each = nt * kLpUnroll;
  const int n = v1 - v0, full = n / each;
  const T* from = row + rs.head + (i64)(v0 + tid) * V;  // of the next stage to be fetched
  auto fetch = [&](int q) {
    uint4* to = ring + (q & (kLpStages - 1)) * each + tid;
    if (q < full) {
#pragma unroll
      for (int k = 0; k < kLpUnroll; ++k) copy_async(to + k * nt, from + k * nt * V);
    } else {
#pragma unroll
      for (int k = 0; k < kLpUnroll; ++k)
        if (q * each + k * nt + tid < n) copy_async(to + k * nt, from + k * nt * V);
    }
    from += each * V;
    copy_async_commit();
  };
  auto take = [&](int q, float (&f)[kLpUnroll * V], bool whole) {
    const uint4* at = ring + (q & (kLpStages - 1)) * each + tid;
    float largest = -INFINITY;
#pragma unroll
    for (int k = 0; k < kLpUnroll; ++k) {
      uint4 raw;
      if (whole || q * each + k * nt + tid < n) raw = at[k * nt];
      else raw = minus_inf<T>();
      float g[V];
      unpack(raw, g, static_cast<const T*>(nullptr));
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[k * V + j] = g[j];
        largest = fmaxf(largest, g[j]);
      }
    }
    return largest;
  };
#pragma unroll
  for (int q = 0; q < kLpStages; ++q) fetch(q);
  float f[kLpUnroll * V];
  if constexpr (TOP) {
    // A bound below which no element can be among the `top` largest: that many threads have one above
    // it in the first stages.  The largest 16-bit prefix of the threads' maxima that `top` of them reach.
    copy_async_wait<0>();
    float largest = fx[0];
#pragma unroll 1
    for (int q = 0; q < kLpStages; ++q) largest = fmaxf(largest, take(q, f, false));
    u32 own = extra || tid < n ? order_of(largest) >> 16 : 0;
    if (own > 0xff80u) own = 0xff80u;  // a NaN: the slow way will see it
    u32 prefix = 0;
    for (int bit = 15; bit >= 0; --bit) {
      const u32 probe = prefix | (1u << bit);
      if (__syncthreads_count(own >= probe) >= a.top) prefix = probe;
    }
    limit = prefix <= 0x7fu ? -INFINITY : value_of(prefix << 16);
    if (extra) push(fx[0], i_extra);
  }
  auto work = [&](int q, bool whole) {
    copy_async_wait<kLpStages - 1>();
    const float largest = take(q, f, whole);
    fetch(q + kLpStages);
    mine.add_all(f, largest, c);
    if constexpr (TOP) {
      if (largest >= limit) {
#pragma unroll
        for (int k = 0; k < kLpUnroll; ++k) {
          const int v = q * each + k * nt + tid;
          if (v < n) {
#pragma unroll
            for (int j = 0; j < V; ++j) push(f[k * V + j], rs.head + (v0 + v) * V + j);
          }
        }
      }
    }
  };
#pragma unroll 1
  for (int q = 0; q < full; ++q) work(q, true);
  if (full * each < n) work(full, false);
  copy_async_wait<0>();
  Soft soft = mine.sum();
  soft.add(fx, fx[0], c);

  if constexpr (TOP) {
    const bool nan = __syncthreads_or(soft.s != soft.s) != 0;
    if (nan || sh.count > kLpCandidates) {
      slow_top<T>(row, rs, v0, v1, extra, fx[0], i_extra, a.top, sh);
      __syncthreads();
    }
    rank_keys(sh.found, sh.count, a.top, sh.best);
  }
  soft.warp_sum(c);
  if ((tid & 31) == 0) sh.warp[tid >> 5] = soft;
  __syncthreads();
  const int warps = nt >> 5;
  if (tid < 32) {
    soft = no_soft();
    if (tid < warps) soft = sh.warp[tid];
    soft.warp_sum(c);
  }
  if (parts > 1) {
    cluster.sync();  // every CTA of the cluster has started: its shared memory may be written
    if (tid == 0) *cluster.map_shared_rank(&sh.part[part], 0) = soft;
    if constexpr (TOP) {
      if (tid < a.top) *cluster.map_shared_rank(&sh.merge[part * a.top + tid], 0) = sh.best[tid];
    }
    cluster.sync();
    if (part != 0) return;
    if (tid < 32) {
      soft = no_soft();
      if (tid < parts) soft = sh.part[tid];
      soft.warp_sum(c);
    }
    if constexpr (TOP) {
      if (tid < kLpMaxTop) sh.best[tid] = 0;
      __syncthreads();
      rank_keys(sh.merge, parts * a.top, a.top, sh.best);
    }
  }
  if (tid == 0) sh.warp[0] = soft;
  __syncthreads();
  soft = sh.warp[0];
  // A row without a finite logit has s = 0: its log probabilities and its normaliser are -inf, its entropy 0.
  const bool none = soft.s == 0.0f;
  const float ln_s = logf(soft.s);
  auto log_prob = [&](float x) { return none ? (x != x ? x : -INFINITY) : (x - soft.m) * a.scale - ln_s; };
  if (tid == 0) {
    a.lse[r] = none ? -INFINITY : fmaf(soft.m, a.scale, ln_s);
    a.entropy[r] = none ? 0.0f : ln_s - kLn2 * (soft.t / soft.s);
  }
  for (int j = tid; j < a.m; j += nt) {
    if (j != tid) {
      tok = token(j);
      if (tok >= 0 && tok < a.vocab) x_tok = to_f32(row[tok]);
    }
    float lp = 0.0f;                              // a negative token is padding
    if (tok >= a.vocab) lp = as_f(0x7fffffffu);   // one that does not exist has no probability to report
    else if (tok >= 0) lp = log_prob(x_tok);
    a.logp[r * a.m + j] = lp;
  }
  if constexpr (TOP) {
    if (tid < a.top) {
      const u64 k = sh.best[tid];
      a.top_logp[r * a.top + tid] = log_prob(value_of((u32)(k >> 32)));
      a.top_ids[r * a.top + tid] = (i64)(0xffffffffu - (u32)k);
    }
  }
}

// Beyond this |lse| the float32 normaliser alone says too little about ln p (its own rounding is 6e-5
// there), and one of -inf does not say whether it stands for a row without a finite logit or for
// logits whose scaled value leaves float32: the gradient then sums the row again.
constexpr float kLpFarLse = 1024.0f;

template <class T>
__device__ __noinline__ Soft row_softmax(const T* row, const RowSplit<T> rs, int vocab, float c) {
  constexpr int V = kVecOf<T>;
  __shared__ Soft warps[8];
  Soft soft = no_soft();
  for (int v = threadIdx.x; v < rs.nvec; v += (int)blockDim.x) {
    float f[V], largest = -INFINITY;
    unpack(*reinterpret_cast<const uint4*>(row + rs.head + (i64)v * V), f, static_cast<const T*>(nullptr));
#pragma unroll
    for (int j = 0; j < V; ++j) largest = fmaxf(largest, f[j]);
    soft.add(f, largest, c);
  }
  if ((int)threadIdx.x < rs.head + rs.tail) {
    const int i = (int)threadIdx.x < rs.head ? threadIdx.x : vocab - rs.tail + threadIdx.x - rs.head;
    const float f[1] = {to_f32(row[i])};
    soft.add(f, f[0], c);
  }
  soft.warp_sum(c);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = soft;
  __syncthreads();
  soft = no_soft();
  if ((threadIdx.x & 31) < blockDim.x >> 5) soft = warps[threadIdx.x & 31];
  soft.warp_sum(c);
  return soft;
}

struct LogprobGradArgs {
  const void* x;
  const void* tokens;
  const float *entropy, *lse, *dlogp, *dentropy, *dlse;
  void* dx;
  i64 row_stride, dx_stride, ts0, ts1;
  int vocab, m, parts;
  float scale;
  bool tok64;
};

// dz = p (A - dH (ln p + H)) + sum of dlogp at the row's tokens, with A = dlse - sum dlogp.
template <class T>
__global__ void __launch_bounds__(256) logprobs_grad_kernel(const __grid_constant__ LogprobGradArgs a) {
  constexpr int V = kVecOf<T>;
  __shared__ float red[8];
  const i64 r = blockIdx.x / (unsigned)a.parts;
  const int part = (int)(blockIdx.x - (unsigned)(r * a.parts)), tid = threadIdx.x, nt = blockDim.x;
  const T* row = static_cast<const T*>(a.x) + r * a.row_stride;
  T* out = static_cast<T*>(a.dx) + r * a.dx_stride;
  const RowSplit<T> rs(row, a.vocab);
  const int per = (rs.nvec + a.parts - 1) / a.parts;
  const int v0 = min(part * per, rs.nvec), v1 = min(v0 + per, rs.nvec);
  auto token = [&](int j) {
    const i64 at = r * a.ts0 + j * a.ts1;
    return a.tok64 ? static_cast<const i64*>(a.tokens)[at] : (i64) static_cast<const int*>(a.tokens)[at];
  };
  uint4 raw[kLpGradUnroll];
#pragma unroll
  for (int k = 0; k < kLpGradUnroll; ++k) {
    const int v = v0 + k * nt + tid;
    if (v < v1) raw[k] = ld_v4(row + rs.head + (i64)v * V);
  }
  float g = 0.0f;  // sum of the gradients of the tokens that count
  if (a.dlogp) {
    for (int j = tid; j < a.m; j += nt) {
      const i64 tok = token(j);
      if (tok >= 0 && tok < a.vocab) g += a.dlogp[r * a.m + j];
    }
    for (int o = 16; o; o >>= 1) g += __shfl_xor_sync(0xffffffffu, g, o);
    if ((tid & 31) == 0) red[tid >> 5] = g;
    __syncthreads();
    g = 0.0f;
    for (int w = 0; w < (nt >> 5); ++w) g += red[w];
  }
  const float lse = a.lse[r], dH = a.dentropy ? a.dentropy[r] : 0.0f, H = a.dentropy ? a.entropy[r] : 0.0f;
  const float A = (a.dlse ? a.dlse[r] : 0.0f) - g;
  const float c = a.scale * kLog2e;
  float m = 0.0f, off = lse * kLog2e;
  if (fabsf(lse) > kLpFarLse) {
    const Soft soft = row_softmax<T>(row, rs, a.vocab, c);
    m = soft.m;
    // no finite logit: no distribution, no gradient; every p becomes 0
    off = soft.s == 0.0f ? INFINITY : log2f(soft.s);
  }
  // with u = ln p / ln 2: dx = 2^u (slope u + level)
  const float slope = -dH * kLn2 * a.scale, level = (A - dH * H) * a.scale;
  const Two minus_m(-m, -m), cc(c, c), minus_off(-off, -off), slopes(slope, slope), levels(level, level);
  auto grad = [&](float& x0, float& x1) {
    float u0, u1;
    fma(add(Two(x0, x1), minus_m), cc, minus_off).get(u0, u1);
    u0 = hold(u0);
    u1 = hold(u1);
    mul(Two(ex2(u0), ex2(u1)), fma(slopes, Two(u0, u1), levels)).get(x0, x1);
  };
  const bool wide = ((reinterpret_cast<u64>(row) ^ reinterpret_cast<u64>(out)) & 15u) == 0;
  for (int base = v0; base < v1; base += nt * kLpGradUnroll) {
    float f[kLpGradUnroll][V];
#pragma unroll
    for (int k = 0; k < kLpGradUnroll; ++k) {
      if (base != v0) {
        const int v = base + k * nt + tid;
        if (v < v1) raw[k] = ld_v4(row + rs.head + (i64)v * V);
      }
    }
#pragma unroll
    for (int k = 0; k < kLpGradUnroll; ++k) {
      const int v = base + k * nt + tid;
      if (v >= v1) break;
      unpack(raw[k], f[k], static_cast<const T*>(nullptr));
#pragma unroll
      for (int j = 0; j < V; j += 2) grad(f[k][j], f[k][j + 1]);
      T* to = out + rs.head + (i64)v * V;
      if (wide) st_v4(to, pack(f[k], static_cast<const T*>(nullptr)));
      else {
#pragma unroll
        for (int j = 0; j < V; ++j) to[j] = from_f32<T>(f[k][j]);
      }
    }
  }
  auto grad_at = [&](i64 i) {
    float x = to_f32(row[i]), y = x;
    grad(x, y);
    return x;
  };
  if (part == 0 && tid < rs.head + rs.tail) {
    const int i = tid < rs.head ? tid : a.vocab - rs.tail + tid - rs.head;
    out[i] = from_f32<T>(grad_at(i));
  }
  if (!a.dlogp || off == INFINITY) return;
  // The tokens' own elements again, with their share: computed in full and rounded once.  The CTA
  // that wrote the element writes it again, and of equal tokens the first one stands for all.
  __syncthreads();
  for (int j = tid; j < a.m; j += nt) {
    const i64 tok = token(j);
    if (tok < 0 || tok >= a.vocab) continue;
    const int v = ((int)tok - rs.head) / V;  // of no vector: CTA 0
    const bool in_vec = tok >= rs.head && v < rs.nvec;
    if (in_vec ? (v < v0 || v >= v1) : part != 0) continue;
    float sum = 0.0f;
    bool mine = true;
    for (int i = 0; i < a.m && mine; ++i) {
      if (i != j && token(i) != tok) continue;
      if (i < j) mine = false;
      sum += a.dlogp[r * a.m + i];
    }
    if (mine) out[tok] = from_f32<T>(fmaf(sum, a.scale, grad_at(tok)));
  }
}

static int check_logprobs(const char* name, const TwgLogprobsDesc* d) {
  TWG_REQUIRE(d != nullptr, "%s: descriptor is null", name);
  TWG_REQUIRE(float_size(d->dtype) != 0, "%s: element type %d is not float32, float16 or bfloat16", name, d->dtype);
  TWG_REQUIRE(d->token_dtype == TWG_DTYPE_I32 || d->token_dtype == TWG_DTYPE_I64, "%s: tokens must be int32 or int64", name);
  TWG_REQUIRE(d->rows >= 0 && d->rows <= (int64_t(1) << 27), "%s: %lld rows are outside 0..2^27", name, (long long)d->rows);
  TWG_REQUIRE(d->vocab >= 1 && d->vocab <= (int64_t(1) << 30), "%s: a vocabulary of %lld is outside 1..2^30", name, (long long)d->vocab);
  TWG_REQUIRE(d->rows <= 1 || d->row_stride >= d->vocab, "%s: row stride %lld is smaller than the vocabulary %lld", name,
              (long long)d->row_stride, (long long)d->vocab);
  TWG_REQUIRE(d->tokens_per_row >= 0 && d->tokens_per_row <= TWG_LOGPROBS_MAX_TOKENS, "%s: %d tokens a row; at most %d are supported", name,
              d->tokens_per_row, TWG_LOGPROBS_MAX_TOKENS);
  TWG_REQUIRE(d->top >= 0 && d->top <= kLpMaxTop && d->top <= d->vocab, "%s: %d alternatives; at most %d and no more than the vocabulary", name,
              d->top, kLpMaxTop);
  TWG_REQUIRE(d->scale > 0.0f && d->scale <= FLT_MAX / 2, "%s: scale must be positive and finite", name);
  return TWG_OK;
}

template <class T>
static int launch_logprobs(const LogprobArgs& a, int64_t rows, cudaStream_t s) {
  const int nvec = std::max(1, a.vocab / kVecOf<T>);
  // CTAs per row: as many as keep two on every SM, while each still has a round of its threads' loads
  int parts = 1;
  while (parts < kLpMaxCluster && rows * parts * 2 <= 2 * sm_count() && nvec / (parts * 2) >= 256) parts *= 2;
  // half the threads where a row has no vector for every one of them
  const int each = (nvec + parts - 1) / parts;
  const int threads = each < kLpMaxThreads ? kLpMaxThreads / 2 : kLpMaxThreads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = sizeof(uint4) * kLpStages * kLpUnroll * (size_t)threads;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)parts, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool small = threads < kLpMaxThreads;
  if (a.top) TWG_CUDA(cudaLaunchKernelEx(&cfg, small ? logprobs_kernel<T, true, kLpMaxThreads / 2> : logprobs_kernel<T, true, kLpMaxThreads>, a));
  else TWG_CUDA(cudaLaunchKernelEx(&cfg, small ? logprobs_kernel<T, false, kLpMaxThreads / 2> : logprobs_kernel<T, false, kLpMaxThreads>, a));
  TWG_CHECK_LAUNCH();
  return TWG_OK;
}
template <class T>
static int launch_logprobs_grad(LogprobGradArgs& a, int64_t rows, cudaStream_t s) {
  const int nvec = std::max(1, a.vocab / kVecOf<T>);
  int threads = 64;
  while (threads < 256 && threads * kLpGradUnroll < nvec) threads *= 2;
  // one round of loads per CTA, two where that would be too many CTAs for the grid
  // one round of loads in a CTA, or kLpGradRounds where the rows still make eight CTAs for every SM: what a
  // CTA does before its first element counts for less then
  const int64_t rounds = rows * nvec >= (int64_t)sm_count() * 8 * threads * kLpGradUnroll * kLpGradRounds ? kLpGradRounds : 1;
  const int64_t each = threads * kLpGradUnroll * rounds;
  int64_t parts = (nvec + each - 1) / each;
  while (parts > 1 && rows * parts > 0x7fffffff) parts = (parts + 1) / 2;
  a.parts = (int)parts;
  logprobs_grad_kernel<T><<<(unsigned)(rows * parts), threads, 0, s>>>(a);
  TWG_CHECK_LAUNCH();
  return TWG_OK;
}

}  // namespace twg

using namespace twg;

extern "C" int twg_token_logprobs(const TwgLogprobsDesc* d, const void* logits, const void* tokens, float* logp, float* entropy,
                                  float* lse, float* top_logp, int64_t* top_ids, void* stream) {
  const char* name = "twg_token_logprobs";
  TWG_TRACE("twg_token_logprobs");
  g_last_path = kPathNone;
  if (int rc = check_logprobs(name, d)) return rc;
  if (d->rows == 0) return TWG_OK;
  TWG_REQUIRE(logits && entropy && lse, "%s: logits, entropy or lse is null", name);
  TWG_REQUIRE(d->tokens_per_row == 0 || (tokens && logp), "%s: tokens or logp is null", name);
  TWG_REQUIRE(d->top == 0 || (top_logp && top_ids), "%s: top_logp or top_ids is null", name);
  TWG_REQUIRE(is_aligned(logits, (size_t)float_size(d->dtype)), "%s: logits are not aligned to their elements", name);
  TWG_REQUIRE(is_aligned(tokens, d->token_dtype == TWG_DTYPE_I64 ? 8 : 4) && is_aligned(top_ids, 8), "%s: tokens or top_ids are misaligned", name);
  LogprobArgs a = {};
  a.x = logits; a.tokens = tokens;
  a.logp = logp; a.entropy = entropy; a.lse = lse; a.top_logp = top_logp;
  a.top_ids = reinterpret_cast<i64*>(top_ids);
  a.row_stride = d->row_stride; a.ts0 = d->token_strides[0]; a.ts1 = d->token_strides[1];
  a.vocab = (int)d->vocab; a.m = d->tokens_per_row; a.top = d->top;
  a.scale = d->scale;
  a.tok64 = d->token_dtype == TWG_DTYPE_I64;
  const int rc = dispatch_float(d->dtype, [&](auto* t) {
    return launch_logprobs<std::remove_pointer_t<decltype(t)>>(a, d->rows, static_cast<cudaStream_t>(stream));
  });
  if (rc == TWG_OK) g_last_path = kPathDense;
  return rc;
}

extern "C" int twg_token_logprobs_backward(const TwgLogprobsDesc* d, const void* logits, const void* tokens, const float* entropy,
                                           const float* lse, const float* dlogp, const float* dentropy, const float* dlse,
                                           void* dlogits, int64_t dlogits_row_stride, void* stream) {
  const char* name = "twg_token_logprobs_backward";
  TWG_TRACE("twg_token_logprobs_backward");
  g_last_path = kPathNone;
  if (int rc = check_logprobs(name, d)) return rc;
  TWG_REQUIRE(d->rows <= 1 || dlogits_row_stride >= d->vocab, "%s: row stride %lld of dlogits is smaller than the vocabulary %lld", name,
              (long long)dlogits_row_stride, (long long)d->vocab);
  if (d->rows == 0) return TWG_OK;
  TWG_REQUIRE(logits && lse && dlogits, "%s: logits, lse or dlogits is null", name);
  TWG_REQUIRE(!dentropy || entropy, "%s: the entropy's gradient needs the entropy", name);
  TWG_REQUIRE(!dlogp || d->tokens_per_row == 0 || tokens, "%s: tokens is null", name);
  TWG_REQUIRE(is_aligned(logits, (size_t)float_size(d->dtype)) && is_aligned(dlogits, (size_t)float_size(d->dtype)),
              "%s: logits or dlogits are not aligned to their elements", name);
  TWG_REQUIRE(is_aligned(tokens, d->token_dtype == TWG_DTYPE_I64 ? 8 : 4), "%s: tokens are misaligned", name);
  LogprobGradArgs a = {};
  a.x = logits; a.tokens = tokens;
  a.entropy = entropy; a.lse = lse;
  a.dlogp = d->tokens_per_row ? dlogp : nullptr;
  a.dentropy = dentropy; a.dlse = dlse;
  a.dx = dlogits;
  a.row_stride = d->row_stride; a.dx_stride = dlogits_row_stride;
  a.ts0 = d->token_strides[0]; a.ts1 = d->token_strides[1];
  a.vocab = (int)d->vocab; a.m = d->tokens_per_row;
  a.scale = d->scale;
  a.tok64 = d->token_dtype == TWG_DTYPE_I64;
  const int rc = dispatch_float(d->dtype, [&](auto* t) {
    return launch_logprobs_grad<std::remove_pointer_t<decltype(t)>>(a, d->rows, static_cast<cudaStream_t>(stream));
  });
  if (rc == TWG_OK) g_last_path = kPathDense;
  return rc;
}
