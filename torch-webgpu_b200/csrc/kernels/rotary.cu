// Rotation of queries and keys by positions on one or several axes, with or without the norm of
// every head in front of it, and the gradient of both.
//
//   theta_j = positions[axis_of[j], b, s] * inv_freq[j]                        j in [0, R/2)
//   (u, v) -> (u cos theta - v sin theta, v cos theta + u sin theta)           pairs (j, j + R/2) or (2j, 2j + 1)
//   norm:     x -> x * rsqrt(mean(x^2) + eps) * w                              before the rotation, over the head
//
// Bound by HBM: every element is read once and written once (the gradient of the norm reads x and
// dy and writes dx), about ten instructions per element in between.  One row is one head of one
// token.  A group of lanes owns a row, each lane two 16-byte vectors that hold both partners of
// its pairs, so a row is in registers between its load and its store and the norm's sum is a few
// shuffles (heads that 16 bytes do not divide take vectors of 8 or 4, or single elements).  The angle is the only part that needs more than 32 bits (a position of 10^6 leaves
// 2^-4 of a turn in float32): it is formed in float64 or as a 64-bit fraction of a turn, once per token
// and frequency, and its sine and cosine wait for every head of the token.
#include "twg_float.cuh"

namespace twg {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;
constexpr int kRotRounds = 10;         // rows of a lane group in a warp's tile, where there are enough
constexpr int kRotMaxTile = 16;        // tokens in such a tile
constexpr int kRotTable = 512;         // entries of its tables
constexpr int kRotStages = 2;          // rounds of the gradient's rows on their way
constexpr int kRotMaxDim = 512;
constexpr int kRotMaxAxes = 8;
constexpr int kRotGradCtas = 148 * 2;  // CTAs of the gradient kernel: one row of weight partial sums each

struct RotaryArgs {
  const void* x[2];  // q, k
  const void* g[2];  // gradients of the outputs (backward only)
  void* y[2];
  const void* w[2];
  i64 xs[2][4], gs[2][4], ys[2][4];  // element strides: batch, seq, head, dim
  int heads[2];
  const void* pos;
  i64 ps[3];  // axis, batch, seq
  const void* freq;
  u32 seq, tokens;
  int D, R, slots, lanes;  // lanes: of a row's group (a power of two where a sum goes over it)
  int tile, head_span, parts;  // forward: tokens and heads per warp, warps per token
  int step[2];             // backward: heads of q and of k that one round of a warp's lane groups takes (a power of two)
  int ctas[2];             // CTAs that work on q and on k (backward)
  float* partial;          // backward: [ctas[0] + ctas[1]][D]
  const float* table;      // backward: rotary_table_kernel's
  float eps;
  float sign;              // -1 rotates backwards
  bool pos64, freq64, w32, adjacent;
  u8 axis_of[TWG_ROTARY_MAX_FREQS];
};

// Where table entry / weight j of slot p lies in shared memory: quads of one j are contiguous over
// the slots, so that the 16-byte reads of a group's lanes hit different banks.
template <int V>
__device__ __forceinline__ int spot(int p, int j, int slots) {
  if constexpr (V <= 2) return p * V + j;
  else return ((j >> 2) * slots + p) * 4 + (j & 3);
}
// First elements of the two vectors of slot p.
__device__ __forceinline__ void slot_elems(const RotaryArgs& a, int p, int V, int* e0, int* e1) {
  const int half = a.R >> 1;
  if (!a.adjacent && p * V < half) { *e0 = p * V; *e1 = p * V + half; }
  else { *e0 = 2 * p * V; *e1 = *e0 + V; }
}
// The elements of pair j of slot p: partners of one angle, or neighbours behind the turned part.
__device__ __forceinline__ void pair_elems(const RotaryArgs& a, int p, int j, int V, int* ea, int* eb) {
  if (a.adjacent) {
    *ea = 2 * (p * V + j);
    *eb = *ea + 1;
  } else {
    slot_elems(a, p, V, ea, eb);
    *ea += j;
    *eb += j;
  }
}

__device__ __forceinline__ void token_place(const RotaryArgs& a, u32 tok, i64* b, i64* s) {
  const u32 q = tok / a.seq;
  *b = q;
  *s = tok - q * a.seq;
}

// Sine and cosine of an angle in 2^-32 turns.  The two top bits round to a quarter turn; what is left
// is at most pi / 4, where the Taylor series reach float32 with y^9 and y^10 (the next terms are below
// 2^-28 of the result), and the quarters swap and negate them.
__device__ __forceinline__ void turn_sincos(u32 turn, float* s, float* c) {
  const u32 quarter = (turn + 0x20000000u) >> 30;
  const float y = (float)(int)(turn - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = y * y;
  float p = fmaf(z, 2.7557319e-6f, -1.9841270e-4f), q = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  p = fmaf(z, p, 8.3333333e-3f);
  q = fmaf(z, q, -1.3888889e-3f);
  p = fmaf(z, p, -1.6666667e-1f);
  q = fmaf(z, q, 4.1666667e-2f);
  q = fmaf(z, q, -0.5f);
  const float sy = fmaf(y * z, p, y), cy = fmaf(z, q, 1.0f);
  const float a = quarter & 1u ? cy : sy, b = quarter & 1u ? sy : cy;
  *s = as_f(as_u(a) ^ ((quarter & 2u) << 30));
  *c = as_f(as_u(b) ^ (((quarter + 1u) & 2u) << 30));
}
__device__ __forceinline__ i64 position_at(const RotaryArgs& a, i64 off) {
  return a.pos64 ? static_cast<const i64*>(a.pos)[off] : (i64) static_cast<const int*>(a.pos)[off];
}
__device__ __forceinline__ double freq_at(const RotaryArgs& a, int f) {
  return a.freq64 ? static_cast<const double*>(a.freq)[f] : (double)static_cast<const float*>(a.freq)[f];
}
// Sine and cosine of frequency f at a token; the identity behind the turned part.
__device__ __forceinline__ void angle(const RotaryArgs& a, int f, i64 at_token, float* c, float* s) {
  *c = 1.0f;
  *s = 0.0f;
  if (f >= (a.R >> 1)) return;
  double turns = (double)position_at(a, (i64)a.axis_of[f] * a.ps[0] + at_token) * freq_at(a, f) * 0.15915494309189533577;  // 1 / (2 pi)
  turns -= rint(turns);
  turn_sincos((u32)__double2int_rn(turns * 4294967296.0), s, c);
  if (!isfinite(turns)) *c = *s = as_f(0x7fffffffu);
  *s *= a.sign;
}

// Weights of one tensor by pairs: of the first partners, then of the second ones.
template <class T, int V>
__device__ __forceinline__ void fill_weights(const RotaryArgs& a, int tensor, float* w) {
  const int row = a.slots * V;
  for (int i = threadIdx.x; i < 2 * row; i += (int)blockDim.x) {
    const int second = i >= row, f = i - second * row;
    int e[2];
    pair_elems(a, f / V, f % V, V, &e[0], &e[1]);
    const int el = e[second];
    float v = 1.0f;
    if (a.w[tensor] && el < a.D)
      v = a.w32 ? static_cast<const float*>(a.w[tensor])[el] : to_f32(static_cast<const T*>(a.w[tensor])[el]);
    w[second * row + spot<V>(f / V, f % V, a.slots)] = v;
  }
}

template <int V>
__device__ __forceinline__ void read_row(const float* tab, int p, int slots, float (&out)[V]) {
  if constexpr (V == 1) out[0] = tab[p];
  else if constexpr (V == 2) {
    const float2 v = *reinterpret_cast<const float2*>(tab + 2 * p);
    out[0] = v.x; out[1] = v.y;
  } else {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const float4 v = *reinterpret_cast<const float4*>(tab + (q * slots + p) * 4);
      out[4 * q] = v.x; out[4 * q + 1] = v.y; out[4 * q + 2] = v.z; out[4 * q + 3] = v.w;
    }
  }
}

// Raw contents of the two vectors of a lane's slot (or its two elements on the scalar path).
template <class T, int V>
struct Raw {
  typename VecBytes<V * (int)sizeof(T)>::type a, b;
};
template <class T>
struct Raw<T, 1> {
  float a, b;
};

// The pairs of a lane's slot.
template <class T, int V, bool ADJ>
__device__ __forceinline__ void to_pairs(const Raw<T, V>& r, float (&a)[V], float (&b)[V]) {
  if constexpr (V == 1) { a[0] = r.a; b[0] = r.b; }
  else if constexpr (!ADJ) {
    unpack(r.a, a, static_cast<const T*>(nullptr));
    unpack(r.b, b, static_cast<const T*>(nullptr));
  } else {
    float u[V], v[V];
    unpack(r.a, u, static_cast<const T*>(nullptr));
    unpack(r.b, v, static_cast<const T*>(nullptr));
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      a[j] = u[2 * j]; b[j] = u[2 * j + 1];
      a[V / 2 + j] = v[2 * j]; b[V / 2 + j] = v[2 * j + 1];
    }
  }
}
template <class T, int V, bool ADJ>
__device__ __forceinline__ void store_pairs(T* row, i64 sd, int e0, int e1, int D, bool on, const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) {
    if (!on) return;
    row[e0 * sd] = from_f32<T>(a[0]);
    if (e1 < D) row[e1 * sd] = from_f32<T>(b[0]);
  } else {
    typename VecBytes<V * (int)sizeof(T)>::type x, y;
    if constexpr (!ADJ) {
      x = pack(a, static_cast<const T*>(nullptr));
      y = pack(b, static_cast<const T*>(nullptr));
    } else {
      float u[V], v[V];
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        u[2 * j] = a[j]; u[2 * j + 1] = b[j];
        v[2 * j] = a[V / 2 + j]; v[2 * j + 1] = b[V / 2 + j];
      }
      x = pack(u, static_cast<const T*>(nullptr));
      y = pack(v, static_cast<const T*>(nullptr));
    }
    if (on) {
      st_vec(row + e0, x);
      st_vec(row + e1, y);
    }
  }
}

// Sum over a row's lane group; LANES: how many where the kernel is made for it, 0: `lanes` of them.
template <int LANES>
__device__ __forceinline__ float group_sum(float v, int lanes) {
  if constexpr (LANES > 0) {
#pragma unroll
    for (int o = LANES / 2; o; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  if (lanes > 16) v += __shfl_xor_sync(0xffffffffu, v, 16);
  if (lanes > 8) v += __shfl_xor_sync(0xffffffffu, v, 8);
  if (lanes > 4) v += __shfl_xor_sync(0xffffffffu, v, 4);
  if (lanes > 2) v += __shfl_xor_sync(0xffffffffu, v, 2);
  if (lanes > 1) v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v;
}

// A lane's V values as they are computed with: two in an instruction, where neighbours are in registers
// side by side, or the one of the element path.  (In scalar form the kernels issued three instructions
// for every two of this one.)
template <int V>
struct Lanes {
  static constexpr int N = V / 2;
  Two x[N];
  __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = Two(f[2 * i], f[2 * i + 1]);
  }
  __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i].get(f[2 * i], f[2 * i + 1]);
  }
  static __device__ __forceinline__ Two all(float f) { return Two(f, f); }
  static __device__ __forceinline__ float sum(Two t) {
    float a, b;
    t.get(a, b);
    return a + b;
  }
};
template <>
struct Lanes<1> {
  static constexpr int N = 1;
  float x[1];
  __device__ __forceinline__ void set(const float (&f)[1]) { x[0] = f[0]; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = x[0]; }
  static __device__ __forceinline__ float all(float f) { return f; }
  static __device__ __forceinline__ float sum(float t) { return t; }
};
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float fma(float a, float b, float c) { return fmaf(a, b, c); }
template <int V>
using Wide = std::conditional_t<V == 1, float, Two>;

// The two vectors (or elements) of a lane's slots in one row.  Without a row the registers keep what
// they hold: a load costs no clearing, and nothing computed from them is stored.
template <class T, int V, int NS>
struct Row {
  Raw<T, V> r[NS];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if constexpr (V == 1) r[i].a = r[i].b = 0.0f;
      else r[i].a = r[i].b = decltype(r[i].a){};
    }
  }
  __device__ __forceinline__ void load(const T* row, i64 sd, const int (&e0)[NS], const int (&e1)[NS], const bool (&has)[NS], int D, bool on) {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if (!has[i]) continue;
      if constexpr (V == 1) {
        r[i].a = to_f32(row[e0[i] * sd]);
        if (e1[i] < D) r[i].b = to_f32(row[e1[i] * sd]);
      } else {
        ld_vec(r[i].a, row + e0[i]);
        ld_vec(r[i].b, row + e1[i]);
      }
    }
  }
};

// The row a lane group works on: token within the warp's tile and head within its span.
struct Place {
  int t, h;
  __device__ __forceinline__ Place(int group, int span) : t(group / span), h(group - t * span) {}
  __device__ __forceinline__ void advance(int groups, int span) {
    h += groups;
    while (h >= span) {
      h -= span;
      ++t;
    }
  }
};

// Forward: every warp works by itself on `tile` tokens and `head_span` of their q and k heads, about
// kRotRounds rows to a lane group.  It issues the loads of its first rows, forms the tables while
// they travel, and from then on always has the next rows on their way.  16384 tokens of 32 + 8 heads
// of 128 in bfloat16 take 60.9 us (5.5 TB/s, 84 % of the copy bandwidth; 61.7 with five CTAs an SM, whose
// 48 registers spill, 64.9 with three).  Measured and dropped: tables
// of a CTA behind a barrier 63.9 us; no loop, one or two rows to a lane group 76 and 61 us (82 us where
// the norm's weights add to what a CTA does first, 59.7 us here); the cosines of a token in registers
// and rows two at a time 66 to 70 us; angles from 64-bit fractions of a turn instead of float64 65 us.
template <class T, int V, int NS, bool NORM, bool ADJ, int LANES>
__global__ void __launch_bounds__(kRotThreads, V > 1 ? 4 : 1) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) float smem[];
  __shared__ i64 all_offs[kRotWarps][kRotMaxTile][4];  // token offsets of q, k, q_out, k_out
  const int row = a.slots * V, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* w = smem;  // NORM: q's weights, then k's
  float* cosine = smem + (NORM ? 4 * row : 0) + warp * 2 * a.tile * row;
  float* sine = cosine + a.tile * row;
  auto& offs = all_offs[warp];
  const u32 unit = blockIdx.x * kRotWarps + warp, tile = unit / (u32)a.parts;
  const int h0 = (int)(unit - tile * (u32)a.parts) * a.head_span, span = min(a.head_span, a.heads[0] + a.heads[1] - h0);
  const i64 tok0 = (i64)tile * a.tile;
  const int ntok = (int)max((i64)0, min((i64)a.tile, (i64)a.tokens - tok0));
  if (lane < ntok) {
    i64 b, s;
    token_place(a, (u32)tok0 + lane, &b, &s);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      offs[lane][t] = b * a.xs[t][0] + s * a.xs[t][1];
      offs[lane][2 + t] = b * a.ys[t][0] + s * a.ys[t][1];
    }
  }
  __syncwarp();

  const int lanes = LANES ? LANES : a.lanes, groups = 32 / lanes, group = lane / lanes, p0 = lane - group * lanes;
  int e0[NS], e1[NS];
  bool has[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    slot_elems(a, p0 + 32 * i, V, &e0[i], &e1[i]);
    has[i] = p0 + 32 * i < a.slots && group < groups;
  }
  Row<T, V, NS> x;
  x.clear();
  auto fetch = [&](const Place& at) {
    const bool on = at.t < ntok;
    const int h = h0 + at.h, z = h >= a.heads[0] ? 1 : 0;
    x.load(static_cast<const T*>(a.x[z]) + (on ? offs[at.t][z] : 0) + (i64)(h - (z ? a.heads[0] : 0)) * a.xs[z][2], a.xs[z][3], e0, e1, has,
           a.D, on);
  };
  Place at(group, span);
  fetch(at);
  for (int t = 0; t < ntok; ++t) {
    i64 b, s;
    token_place(a, (u32)tok0 + (u32)t, &b, &s);
    for (int f = lane; f < row; f += 32) {
      float c, sn;
      angle(a, f, b * a.ps[1] + s * a.ps[2], &c, &sn);
      cosine[t * row + spot<V>(f / V, f % V, a.slots)] = c;
      sine[t * row + spot<V>(f / V, f % V, a.slots)] = sn;
    }
  }
  if constexpr (NORM) {
    fill_weights<T, V>(a, 0, w);
    fill_weights<T, V>(a, 1, w + 2 * row);
    __syncthreads();
  } else {
    __syncwarp();
  }
  const float inv_d = 1.0f / (float)a.D;
  for (int left = ntok * span; left > 0; left -= groups) {
    const bool on = at.t < ntok;
    const int t = on ? at.t : 0, h = h0 + at.h, z = h >= a.heads[0] ? 1 : 0;
    Lanes<V> u[NS], v[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float f[V], g[V];
      to_pairs<T, V, ADJ>(x.r[i], f, g);
      u[i].set(f);
      v[i].set(g);
    }
    at.advance(groups, span);
    fetch(at);
    if constexpr (NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        Wide<V> s0 = mul(u[i].x[0], u[i].x[0]), s1 = mul(v[i].x[0], v[i].x[0]);
#pragma unroll
        for (int j = 1; j < Lanes<V>::N; ++j) {
          s0 = fma(u[i].x[j], u[i].x[j], s0);
          s1 = fma(v[i].x[j], v[i].x[j], s1);
        }
        ss += Lanes<V>::sum(s0) + Lanes<V>::sum(s1);
      }
      const Wide<V> r = Lanes<V>::all(rsqrtf(fmaf(group_sum<LANES>(ss, lanes), inv_d, a.eps)));
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        float f[V], g[V];
        const float* wz = w + z * 2 * row;
        const int p = has[i] ? p0 + 32 * i : 0;
        read_row<V>(wz, p, a.slots, f);
        read_row<V>(wz + row, p, a.slots, g);
        Lanes<V> A, B;
        A.set(f);
        B.set(g);
#pragma unroll
        for (int j = 0; j < Lanes<V>::N; ++j) {
          u[i].x[j] = mul(u[i].x[j], mul(A.x[j], r));
          v[i].x[j] = mul(v[i].x[j], mul(B.x[j], r));
        }
      }
    }
    T* out = static_cast<T*>(a.y[z]) + offs[t][2 + z] + (i64)(h - (z ? a.heads[0] : 0)) * a.ys[z][2];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float f[V], g[V];
      const int p = has[i] ? p0 + 32 * i : 0;
      read_row<V>(cosine + t * row, p, a.slots, f);
      read_row<V>(sine + t * row, p, a.slots, g);
      Lanes<V> C, S, A, B;
      C.set(f);
      S.set(g);
#pragma unroll
      for (int j = 0; j < Lanes<V>::N; ++j) {
        A.x[j] = fma(u[i].x[j], C.x[j], mul(v[i].x[j], mul(S.x[j], Lanes<V>::all(-1.0f))));
        B.x[j] = fma(v[i].x[j], C.x[j], mul(u[i].x[j], S.x[j]));
      }
      A.get(f);
      B.get(g);
      store_pairs<T, V, ADJ>(out, a.ys[z][3], e0[i], e1[i], a.D, on && has[i], f, g);
    }
  }
}

// Cosines and sines of the gradient's tokens: [tokens][2][slots V], quads of a slot as in shared memory.
// A thread keeps its frequency, as a 64-bit fraction of a turn: positions are whole numbers, so the
// product modulo 2^64 is the angle without its whole turns.
constexpr int kRotTableTokens = 16;  // tokens of a thread, at most
template <int V>
__global__ void __launch_bounds__(kRotThreads) rotary_table_kernel(const __grid_constant__ RotaryArgs a, float* table, int each) {
  const int row = a.slots * V, f = blockIdx.y * blockDim.x + threadIdx.x;
  if (f >= row) return;
  const bool turned = f < (a.R >> 1);
  u64 part = 0;
  float nan = 0.0f;
  if (turned) {
    double turns = freq_at(a, f) * 0.15915494309189533577;  // 1 / (2 pi)
    if (!isfinite(turns)) nan = as_f(0x7fffffffu);
    turns -= floor(turns);
    part = __double2ull_rn(turns * 18446744073709551616.0);
  }
  const i64 axis = turned ? (i64)a.axis_of[f] * a.ps[0] : 0;
  const i64 first = ((i64)blockIdx.x * blockDim.y + threadIdx.y) * each;
  for (i64 tok = first; tok < min(first + each, (i64)a.tokens); ++tok) {
    float c = 1.0f, s = 0.0f;
    if (turned) {
      i64 b, q;
      token_place(a, (u32)tok, &b, &q);
      turn_sincos((u32)((part * (u64)position_at(a, axis + b * a.ps[1] + q * a.ps[2])) >> 32), &s, &c);
      c += nan;
      s = (s + nan) * a.sign;
    }
    float* to = table + tok * 2 * row + spot<V>(f / V, f % V, a.slots);
    to[0] = c;
    to[row] = s;
  }
}

// Gradient of norm and rotation.  With n = x r, r = rsqrt(mean(x^2) + eps), g = dy rotated back and
// h = g w:  dx = r h - x r^3 mean(h x),  dw = sum over rows of g n.  Both sums over the head come
// out of one round of shuffles.  A warp walks the tokens of one tensor, `tp` at a time, and their heads,
// `hp` at a time: lane group g has token g / hp and head g % hp of them.  The next rows are always on
// their way.  dw stays in registers (a lane always owns the same elements); the CTAs' sums are added
// in a fixed order by rotary_weight_grad_kernel, so the gradient does not depend on scheduling.
// The tables come from memory: formed here, between a warp's rows, they cost 40 of 140 us for 16384
// tokens of 32 + 4 heads of 128 in bfloat16.  With them 91 us (5.0 TB/s of x, dy and dx; 16 warps an SM
// by registers, of which half hold dw and the row at hand): neither more rounds on their way nor fewer
// instructions moved it further; one round less (1) costs 8 us, four CTAs an SM in two waves 2 us.
template <class T, int V, int NS, bool ADJ, int LANES>
__global__ void __launch_bounds__(kRotThreads, NS < 8 ? 2 : 1) rotary_grad_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) float smem[];
  const int row = a.slots * V, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* w = smem;
  const int z = (int)blockIdx.x >= a.ctas[0] ? 1 : 0, H = a.heads[z];
  fill_weights<T, V>(a, z, w);
  __syncthreads();

  const int lanes = LANES ? LANES : a.lanes, group = lane / lanes, p0 = lane & (lanes - 1);
  const int hp = a.step[z], tp = 32 / lanes / hp, tl = group / hp, hl = group & (hp - 1);
  const i64 sx = a.xs[z][2] * hp, sg = a.gs[z][2] * hp, sy = a.ys[z][2] * hp;
  const float inv_d = 1.0f / (float)a.D;
  int e0[NS], e1[NS];
  bool has[NS];
  Lanes<V> dwa[NS], dwb[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    slot_elems(a, p0 + 32 * i, V, &e0[i], &e1[i]);
    has[i] = p0 + 32 * i < a.slots;
#pragma unroll
    for (int j = 0; j < Lanes<V>::N; ++j) dwa[i].x[j] = dwb[i].x[j] = Lanes<V>::all(0.0f);
  }
  // A walk over this warp's rounds: the loads' walk is kRotStages rounds ahead of the other one.
  struct Walk {
    u32 tok;  // first of the round's tokens
    int h0;
  };
  const u32 step = (u32)a.ctas[z] * kRotWarps * (u32)tp;
  const u32 start = ((blockIdx.x - (z ? (u32)a.ctas[0] : 0u)) * kRotWarps + warp) * (u32)tp;
  Walk ahead{start, 0}, at{start, 0};
  const T *px = nullptr, *pg = nullptr;
  T* py = nullptr;
  const float* tab = nullptr;
  auto place_in = [&] {  // addresses of this group's token
    i64 b, s;
    token_place(a, min(ahead.tok + (u32)tl, a.tokens - 1), &b, &s);
    px = static_cast<const T*>(a.x[z]) + b * a.xs[z][0] + s * a.xs[z][1] + hl * a.xs[z][2];
    pg = static_cast<const T*>(a.g[z]) + b * a.gs[z][0] + s * a.gs[z][1] + hl * a.gs[z][2];
  };
  auto place_out = [&] {
    const u32 t = min(at.tok + (u32)tl, a.tokens - 1);
    i64 b, s;
    token_place(a, t, &b, &s);
    py = static_cast<T*>(a.y[z]) + b * a.ys[z][0] + s * a.ys[z][1] + hl * a.ys[z][2];
    tab = a.table + (i64)t * 2 * row;
  };
  auto holds = [&](const Walk& w) { return w.tok < a.tokens && w.h0 + hl < H && w.tok + (u32)tl < a.tokens; };
  // Rows on their way: in shared memory, every lane's vectors in its own places (no barrier, and no
  // registers held); the element path reads into registers when it gets there.  Places are zero at
  // first; where a group has no row they hold an earlier row of the same lanes and elements, which
  // then counts times r = 0.
  constexpr int S = V > 1 ? kRotStages : 1;
  using Vec = std::remove_reference_t<decltype(Raw<T, V>::a)>;
  Vec* const ring = reinterpret_cast<Vec*>(w + 2 * row) + threadIdx.x;  // [S][4][threads]
  Row<T, V, NS> xr, gr;
  xr.clear();
  gr.clear();
  int stage_in = 0, stage_out = 0;
  auto fetch = [&] {
    const bool on = holds(ahead);
    if constexpr (V > 1) {
      if (on && has[0]) {
        Vec* to = ring + stage_in * 4 * kRotThreads;
        copy_async(to, px + e0[0]);
        copy_async(to + kRotThreads, px + e1[0]);
        copy_async(to + 2 * kRotThreads, pg + e0[0]);
        copy_async(to + 3 * kRotThreads, pg + e1[0]);
      }
      copy_async_commit();
      stage_in = stage_in + 1 == S ? 0 : stage_in + 1;
    } else {
      xr.load(px, a.xs[z][3], e0, e1, has, a.D, on);
      gr.load(pg, a.gs[z][3], e0, e1, has, a.D, on);
    }
    if (ahead.tok >= a.tokens) return;
    ahead.h0 += hp;
    px += sx;
    pg += sg;
    if (ahead.h0 >= H) {
      ahead.h0 = 0;
      ahead.tok += step;
      if (ahead.tok < a.tokens) place_in();
    }
  };
  if (start < a.tokens) {
    place_in();
    place_out();
  }
  if constexpr (V > 1) {
#pragma unroll
    for (int k = 0; k < 4 * S; ++k) ring[k * kRotThreads] = Vec{};
  }
#pragma unroll
  for (int k = 0; k < S; ++k) fetch();
  while (at.tok < a.tokens) {
    if constexpr (V > 1) {
      copy_async_wait<S - 1>();
      const Vec* from = ring + stage_out * 4 * kRotThreads;
      xr.r[0].a = from[0];
      xr.r[0].b = from[kRotThreads];
      gr.r[0].a = from[2 * kRotThreads];
      gr.r[0].b = from[3 * kRotThreads];
      stage_out = stage_out + 1 == S ? 0 : stage_out + 1;
    }
    const bool now = holds(at);
    Lanes<V> xa[NS], xb[NS], ga[NS], gb[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float f[V], g[V];
      to_pairs<T, V, ADJ>(xr.r[i], f, g);
      xa[i].set(f);
      xb[i].set(g);
      to_pairs<T, V, ADJ>(gr.r[i], f, g);
      ga[i].set(f);
      gb[i].set(g);
    }
    fetch();

    float ss = 0.0f, hx = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float c[V], sn[V], wa[V], wb[V];
      const int p = has[i] ? p0 + 32 * i : 0;
      read_row<V>(tab, p, a.slots, c);
      read_row<V>(tab + row, p, a.slots, sn);
      read_row<V>(w, p, a.slots, wa);
      read_row<V>(w + row, p, a.slots, wb);
      Lanes<V> A, B, C, S;
      A.set(wa);
      B.set(wb);
      C.set(c);
      S.set(sn);
      Wide<V> s0, s1, q0, q1;
#pragma unroll
      for (int j = 0; j < Lanes<V>::N; ++j) {
        const Wide<V> u = ga[i].x[j], v = gb[i].x[j];
        ga[i].x[j] = fma(u, C.x[j], mul(v, mul(S.x[j], Lanes<V>::all(-1.0f))));
        gb[i].x[j] = fma(v, C.x[j], mul(u, S.x[j]));
        const Wide<V> g0 = mul(ga[i].x[j], xa[i].x[j]), g1 = mul(gb[i].x[j], xb[i].x[j]);
        s0 = j ? fma(xa[i].x[j], xa[i].x[j], s0) : mul(xa[i].x[j], xa[i].x[j]);
        s1 = j ? fma(xb[i].x[j], xb[i].x[j], s1) : mul(xb[i].x[j], xb[i].x[j]);
        q0 = j ? fma(g0, A.x[j], q0) : mul(g0, A.x[j]);
        q1 = j ? fma(g1, B.x[j], q1) : mul(g1, B.x[j]);
      }
      ss += Lanes<V>::sum(s0) + Lanes<V>::sum(s1);
      hx += Lanes<V>::sum(q0) + Lanes<V>::sum(q1);
    }
    ss = group_sum<LANES>(ss, lanes);
    hx = group_sum<LANES>(hx, lanes);
    const float r = now ? rsqrtf(fmaf(ss, inv_d, a.eps)) : 0.0f;
    const Wide<V> rr = Lanes<V>::all(r), kk = Lanes<V>::all(-(r * r * r) * (hx * inv_d));
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float wa[V], wb[V], f[V], g[V];
      const int p = has[i] ? p0 + 32 * i : 0;
      read_row<V>(w, p, a.slots, wa);
      read_row<V>(w + row, p, a.slots, wb);
      Lanes<V> A, B;
      A.set(wa);
      B.set(wb);
#pragma unroll
      for (int j = 0; j < Lanes<V>::N; ++j) {
        const Wide<V> g0 = mul(ga[i].x[j], rr), g1 = mul(gb[i].x[j], rr);
        dwa[i].x[j] = fma(g0, xa[i].x[j], dwa[i].x[j]);
        dwb[i].x[j] = fma(g1, xb[i].x[j], dwb[i].x[j]);
        A.x[j] = fma(g0, A.x[j], mul(xa[i].x[j], kk));
        B.x[j] = fma(g1, B.x[j], mul(xb[i].x[j], kk));
      }
      A.get(f);
      B.get(g);
      store_pairs<T, V, ADJ>(py, a.ys[z][3], e0[i], e1[i], a.D, now && has[i], f, g);
    }
    at.h0 += hp;
    py += sy;
    if (at.h0 >= H) {
      at.h0 = 0;
      at.tok += step;
      if (at.tok < a.tokens) place_out();
    }
  }
  if constexpr (V > 1) copy_async_wait<0>();
  if (!a.partial) return;
  // lanes with the same slots in a warp, then the warps (in the rows' place)
  __syncthreads();
  float* red = w + 2 * row;  // [warps][2 * row]
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    float f[V], g[V];
    dwa[i].get(f);
    dwb[i].get(g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float s0 = f[j], s1 = g[j];
      for (int o = lanes; o < 32; o <<= 1) {
        s0 += __shfl_xor_sync(0xffffffffu, s0, o);
        s1 += __shfl_xor_sync(0xffffffffu, s1, o);
      }
      if (lane < lanes && has[i]) {
        red[warp * 2 * row + (p0 + 32 * i) * V + j] = s0;
        red[warp * 2 * row + row + (p0 + 32 * i) * V + j] = s1;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * row; i += kRotThreads) {
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kRotWarps; ++k) sum += red[k * 2 * row + i];
    const int second = i >= row, f = i - second * row;
    int e[2];
    pair_elems(a, f / V, f % V, V, &e[0], &e[1]);
    const int el = e[second];
    if (el < a.D) a.partial[(i64)blockIdx.x * a.D + el] = sum;
  }
}

// dw[tensor][e] = sum of the CTAs' partial sums, in CTA order within each of 32 strands.
template <class T>
__global__ void __launch_bounds__(1024) rotary_weight_grad_kernel(const float* partial, int ctas_q, int ctas_k, int D, void* dw_q,
                                                                   void* dw_k, bool w32) {
  __shared__ float red[32][33];
  void* dw = blockIdx.y ? dw_k : dw_q;
  if (!dw) return;
  const int e = blockIdx.x * 32 + threadIdx.x;
  const int lo = blockIdx.y ? ctas_q : 0, hi = blockIdx.y ? ctas_q + ctas_k : ctas_q;
  float s = 0.0f;
  if (e < D)
    for (int i = lo + (int)threadIdx.y; i < hi; i += 32) s += partial[(i64)i * D + e];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && e < D) {
    float sum = 0.0f;
    for (int i = 0; i < 32; ++i) sum += red[i][threadIdx.x];
    if (w32) static_cast<float*>(dw)[e] = sum;
    else static_cast<T*>(dw)[e] = from_f32<T>(sum);
  }
}

// ------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------
static int check_rotary(const char* name, const TwgRotaryDesc* d) {
  TWG_REQUIRE(d != nullptr, "%s: descriptor is null", name);
  TWG_REQUIRE(float_size(d->dtype) != 0, "%s: element type %d is not float32, float16 or bfloat16", name, d->dtype);
  TWG_REQUIRE(d->weight_dtype == d->dtype || d->weight_dtype == TWG_DTYPE_F32,
              "%s: weights must be float32 or of the type of q and k", name);
  TWG_REQUIRE(d->position_dtype == TWG_DTYPE_I32 || d->position_dtype == TWG_DTYPE_I64, "%s: positions must be int32 or int64", name);
  TWG_REQUIRE(d->freq_dtype == TWG_DTYPE_F32 || d->freq_dtype == TWG_DTYPE_F64, "%s: inverse frequencies must be float32 or float64", name);
  TWG_REQUIRE(d->head_dim >= 2 && d->head_dim <= kRotMaxDim, "%s: head_dim %d is outside 2..%d", name, d->head_dim, kRotMaxDim);
  TWG_REQUIRE(d->rot_dim >= 2 && d->rot_dim <= d->head_dim && d->rot_dim % 2 == 0,
              "%s: rot_dim %d must be even and within 2..head_dim (%d)", name, d->rot_dim, d->head_dim);
  TWG_REQUIRE(d->axes >= 1 && d->axes <= kRotMaxAxes, "%s: %d axes; 1..%d are supported", name, d->axes, kRotMaxAxes);
  for (int j = 0; j < d->rot_dim / 2; ++j)
    TWG_REQUIRE(d->axis_of[j] < d->axes, "%s: frequency %d belongs to axis %d of %d", name, j, (int)d->axis_of[j], d->axes);
  TWG_REQUIRE(d->batch >= 0 && d->seq >= 0, "%s: negative batch or sequence length", name);
  TWG_REQUIRE(d->batch == 0 || d->seq <= ((int64_t(1) << 31) - 1) / d->batch, "%s: more than 2^31 - 1 tokens", name);
  for (int t = 0; t < 2; ++t)
    TWG_REQUIRE(d->heads[t] >= 0 && d->heads[t] <= 65536, "%s: %lld heads; at most 65536 are supported", name, (long long)d->heads[t]);
  TWG_REQUIRE(d->eps >= 0.0f, "%s: eps must not be negative", name);
  return TWG_OK;
}

// Fills everything but the pointers.
static void fill_rotary(const TwgRotaryDesc* d, RotaryArgs* a) {
  memset(a, 0, sizeof(*a));
  memcpy(a->xs, d->in_strides, sizeof(a->xs));
  memcpy(a->ys, d->out_strides, sizeof(a->ys));
  memcpy(a->gs, d->grad_strides, sizeof(a->gs));
  memcpy(a->ps, d->position_strides, sizeof(a->ps));
  memcpy(a->axis_of, d->axis_of, sizeof(a->axis_of));
  for (int t = 0; t < 2; ++t) a->heads[t] = (int)d->heads[t];
  a->seq = (u32)d->seq;
  a->tokens = (u32)(d->batch * d->seq);
  a->D = d->head_dim;
  a->R = d->rot_dim;
  a->eps = d->eps;
  a->pos64 = d->position_dtype == TWG_DTYPE_I64;
  a->freq64 = d->freq_dtype == TWG_DTYPE_F64;
  a->w32 = d->weight_dtype == TWG_DTYPE_F32;
  a->adjacent = d->adjacent != 0;
}
// Elements of the widest vectors in which every row can be read and written, with both partners of
// their pairs in one lane: 16 bytes, or 8 or 4 where sizes, strides or addresses ask for it; 1: none.
static int vector_width(const TwgRotaryDesc* d, const RotaryArgs& a, bool grad) {
  const int size = float_size(d->dtype);
  const int64_t extent[2] = {d->batch, d->seq};
  for (int V = 16 / size; V >= 2; V /= 2) {
    bool ok = a.D % (2 * V) == 0 && a.D / (2 * V) <= 32 && (a.adjacent || (a.R / 2) % V == 0);
    for (int t = 0; t < 2 && ok; ++t) {
      if (a.heads[t] == 0) continue;
      for (int k = 0; k < 3; ++k) {
        if ((k < 2 ? extent[k] : d->heads[t]) <= 1) continue;
        ok = ok && a.xs[t][k] % V == 0 && a.ys[t][k] % V == 0 && (!grad || a.gs[t][k] % V == 0);
      }
      ok = ok && a.xs[t][3] == 1 && a.ys[t][3] == 1 && (!grad || a.gs[t][3] == 1);
      ok = ok && is_aligned(a.x[t], V * size) && is_aligned(a.y[t], V * size) && (!grad || is_aligned(a.g[t], V * size));
    }
    if (ok) return V;
  }
  return 1;
}
// Slots of a row and lanes of its group.
static void set_slots(RotaryArgs* a, int V) {
  a->slots = V == 1 ? (a->D + 1) / 2 : a->D / (2 * V);
  a->lanes = 1;
  while (a->lanes < a->slots && a->lanes < 32) a->lanes *= 2;
}
static int slots_per_lane(const RotaryArgs& a) {
  int ns = 1;
  while (ns * 32 < a.slots) ns *= 2;
  return ns;
}

// Kernels whose lane groups are known when they are compiled, for the sizes of heads of 33 to 256
// elements: without them every sum over a head tests which of five exchanges it takes part in.
template <bool WIDE, class Fn>
static void by_lanes(int lanes, Fn&& fn) {
  if constexpr (WIDE) {
    if (lanes == 4) return fn(std::integral_constant<int, 4>());
    if (lanes == 8) return fn(std::integral_constant<int, 8>());
    if (lanes == 16) return fn(std::integral_constant<int, 16>());
  }
  fn(std::integral_constant<int, 0>());
}

template <class T, int V, int NS, bool ADJ>
static int launch_forward(RotaryArgs& a, bool norm, cudaStream_t s) {
  set_slots(&a, V);
  // without a sum over the head a group may have as many lanes as slots: three rows of ten slots to a warp
  if (!norm && V > 1) a.lanes = a.slots;
  const int H = a.heads[0] + a.heads[1], row = a.slots * V;
  const int groups = 32 / a.lanes;
  // rows per warp: what leaves 40 warps to an SM, between one round of the lane groups and kRotRounds
  const int64_t rows = (int64_t)a.tokens * H;
  const int want = (int)std::min<int64_t>(std::max<int64_t>(rows / (sm_count() * 40), groups), kRotRounds * groups);
  a.tile = std::max(1, std::min(std::min(want / H, kRotMaxTile), kRotTable / row));
  a.parts = (H + want - 1) / want;
  a.head_span = (H + a.parts - 1) / a.parts;
  a.parts = (H + a.head_span - 1) / a.head_span;
  const int64_t units = ((int64_t)a.tokens + a.tile - 1) / a.tile * a.parts, grid = (units + kRotWarps - 1) / kRotWarps;
  TWG_REQUIRE(units + kRotWarps < (int64_t(1) << 32), "too many rows: %lld tokens of %d heads", (long long)a.tokens, H);
  const size_t smem = sizeof(float) * (size_t)row * (2 * a.tile * kRotWarps + (norm ? 4 : 0));
  auto launch = [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value;
    if (norm) rotary_kernel<T, V, NS, true, ADJ, LANES><<<(unsigned)grid, kRotThreads, smem, s>>>(a);
    else rotary_kernel<T, V, NS, false, ADJ, LANES><<<(unsigned)grid, kRotThreads, smem, s>>>(a);
  };
  by_lanes<V == kVecOf<T>>(a.lanes, launch);
  TWG_CHECK_LAUNCH();
  g_last_path = V == 1 ? kPathStrided64 : kPathDense;
  return TWG_OK;
}
template <class T>
static int forward(RotaryArgs& a, int V, bool norm, cudaStream_t s) {
  auto wide = [&](auto v) {
    constexpr int W = decltype(v)::value;
    return a.adjacent ? launch_forward<T, W, 1, true>(a, norm, s) : launch_forward<T, W, 1, false>(a, norm, s);
  };
  if (V == 2) return wide(std::integral_constant<int, 2>());
  if (V == 4) return wide(std::integral_constant<int, 4>());
  if constexpr (kVecOf<T> == 8) {
    if (V == 8) return wide(std::integral_constant<int, 8>());
  }
  set_slots(&a, 1);
  switch (slots_per_lane(a)) {
    case 1: return launch_forward<T, 1, 1, false>(a, norm, s);
    case 2: return launch_forward<T, 1, 2, false>(a, norm, s);
    case 4: return launch_forward<T, 1, 4, false>(a, norm, s);
    default: return launch_forward<T, 1, 8, false>(a, norm, s);
  }
}

static int run_forward(const char* name, const TwgRotaryDesc* d, const void* q, const void* k, const void* qw, const void* kw,
                       bool norm, const void* positions, const void* inv_freq, void* q_out, void* k_out, void* stream) {
  g_last_path = kPathNone;
  if (int rc = check_rotary(name, d)) return rc;
  RotaryArgs a;
  fill_rotary(d, &a);
  if (a.tokens == 0 || a.heads[0] + a.heads[1] == 0) return TWG_OK;
  TWG_REQUIRE(positions && inv_freq, "%s: positions or inv_freq is null", name);
  TWG_REQUIRE(a.heads[0] == 0 || (q && q_out), "%s: q or its output is null", name);
  TWG_REQUIRE(a.heads[1] == 0 || (k && k_out), "%s: k or its output is null", name);
  const size_t e = (size_t)float_size(d->dtype);
  TWG_REQUIRE(is_aligned(q, e) && is_aligned(k, e) && is_aligned(q_out, e) && is_aligned(k_out, e),
              "%s: a tensor is not aligned to its elements", name);
  a.x[0] = q; a.x[1] = k; a.y[0] = q_out; a.y[1] = k_out;
  a.w[0] = qw; a.w[1] = kw;
  a.pos = positions;
  a.freq = inv_freq;
  a.sign = d->inverse ? -1.0f : 1.0f;
  const int V = vector_width(d, a, false);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dispatch_float(d->dtype, [&](auto* t) { return forward<std::remove_pointer_t<decltype(t)>>(a, V, norm, s); });
}

// CTAs of q and of k in the gradient kernel, in proportion to what a token of each takes: its rounds, and
// the addresses of a new token, which cost about kRotTokenCost rounds.  (Shares by rows alone left a tensor
// of few heads, with a new token in every round, working for longer than the other: 124 us in place of
// 91 for 16384 tokens of 32 + 4 heads of 128.)  A function of the sizes alone, so that the workspace
// can be sized without a device.
constexpr double kRotTokenCost = 2.0;
static void grad_ctas(const TwgRotaryDesc* d, int* cq, int* ck) {
  const int64_t tokens = d->batch * d->seq;
  *cq = *ck = 0;
  if (tokens == 0) return;
  int groups = 32;
  while (groups > 1 && 32 / groups * 32 < d->head_dim * float_size(d->dtype)) groups /= 2;
  double cost[2] = {};
  for (int t = 0; t < 2; ++t) {
    int hp = 1;
    while (hp < d->heads[t] && hp < groups) hp *= 2;
    if (d->heads[t]) cost[t] = ((double)((d->heads[t] + hp - 1) / hp) + kRotTokenCost) * hp / groups;
  }
  if (cost[0] + cost[1] == 0.0) return;
  int share = (int)(kRotGradCtas * cost[0] / (cost[0] + cost[1]) + 0.5);
  if (cost[0] > 0.0 && cost[1] > 0.0) share = std::min(std::max(share, 1), kRotGradCtas - 1);
  const int64_t most = (tokens + kRotWarps - 1) / kRotWarps;  // a token to every warp
  if (cost[0] > 0.0) *cq = (int)std::min<int64_t>(share, most);
  if (cost[1] > 0.0) *ck = (int)std::min<int64_t>(kRotGradCtas - share, most);
}

// The workspace: the CTAs' partial sums, then (on a 256-byte boundary) the tables.
static size_t grad_table_offset(const TwgRotaryDesc* d) {
  int cq, ck;
  grad_ctas(d, &cq, &ck);
  return (std::max<size_t>(256, sizeof(float) * (size_t)(cq + ck) * (size_t)d->head_dim) + 255) / 256 * 256;
}

template <class T, int V, int NS, bool ADJ>
static int launch_grad(RotaryArgs& a, float* table, cudaStream_t s) {
  set_slots(&a, V);
  const int row = a.slots * V;
  for (int t = 0; t < 2; ++t) {
    a.step[t] = 1;
    while (a.step[t] < a.heads[t] && a.step[t] < 32 / a.lanes) a.step[t] *= 2;
  }
  int wide = 32;  // threads along the frequencies, the rest of a CTA along the tokens
  while (wide < row && wide < kRotThreads) wide *= 2;
  // tokens of a thread: what leaves eight CTAs to an SM (they come one after the other)
  const int high = kRotThreads / wide;
  const int each = (int)std::min<int64_t>(std::max<int64_t>((int64_t)a.tokens * wide / ((int64_t)sm_count() * 8 * kRotThreads), 1), kRotTableTokens);
  const int per = high * each;
  rotary_table_kernel<V><<<dim3((a.tokens + per - 1) / per, (row + wide - 1) / wide), dim3(wide, high), 0, s>>>(a, table, each);
  TWG_CHECK_LAUNCH();
  a.table = table;
  const size_t smem = sizeof(float) * (size_t)row * 2 + std::max(sizeof(float) * (size_t)row * 2 * kRotWarps,
                                                                 V > 1 ? sizeof(T) * V * 4 * kRotStages * kRotThreads : (size_t)0);
  by_lanes<V == kVecOf<T>>(a.lanes, [&](auto lanes) {
    rotary_grad_kernel<T, V, NS, ADJ, decltype(lanes)::value><<<a.ctas[0] + a.ctas[1], kRotThreads, smem, s>>>(a);
  });
  TWG_CHECK_LAUNCH();
  g_last_path = V == 1 ? kPathStrided64 : kPathDense;
  return TWG_OK;
}
template <class T>
static int backward(RotaryArgs& a, int V, float* table, cudaStream_t s) {
  auto wide = [&](auto v) {
    constexpr int W = decltype(v)::value;
    return a.adjacent ? launch_grad<T, W, 1, true>(a, table, s) : launch_grad<T, W, 1, false>(a, table, s);
  };
  if (V == 2) return wide(std::integral_constant<int, 2>());
  if (V == 4) return wide(std::integral_constant<int, 4>());
  if constexpr (kVecOf<T> == 8) {
    if (V == 8) return wide(std::integral_constant<int, 8>());
  }
  set_slots(&a, 1);
  switch (slots_per_lane(a)) {
    case 1: return launch_grad<T, 1, 1, false>(a, table, s);
    case 2: return launch_grad<T, 1, 2, false>(a, table, s);
    case 4: return launch_grad<T, 1, 4, false>(a, table, s);
    default: return launch_grad<T, 1, 8, false>(a, table, s);
  }
}

}  // namespace twg

using namespace twg;

extern "C" int twg_rotary(const TwgRotaryDesc* d, const void* q, const void* k, const void* positions, const void* inv_freq,
                          void* q_out, void* k_out, void* stream) {
  TWG_TRACE("twg_rotary");
  return run_forward("twg_rotary", d, q, k, nullptr, nullptr, false, positions, inv_freq, q_out, k_out, stream);
}

extern "C" int twg_qk_norm_rotary(const TwgRotaryDesc* d, const void* q, const void* k, const void* q_weight, const void* k_weight,
                                  const void* positions, const void* inv_freq, void* q_out, void* k_out, void* stream) {
  TWG_TRACE("twg_qk_norm_rotary");
  if (d) TWG_REQUIRE(!d->inverse, "twg_qk_norm_rotary: inverse belongs to twg_rotary");
  return run_forward("twg_qk_norm_rotary", d, q, k, q_weight, k_weight, true, positions, inv_freq, q_out, k_out, stream);
}

extern "C" size_t twg_qk_norm_rotary_workspace_bytes(const TwgRotaryDesc* d) {
  if (check_rotary("twg_qk_norm_rotary_workspace_bytes", d) != TWG_OK) return 0;
  return grad_table_offset(d) + sizeof(float) * 2 * (size_t)(d->batch * d->seq) * (size_t)((d->head_dim + 1) / 2);
}

extern "C" int twg_qk_norm_rotary_backward(const TwgRotaryDesc* d, const void* q, const void* k, const void* q_weight,
                                           const void* k_weight, const void* positions, const void* inv_freq, const void* dq_out,
                                           const void* dk_out, void* dq, void* dk, void* dq_weight, void* dk_weight,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  const char* name = "twg_qk_norm_rotary_backward";
  TWG_TRACE("twg_qk_norm_rotary_backward");
  g_last_path = kPathNone;
  if (int rc = check_rotary(name, d)) return rc;
  TWG_REQUIRE(!d->inverse, "%s: inverse belongs to twg_rotary", name);
  RotaryArgs a;
  fill_rotary(d, &a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  grad_ctas(d, &a.ctas[0], &a.ctas[1]);
  const bool any = a.ctas[0] + a.ctas[1] > 0;
  const bool sums = dq_weight || dk_weight;
  if (any) {
    TWG_REQUIRE(positions && inv_freq, "%s: positions or inv_freq is null", name);
    TWG_REQUIRE(a.heads[0] == 0 || (q && dq_out && dq), "%s: q, dq_out or dq is null", name);
    TWG_REQUIRE(a.heads[1] == 0 || (k && dk_out && dk), "%s: k, dk_out or dk is null", name);
    const size_t e = (size_t)float_size(d->dtype);
    TWG_REQUIRE(is_aligned(q, e) && is_aligned(k, e) && is_aligned(dq_out, e) && is_aligned(dk_out, e) && is_aligned(dq, e) && is_aligned(dk, e),
                "%s: a tensor is not aligned to its elements", name);
    const size_t need = twg_qk_norm_rotary_workspace_bytes(d);
    TWG_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes is smaller than the %zu needed", name,
                workspace ? workspace_bytes : (size_t)0, need);
    TWG_REQUIRE(is_aligned(workspace, 16), "%s: workspace must be 16-byte aligned", name);
    float* table = reinterpret_cast<float*>(static_cast<char*>(workspace) + grad_table_offset(d));
    a.x[0] = q; a.x[1] = k; a.g[0] = dq_out; a.g[1] = dk_out; a.y[0] = dq; a.y[1] = dk;
    a.w[0] = q_weight; a.w[1] = k_weight;
    a.pos = positions;
    a.freq = inv_freq;
    a.sign = -1.0f;
    a.partial = sums ? static_cast<float*>(workspace) : nullptr;
    const int V = vector_width(d, a, true);
    const int rc = dispatch_float(d->dtype, [&](auto* t) { return backward<std::remove_pointer_t<decltype(t)>>(a, V, table, s); });
    if (rc != TWG_OK) return rc;
  }
  if (!sums) return TWG_OK;
  const int path = g_last_path;
  const dim3 grid((a.D + 31) / 32, 2), block(32, 32);
  const float* part = static_cast<const float*>(workspace);
  const int rc = dispatch_float(d->dtype, [&](auto* t) -> int {
    rotary_weight_grad_kernel<std::remove_pointer_t<decltype(t)>><<<grid, block, 0, s>>>(part, a.ctas[0], a.ctas[1], a.D, dq_weight, dk_weight, a.w32);
    TWG_CHECK_LAUNCH();
    return TWG_OK;
  });
  g_last_path = path;
  return rc;
}
