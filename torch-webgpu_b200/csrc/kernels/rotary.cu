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
// shuffles.  The angle is the only part that needs more than 32 bits (a position of 10^6 leaves
// 2^-4 of a turn in float32): it is formed and reduced to half turns in float64, once per token
// and frequency, and its sine and cosine wait in shared memory for every head of the token.
#include "twg_float.cuh"

namespace twg {

constexpr int kRotThreads = 256;
constexpr int kRotMaxTile = 16;        // tokens whose tables one CTA holds at a time
constexpr int kRotMaxDim = 512;
constexpr int kRotMaxAxes = 8;
constexpr int kRotGradCtas = 148 * 4;  // CTAs of the gradient kernel: one row of weight partial sums each

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
  int D, R, slots, lanes;  // lanes: lanes of a row's group (a power of two)
  int tile;                // tokens per CTA (and round)
  int head_span;           // heads per CTA (forward)
  int ctas[2];             // CTAs that work on q and on k (backward)
  float* partial;          // backward: [ctas[0] + ctas[1]][D]
  float eps;
  float sign;              // -1 rotates backwards
  bool pos64, freq64, w32, adjacent;
  u8 axis_of[TWG_ROTARY_MAX_FREQS];
};

// Where table entry / weight j of slot p lies in shared memory: quads of one j are contiguous over
// the slots, so that the 16-byte reads of a group's lanes hit different banks.
template <int V>
__device__ __forceinline__ int spot(int p, int j, int slots) {
  if constexpr (V == 1) return p;
  else return ((j >> 2) * slots + p) * 4 + (j & 3);
}
// First elements of the two vectors of slot p.
__device__ __forceinline__ void slot_elems(const RotaryArgs& a, int p, int V, int* e0, int* e1) {
  const int half = a.R >> 1;
  if (!a.adjacent && p * V < half) { *e0 = p * V; *e1 = p * V + half; }
  else { *e0 = 2 * p * V; *e1 = *e0 + V; }
}

__device__ __forceinline__ void token_place(const RotaryArgs& a, u32 tok, i64* b, i64* s) {
  const u32 q = tok / a.seq;
  *b = q;
  *s = tok - q * a.seq;
}

// Sine and cosine of every frequency for `n` tokens from `tok0`; entries beyond the rotated part
// are the identity.
template <int V>
__device__ __forceinline__ void fill_tables(const RotaryArgs& a, u32 tok0, int n, float* cosine, float* sine) {
  const int row = a.slots * V;
  for (int i = threadIdx.x; i < n * row; i += kRotThreads) {
    const int t = i / row, f = i - t * row;
    float c = 1.0f, s = 0.0f;
    if (f < (a.R >> 1)) {
      i64 b, q;
      token_place(a, tok0 + (u32)t, &b, &q);
      const i64 off = (i64)a.axis_of[f] * a.ps[0] + b * a.ps[1] + q * a.ps[2];
      const double pos = a.pos64 ? (double)static_cast<const i64*>(a.pos)[off] : (double)static_cast<const int*>(a.pos)[off];
      const double fr = a.freq64 ? static_cast<const double*>(a.freq)[f] : (double)static_cast<const float*>(a.freq)[f];
      double turns = pos * fr * 0.15915494309189533577;  // 1 / (2 pi)
      turns -= rint(turns);
      sincospif((float)(2.0 * turns), &s, &c);
      s *= a.sign;
    }
    const int at = t * row + spot<V>(f / V, f % V, a.slots);
    cosine[at] = c;
    sine[at] = s;
  }
}

// Weights of one tensor in slot order: vector 0 of every slot, then vector 1.
template <class T, int V>
__device__ __forceinline__ void fill_weights(const RotaryArgs& a, int tensor, float* w) {
  const int row = a.slots * V;
  for (int i = threadIdx.x; i < 2 * row; i += kRotThreads) {
    const int second = i >= row, f = i - second * row, p = f / V, j = f % V;
    int e[2];
    slot_elems(a, p, V, &e[0], &e[1]);
    const int el = e[second] + j;
    float v = 1.0f;
    if (a.w[tensor] && el < a.D)
      v = a.w32 ? static_cast<const float*>(a.w[tensor])[el] : to_f32(static_cast<const T*>(a.w[tensor])[el]);
    w[second * row + spot<V>(p, j, a.slots)] = v;
  }
}

template <int V>
__device__ __forceinline__ void read_row(const float* tab, int p, int slots, float (&out)[V]) {
  if constexpr (V == 1) out[0] = tab[p];
  else {
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
  uint4 a, b;
};
template <class T>
struct Raw<T, 1> {
  float a, b;
};

template <class T, int V>
__device__ __forceinline__ void load_raw(Raw<T, V>& r, const T* row, i64 sd, int e0, int e1, int D, bool on) {
  if constexpr (V == 1) {
    r.a = on ? to_f32(row[e0 * sd]) : 0.0f;
    r.b = on && e1 < D ? to_f32(row[e1 * sd]) : 0.0f;
  } else {
    r.a = r.b = make_uint4(0, 0, 0, 0);
    if (on) {
      r.a = ld_v4(row + e0);
      r.b = ld_v4(row + e1);
    }
  }
}
template <class T, int V>
__device__ __forceinline__ void to_floats(const Raw<T, V>& r, float (&u)[V], float (&v)[V]) {
  if constexpr (V == 1) { u[0] = r.a; v[0] = r.b; }
  else {
    unpack(r.a, u, static_cast<const T*>(nullptr));
    unpack(r.b, v, static_cast<const T*>(nullptr));
  }
}
template <class T, int V>
__device__ __forceinline__ void store_row(T* row, i64 sd, int e0, int e1, int D, bool on, const float (&u)[V], const float (&v)[V]) {
  if (!on) return;
  if constexpr (V == 1) {
    row[e0 * sd] = from_f32<T>(u[0]);
    if (e1 < D) row[e1 * sd] = from_f32<T>(v[0]);
  } else {
    st_v4(row + e0, pack(u, static_cast<const T*>(nullptr)));
    st_v4(row + e1, pack(v, static_cast<const T*>(nullptr)));
  }
}

template <int V, bool ADJ>
__device__ __forceinline__ void rotate(float (&u)[V], float (&v)[V], const float (&c)[V], const float (&s)[V]) {
  if constexpr (ADJ) {  // partners are neighbours within a vector
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float a = u[2 * j], b = u[2 * j + 1];
      u[2 * j] = a * c[j] - b * s[j];
      u[2 * j + 1] = b * c[j] + a * s[j];
      const float d = v[2 * j], e = v[2 * j + 1];
      v[2 * j] = d * c[V / 2 + j] - e * s[V / 2 + j];
      v[2 * j + 1] = e * c[V / 2 + j] + d * s[V / 2 + j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float a = u[j], b = v[j];
      u[j] = a * c[j] - b * s[j];
      v[j] = b * c[j] + a * s[j];
    }
  }
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Forward: a CTA takes `tile` tokens and `head_span` of their q and k heads.
template <class T, int V, int NS, bool NORM, bool ADJ>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) float smem[];
  __shared__ i64 offs[kRotMaxTile][4];  // token offsets of q, k, q_out, k_out
  const int row = a.slots * V;
  float* cosine = smem;
  float* sine = cosine + a.tile * row;
  float* w = sine + a.tile * row;  // NORM: q's weights, then k's
  const int H = a.heads[0] + a.heads[1];
  const int h0 = (int)blockIdx.y * a.head_span, span = min(a.head_span, H - h0);
  const u32 tok0 = blockIdx.x * (u32)a.tile;
  const int ntok = (int)min((u32)a.tile, a.tokens - tok0);
  fill_tables<V>(a, tok0, ntok, cosine, sine);
  if constexpr (NORM) {
    fill_weights<T, V>(a, 0, w);
    fill_weights<T, V>(a, 1, w + 2 * row);
  }
  if ((int)threadIdx.x < ntok) {
    i64 b, s;
    token_place(a, tok0 + threadIdx.x, &b, &s);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      offs[threadIdx.x][t] = b * a.xs[t][0] + s * a.xs[t][1];
      offs[threadIdx.x][2 + t] = b * a.ys[t][0] + s * a.ys[t][1];
    }
  }
  __syncthreads();

  const int groups = kRotThreads / a.lanes, group = threadIdx.x / a.lanes, p0 = threadIdx.x & (a.lanes - 1);
  const int items = ntok * span;
  int e0[NS], e1[NS];
  bool has[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    slot_elems(a, p0 + 32 * i, V, &e0[i], &e1[i]);
    has[i] = p0 + 32 * i < a.slots;
  }
  Raw<T, V> cur[NS], nxt[NS];
  auto fetch = [&](Raw<T, V>(&r)[NS], int item) {
    const bool on = item < items;
    const int t = on ? item / span : 0, h = h0 + (on ? item - t * span : 0);
    const int z = h >= a.heads[0] ? 1 : 0;
    const T* base = static_cast<const T*>(a.x[z]) + offs[t][z] + (i64)(h - (z ? a.heads[0] : 0)) * a.xs[z][2];
#pragma unroll
    for (int i = 0; i < NS; ++i) load_raw<T, V>(r[i], base, a.xs[z][3], e0[i], e1[i], a.D, on && has[i]);
  };
  fetch(cur, group);
  for (int first = 0; first < items; first += groups) {
    const int item = first + group;
    fetch(nxt, item + groups);
    const bool on = item < items;
    const int t = on ? item / span : 0, h = h0 + (on ? item - t * span : 0);
    const int z = h >= a.heads[0] ? 1 : 0;
    float u[NS][V], v[NS][V];
#pragma unroll
    for (int i = 0; i < NS; ++i) to_floats<T, V>(cur[i], u[i], v[i]);
    if constexpr (NORM) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) ss = fmaf(u[i][j], u[i][j], fmaf(v[i][j], v[i][j], ss));
      const float r = rsqrtf(group_sum(ss, a.lanes) / (float)a.D + a.eps);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        float w0[V], w1[V];
        const float* wz = w + z * 2 * row;
        const int p = has[i] ? p0 + 32 * i : 0;
        read_row<V>(wz, p, a.slots, w0);
        read_row<V>(wz + row, p, a.slots, w1);
#pragma unroll
        for (int j = 0; j < V; ++j) { u[i][j] *= r * w0[j]; v[i][j] *= r * w1[j]; }
      }
    }
    T* out = static_cast<T*>(a.y[z]) + offs[t][2 + z] + (i64)(h - (z ? a.heads[0] : 0)) * a.ys[z][2];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float c[V], s[V];
      const int p = has[i] ? p0 + 32 * i : 0;
      read_row<V>(cosine + t * row, p, a.slots, c);
      read_row<V>(sine + t * row, p, a.slots, s);
      rotate<V, ADJ>(u[i], v[i], c, s);
      store_row<T, V>(out, a.ys[z][3], e0[i], e1[i], a.D, on && has[i], u[i], v[i]);
      cur[i] = nxt[i];
    }
  }
}

// Gradient of norm and rotation.  With n = x r, r = rsqrt(mean(x^2) + eps), g = dy rotated back and
// h = g w:  dx = r h - x r^3 mean(h x),  dw = sum over rows of g n.  Both sums over the head come
// out of one round of shuffles.  A CTA walks token tiles of one tensor and keeps dw in registers
// (a lane always owns the same elements); the CTAs' sums are added in a fixed order by
// rotary_weight_grad_kernel, so the gradient does not depend on scheduling.
template <class T, int V, int NS, bool ADJ>
__global__ void __launch_bounds__(kRotThreads) rotary_grad_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) float smem[];
  __shared__ i64 offs[kRotMaxTile][3];  // token offsets of x, dy, dx
  const int row = a.slots * V;
  float* cosine = smem;
  float* sine = cosine + a.tile * row;
  float* w = sine + a.tile * row;
  float* red = w + 2 * row;  // [warps][2 * row]
  const int z = (int)blockIdx.x >= a.ctas[0] ? 1 : 0;
  const u32 mine = blockIdx.x - (z ? (u32)a.ctas[0] : 0u), stride = (u32)a.ctas[z] * (u32)a.tile;
  const int H = a.heads[z];
  fill_weights<T, V>(a, z, w);

  const int groups = kRotThreads / a.lanes, group = threadIdx.x / a.lanes, p0 = threadIdx.x & (a.lanes - 1);
  int e0[NS], e1[NS];
  bool has[NS];
  float dw0[NS][V], dw1[NS][V];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    slot_elems(a, p0 + 32 * i, V, &e0[i], &e1[i]);
    has[i] = p0 + 32 * i < a.slots;
#pragma unroll
    for (int j = 0; j < V; ++j) dw0[i][j] = dw1[i][j] = 0.0f;
  }
  for (u32 tok0 = mine * (u32)a.tile; tok0 < a.tokens; tok0 += stride) {
    const int ntok = (int)min((u32)a.tile, a.tokens - tok0);
    __syncthreads();  // the previous round's tables are no longer read
    fill_tables<V>(a, tok0, ntok, cosine, sine);
    if ((int)threadIdx.x < ntok) {
      i64 b, s;
      token_place(a, tok0 + threadIdx.x, &b, &s);
      offs[threadIdx.x][0] = b * a.xs[z][0] + s * a.xs[z][1];
      offs[threadIdx.x][1] = b * a.gs[z][0] + s * a.gs[z][1];
      offs[threadIdx.x][2] = b * a.ys[z][0] + s * a.ys[z][1];
    }
    __syncthreads();
    const int items = ntok * H;
    for (int first = 0; first < items; first += groups) {
      const int item = first + group;
      const bool on = item < items;
      const int t = on ? item / H : 0;
      const i64 h = on ? item - t * H : 0;
      const T* xp = static_cast<const T*>(a.x[z]) + offs[t][0] + h * a.xs[z][2];
      const T* gp = static_cast<const T*>(a.g[z]) + offs[t][1] + h * a.gs[z][2];
      Raw<T, V> rx[NS], rg[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        load_raw<T, V>(rx[i], xp, a.xs[z][3], e0[i], e1[i], a.D, on && has[i]);
        load_raw<T, V>(rg[i], gp, a.gs[z][3], e0[i], e1[i], a.D, on && has[i]);
      }
      float x0[NS][V], x1[NS][V], g0[NS][V], g1[NS][V];
      float ss = 0.0f, hx = 0.0f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        to_floats<T, V>(rx[i], x0[i], x1[i]);
        to_floats<T, V>(rg[i], g0[i], g1[i]);
        float c[V], s[V], w0[V], w1[V];
        const int p = has[i] ? p0 + 32 * i : 0;
        read_row<V>(cosine + t * row, p, a.slots, c);
        read_row<V>(sine + t * row, p, a.slots, s);
        rotate<V, ADJ>(g0[i], g1[i], c, s);
        read_row<V>(w, p, a.slots, w0);
        read_row<V>(w + row, p, a.slots, w1);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          ss = fmaf(x0[i][j], x0[i][j], fmaf(x1[i][j], x1[i][j], ss));
          hx = fmaf(g0[i][j] * w0[j], x0[i][j], fmaf(g1[i][j] * w1[j], x1[i][j], hx));
        }
      }
      for (int o = a.lanes >> 1; o; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        hx += __shfl_xor_sync(0xffffffffu, hx, o);
      }
      // a group without a row has r = rsqrt(eps) and zeros everywhere else: with eps = 0 that would be 0 * inf
      const float r = on ? rsqrtf(ss / (float)a.D + a.eps) : 0.0f;
      const float k = r * r * r * (hx / (float)a.D);
      T* out = static_cast<T*>(a.y[z]) + offs[t][2] + h * a.ys[z][2];
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        float w0[V], w1[V];
        const int p = has[i] ? p0 + 32 * i : 0;
        read_row<V>(w, p, a.slots, w0);
        read_row<V>(w + row, p, a.slots, w1);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          dw0[i][j] = fmaf(g0[i][j], x0[i][j] * r, dw0[i][j]);
          dw1[i][j] = fmaf(g1[i][j], x1[i][j] * r, dw1[i][j]);
          g0[i][j] = r * g0[i][j] * w0[j] - x0[i][j] * k;
          g1[i][j] = r * g1[i][j] * w1[j] - x1[i][j] * k;
        }
        store_row<T, V>(out, a.ys[z][3], e0[i], e1[i], a.D, on && has[i], g0[i], g1[i]);
      }
    }
  }
  if (!a.partial) return;
  // lanes with the same slots in a warp, then the warps
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NS; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float s0 = dw0[i][j], s1 = dw1[i][j];
      for (int o = a.lanes; o < 32; o <<= 1) {
        s0 += __shfl_xor_sync(0xffffffffu, s0, o);
        s1 += __shfl_xor_sync(0xffffffffu, s1, o);
      }
      if (lane < a.lanes && has[i]) {
        red[warp * 2 * row + (p0 + 32 * i) * V + j] = s0;
        red[warp * 2 * row + row + (p0 + 32 * i) * V + j] = s1;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * row; i += kRotThreads) {
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kRotThreads / 32; ++k) sum += red[k * 2 * row + i];
    const int second = i >= row, f = i - second * row;
    int e[2];
    slot_elems(a, f / V, V, &e[0], &e[1]);
    const int el = e[second] + f % V;
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

// Fills everything but the pointers that only one direction has; *vec says whether every row can be
// read and written as 16-byte vectors whose lanes hold both partners of their pairs.
static void fill_rotary(const TwgRotaryDesc* d, bool grad, RotaryArgs* a, bool* vec) {
  const int V = 16 / float_size(d->dtype);
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
  bool ok = a->D % (2 * V) == 0 && a->D / (2 * V) <= 32 && (a->adjacent || (a->R / 2) % V == 0);
  const int64_t size[3] = {d->batch, d->seq, 0};
  for (int t = 0; t < 2 && ok; ++t) {
    if (a->heads[t] == 0) continue;
    for (int k = 0; k < 3; ++k) {
      if ((k < 2 ? size[k] : d->heads[t]) <= 1) continue;
      ok = ok && a->xs[t][k] % V == 0 && a->ys[t][k] % V == 0 && (!grad || a->gs[t][k] % V == 0);
    }
    ok = ok && a->xs[t][3] == 1 && a->ys[t][3] == 1 && (!grad || a->gs[t][3] == 1);
  }
  *vec = ok;
}
static bool rows_aligned(const RotaryArgs& a, bool grad) {
  for (int t = 0; t < 2; ++t) {
    if (a.heads[t] == 0) continue;
    if (!is_aligned(a.x[t], 16) || !is_aligned(a.y[t], 16) || (grad && !is_aligned(a.g[t], 16))) return false;
  }
  return true;
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

template <class T, int V, int NS, bool ADJ>
static int launch_forward(RotaryArgs& a, bool norm, cudaStream_t s) {
  set_slots(&a, V);
  const int H = a.heads[0] + a.heads[1], groups = kRotThreads / a.lanes;
  // rows per CTA: enough CTAs for every SM to hold several, at most eight rounds of the groups
  const int64_t rows = (int64_t)a.tokens * H;
  const int64_t want = std::min<int64_t>(std::max<int64_t>(rows / (sm_count() * 6), groups), 8 * groups);
  if (H <= want) {
    a.head_span = H;
    a.tile = (int)std::min<int64_t>(std::max<int64_t>(want / H, 1), kRotMaxTile);
  } else {
    const int parts = (int)((H + want - 1) / want);
    a.head_span = (H + parts - 1) / parts;
    a.tile = 1;
  }
  const dim3 grid((a.tokens + a.tile - 1) / a.tile, (H + a.head_span - 1) / a.head_span);
  const size_t smem = sizeof(float) * (size_t)a.slots * V * (2 * a.tile + (norm ? 4 : 0));
  if (norm) rotary_kernel<T, V, NS, true, ADJ><<<grid, kRotThreads, smem, s>>>(a);
  else rotary_kernel<T, V, NS, false, ADJ><<<grid, kRotThreads, smem, s>>>(a);
  TWG_CHECK_LAUNCH();
  g_last_path = V == 1 ? kPathStrided64 : kPathDense;
  return TWG_OK;
}
template <class T>
static int forward(RotaryArgs& a, bool vec, bool norm, cudaStream_t s) {
  constexpr int V = kVecOf<T>;
  if (vec) return a.adjacent ? launch_forward<T, V, 1, true>(a, norm, s) : launch_forward<T, V, 1, false>(a, norm, s);
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
  bool vec;
  fill_rotary(d, false, &a, &vec);
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
  vec = vec && rows_aligned(a, false);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dispatch_float(d->dtype, [&](auto* t) { return forward<std::remove_pointer_t<decltype(t)>>(a, vec, norm, s); });
}

// CTAs of q and of k in the gradient kernel, in proportion to their rows.  A function of the sizes
// alone, so that the workspace can be sized without a device.
static void grad_ctas(const TwgRotaryDesc* d, int* cq, int* ck) {
  const int64_t tokens = d->batch * d->seq, hq = d->heads[0], hk = d->heads[1];
  *cq = *ck = 0;
  if (tokens == 0 || hq + hk == 0) return;
  const int64_t share = hq == 0 ? 0 : hk == 0 ? kRotGradCtas : std::min<int64_t>(std::max<int64_t>(kRotGradCtas * hq / (hq + hk), 1), kRotGradCtas - 1);
  if (hq) *cq = (int)std::min<int64_t>(share, tokens);
  if (hk) *ck = (int)std::min<int64_t>(kRotGradCtas - share, tokens);
}

template <class T, int V, int NS, bool ADJ>
static int launch_grad(RotaryArgs& a, cudaStream_t s) {
  set_slots(&a, V);
  const int groups = kRotThreads / a.lanes;
  // tokens per round: about four rounds of the groups, no more than an even share of the tokens
  const int h = std::max(std::max(a.heads[0], a.heads[1]), 1), c = std::max(std::max(a.ctas[0], a.ctas[1]), 1);
  a.tile = std::max(1, std::min(std::min(4 * groups / h, kRotMaxTile), (int)((a.tokens + c - 1) / c)));
  // and tables, weights and the warps' sums within 47 KB of shared memory
  constexpr int kFixedRows = 2 + 2 * (kRotThreads / 32);
  a.tile = std::max(1, std::min(a.tile, (47 * 256 / (a.slots * V) - kFixedRows) / 2));
  const size_t smem = sizeof(float) * (size_t)a.slots * V * (2 * a.tile + kFixedRows);
  rotary_grad_kernel<T, V, NS, ADJ><<<a.ctas[0] + a.ctas[1], kRotThreads, smem, s>>>(a);
  TWG_CHECK_LAUNCH();
  g_last_path = V == 1 ? kPathStrided64 : kPathDense;
  return TWG_OK;
}
template <class T>
static int backward(RotaryArgs& a, bool vec, cudaStream_t s) {
  constexpr int V = kVecOf<T>;
  if (vec) return a.adjacent ? launch_grad<T, V, 1, true>(a, s) : launch_grad<T, V, 1, false>(a, s);
  set_slots(&a, 1);
  switch (slots_per_lane(a)) {
    case 1: return launch_grad<T, 1, 1, false>(a, s);
    case 2: return launch_grad<T, 1, 2, false>(a, s);
    case 4: return launch_grad<T, 1, 4, false>(a, s);
    default: return launch_grad<T, 1, 8, false>(a, s);
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
  int cq, ck;
  grad_ctas(d, &cq, &ck);
  return std::max<size_t>(256, sizeof(float) * (size_t)(cq + ck) * (size_t)d->head_dim);
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
  bool vec;
  fill_rotary(d, true, &a, &vec);
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
    if (sums) {
      const size_t need = twg_qk_norm_rotary_workspace_bytes(d);
      TWG_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %zu bytes is smaller than the %zu needed", name,
                  workspace ? workspace_bytes : (size_t)0, need);
      TWG_REQUIRE(is_aligned(workspace, 16), "%s: workspace must be 16-byte aligned", name);
    }
    a.x[0] = q; a.x[1] = k; a.g[0] = dq_out; a.g[1] = dk_out; a.y[0] = dq; a.y[1] = dk;
    a.w[0] = q_weight; a.w[1] = k_weight;
    a.pos = positions;
    a.freq = inv_freq;
    a.sign = -1.0f;
    a.partial = sums ? static_cast<float*>(workspace) : nullptr;
    vec = vec && rows_aligned(a, true);
    const int rc = dispatch_float(d->dtype, [&](auto* t) { return backward<std::remove_pointer_t<decltype(t)>>(a, vec, s); });
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
