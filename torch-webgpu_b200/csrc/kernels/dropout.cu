// Dropout from a counter-based generator: out = (word(i) >= p 2^32 ? x / (1 - p) : 0) [+ residual].
//
// word(i) is word i % 4 of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", 2011) with the seed as key and (i / 4, offset) as counter, i being the
// element's place in logical row-major order.  Nothing of the mask is stored: the gradient is the
// same call on the incoming gradient, and it may see other strides than the forward pass did.
//
// Bound by HBM (4 to 12 bytes an element) with the generator close behind: ten rounds of two wide
// multiplications for four elements.  Dense operands move as 16-byte vectors, so a thread computes
// one block of four words for a float32 vector and two for a 16-bit one.
#include "twg_float.cuh"

namespace twg {

struct DropoutArgs {
  const void* x;
  const void* residual;  // null: nothing is added
  void* out;
  u64 seed, offset;
  const u64* state;  // device {seed, offset}, null: the values above
  u32 threshold;     // kept where the word is not below it
  bool drop_all;     // p rounds to 1
  float scale;
};

__device__ __forceinline__ void philox_block(u64 block, u64 seed, u64 offset, u32 (&r)[4]) {
  u32 c0 = (u32)block, c1 = (u32)(block >> 32), c2 = (u32)offset, c3 = (u32)(offset >> 32);
  u32 k0 = (u32)seed, k1 = (u32)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const u64 a = (u64)c0 * 0xD2511F53u, b = (u64)c2 * 0xCD9E8D57u;
    c0 = (u32)(b >> 32) ^ c1 ^ k0;
    c2 = (u32)(a >> 32) ^ c3 ^ k1;
    c1 = (u32)b;
    c3 = (u32)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  r[0] = c0; r[1] = c1; r[2] = c2; r[3] = c3;
}

// What does not depend on the block's number, for blocks below 2^32: the keys of ten rounds and the
// products of the first two, folded into one word for each exclusive or.  In the kernel's arguments
// they cost no instruction; worked out by every thread they were 4 of 23 instructions an element.
struct PhiloxPlan {
  u32 x[10][2];  // what words 0 and 2 of each round are combined with besides the products' halves
};
__host__ __device__ __forceinline__ PhiloxPlan make_plan(u64 seed, u64 offset) {
  PhiloxPlan p;
  u32 k0 = (u32)seed, k1 = (u32)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    p.x[i][0] = k0;
    p.x[i][1] = k1;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const u64 b = (u64)(u32)offset * 0xCD9E8D57u;      // round 0: word 2 is the offset's low word, word 1 is zero
  const u32 w0 = (u32)(b >> 32) ^ p.x[0][0], w1 = (u32)b;
  p.x[0][1] ^= (u32)(offset >> 32);
  const u64 a = (u64)w0 * 0xD2511F53u;               // round 1: word 0 is w0
  p.x[1][0] ^= w1;
  p.x[1][1] ^= (u32)(a >> 32);
  p.x[2][1] ^= (u32)a;                               // round 2: word 3
  return p;
}
__device__ __forceinline__ void philox_planned(u32 block, const PhiloxPlan& p, u32 (&r)[4]) {
  u64 a = (u64)block * 0xD2511F53u, b;
  u32 c0, c1, c2 = (u32)(a >> 32) ^ p.x[0][1], c3 = (u32)a;  // round 0
  b = (u64)c2 * 0xCD9E8D57u;
  c0 = (u32)(b >> 32) ^ p.x[1][0];                           // round 1
  c1 = (u32)b;
  c2 = c3 ^ p.x[1][1];
  a = (u64)c0 * 0xD2511F53u;
  b = (u64)c2 * 0xCD9E8D57u;
  c0 = (u32)(b >> 32) ^ c1 ^ p.x[2][0];                      // round 2
  c1 = (u32)b;
  c2 = (u32)(a >> 32) ^ p.x[2][1];
  c3 = (u32)a;
#pragma unroll
  for (int i = 3; i < 10; ++i) {
    a = (u64)c0 * 0xD2511F53u;
    b = (u64)c2 * 0xCD9E8D57u;
    c0 = (u32)(b >> 32) ^ c1 ^ p.x[i][0];
    c2 = (u32)(a >> 32) ^ c3 ^ p.x[i][1];
    c1 = (u32)b;
    c3 = (u32)a;
  }
  r[0] = c0; r[1] = c1; r[2] = c2; r[3] = c3;
}

__device__ __forceinline__ void load_state(const DropoutArgs& a, u64* seed, u64* offset) {
  *seed = a.state ? a.state[0] : a.seed;
  *offset = a.state ? a.state[1] + a.offset : a.offset;
}
// A dropped element counts as zero whatever x holds there, NaN and infinities included.  Product and
// sum are one operation with one rounding, in both kernels.
__device__ __forceinline__ float drop(const DropoutArgs& a, u32 word, float x, float residual) {
  return fmaf(word >= a.threshold && !a.drop_all ? x : 0.0f, a.scale, residual);
}

constexpr int kDropUnroll = 4;  // 16-byte vectors per thread

// Dense operands of fewer than 2^34 elements and p below 1: `vecs` whole 16-byte vectors; the last CTA
// also takes the tail of n.  STATE: seed and offset are on the device, every thread works its plan out.
template <class T, bool RES, bool STATE>
__global__ void __launch_bounds__(kBlock) dropout_dense_kernel(const __grid_constant__ DropoutArgs a, const __grid_constant__ PhiloxPlan host_plan,
                                                                i64 vecs, i64 n) {
  constexpr int V = kVecOf<T>;
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  T* out = static_cast<T*>(a.out);
  const i64 base = (i64)blockIdx.x * (kBlock * kDropUnroll) + threadIdx.x;
  uint4 rx[kDropUnroll], rr[kDropUnroll];
#pragma unroll
  for (int k = 0; k < kDropUnroll; ++k) {
    const i64 v = base + k * kBlock;
    if (v < vecs) {
      rx[k] = ld_v4(x + v * V);
      if constexpr (RES) rr[k] = ld_v4(res + v * V);
    }
  }
  PhiloxPlan own;
  if constexpr (STATE) {
    u64 seed, offset;
    load_state(a, &seed, &offset);
    own = make_plan(seed, offset);
  }
  const PhiloxPlan& plan = STATE ? own : host_plan;
#pragma unroll
  for (int k = 0; k < kDropUnroll; ++k) {
    const i64 v = base + k * kBlock;
    if (v >= vecs) break;
    float f[V], y[V];
    unpack(rx[k], f, static_cast<const T*>(nullptr));
    if constexpr (RES) unpack(rr[k], y, static_cast<const T*>(nullptr));
#pragma unroll
    for (int b = 0; b < V / 4; ++b) {
      u32 w[4];
      philox_planned((u32)v * (u32)(V / 4) + (u32)b, plan, w);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const int i = 4 * b + j;
        const Two kept(w[j] >= a.threshold ? f[i] : 0.0f, w[j + 1] >= a.threshold ? f[i + 1] : 0.0f), scale(a.scale, a.scale);
        Two r;
        if constexpr (RES) r = fma(kept, scale, Two(y[i], y[i + 1]));
        else r = mul(kept, scale);
        r.get(y[i], y[i + 1]);
      }
    }
    st_v4(out + v * V, pack(y, static_cast<const T*>(nullptr)));
  }
  const i64 tail = vecs * V;
  if (blockIdx.x == gridDim.x - 1 && tail + threadIdx.x < n) {
    const i64 i = tail + threadIdx.x;
    u32 w[4];
    philox_planned((u32)(i >> 2), plan, w);
    const u32 word = i & 2 ? (i & 1 ? w[3] : w[2]) : (i & 1 ? w[1] : w[0]);
    const float kept = word >= a.threshold ? to_f32(x[i]) : 0.0f;
    float y = kept * a.scale;
    if constexpr (RES) y = fmaf(kept, a.scale, to_f32(res[i]));
    out[i] = from_f32<T>(y);
  }
}

// Any strides, p = 1, 2^34 elements and more: a thread takes the four elements of one block, one after the
// other along dimension 0.
template <class T, bool RES, class IDX>
__global__ void __launch_bounds__(kBlock) dropout_strided_kernel(const __grid_constant__ DropoutArgs a, const __grid_constant__ StridedDesc<3, IDX> d, i64 n) {
  u64 seed, offset;
  load_state(a, &seed, &offset);
  const i64 blocks = (n + 3) / 4;
  for (i64 blk = (i64)blockIdx.x * kBlock + threadIdx.x; blk < blocks; blk += (i64)gridDim.x * kBlock) {
    u32 w[4];
    philox_block((u64)blk, seed, offset, w);
    i64 off[4][3];
    float x[4], r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (4 * blk + j >= n) break;
      linear_to_offsets<3>(d, (IDX)(4 * blk + j), off[j]);
      x[j] = to_f32(static_cast<const T*>(a.x)[off[j][1]]);
      if constexpr (RES) r[j] = to_f32(static_cast<const T*>(a.residual)[off[j][2]]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (4 * blk + j >= n) break;
      // without a residual -0: a product of -0 keeps its sign
      static_cast<T*>(a.out)[off[j][0]] = from_f32<T>(drop(a, w[j], x[j], RES ? r[j] : -0.0f));
    }
  }
}

template <class T, bool RES>
static int launch_dropout(const DropoutArgs& a, const TwgIterDesc& d, cudaStream_t s) {
  constexpr int V = kVecOf<T>;
  const int nt = RES ? 3 : 2;
  bool dense = d.ndim <= 1 && is_aligned(a.x, 16) && is_aligned(a.out, 16) && (!RES || is_aligned(a.residual, 16));
  for (int t = 0; t < nt && dense; ++t) dense = d.numel <= 1 || d.strides[t][0] == 1;
  if (dense) {
    const i64 vecs = d.numel / V, per = kBlock * kDropUnroll;
    const i64 grid = std::max<i64>(1, (vecs + per - 1) / per);
    if (d.numel < (i64(1) << 34) && !a.drop_all) {
      const PhiloxPlan plan = make_plan(a.seed, a.offset);
      if (a.state) dropout_dense_kernel<T, RES, true><<<(unsigned)grid, kBlock, 0, s>>>(a, plan, vecs, d.numel);
      else dropout_dense_kernel<T, RES, false><<<(unsigned)grid, kBlock, 0, s>>>(a, plan, vecs, d.numel);
      TWG_CHECK_LAUNCH();
      g_last_path = kPathDense;
      return TWG_OK;
    }
  }
  const unsigned grid = (unsigned)std::min<i64>((d.numel / 4 + kBlock) / kBlock, 148 * 64);
  if (fits_32bit(d, nt)) {
    StridedDesc<3, u32> sd;
    fill_strided_desc<3>(d, &sd);
    dropout_strided_kernel<T, RES, u32><<<grid, kBlock, 0, s>>>(a, sd, d.numel);
    TWG_CHECK_LAUNCH();
    g_last_path = kPathStrided32;
  } else {
    StridedDesc<3, u64> sd;
    fill_strided_desc<3>(d, &sd);
    dropout_strided_kernel<T, RES, u64><<<grid, kBlock, 0, s>>>(a, sd, d.numel);
    TWG_CHECK_LAUNCH();
    g_last_path = kPathStrided64;
  }
  return TWG_OK;
}

}  // namespace twg

using namespace twg;

extern "C" int twg_dropout(const TwgIterDesc* desc, int dtype, const void* x, const void* residual, void* out, double p,
                           uint64_t seed, uint64_t offset, const uint64_t* state, void* stream) {
  TWG_TRACE("twg_dropout");
  g_last_path = kPathNone;
  const int nt = residual ? 3 : 2;
  if (int rc = check_desc(desc, nt)) return rc;
  TWG_REQUIRE(float_size(dtype) != 0, "twg_dropout: element type %d is not float32, float16 or bfloat16", dtype);
  TWG_REQUIRE(p >= 0.0 && p <= 1.0, "twg_dropout: p = %g is not a probability", p);
  if (desc->numel == 0) return TWG_OK;
  TWG_REQUIRE(x && out, "twg_dropout: x or out is null");
  const size_t e = (size_t)float_size(dtype);
  TWG_REQUIRE(is_aligned(x, e) && is_aligned(residual, e) && is_aligned(out, e), "twg_dropout: a tensor is not aligned to its elements");
  TWG_REQUIRE(is_aligned(state, 8), "twg_dropout: state must be 8-byte aligned");
  TwgIterDesc d = *desc;
  d.ntensors = nt;
  for (int k = 0; k < d.ndim; ++k)
    TWG_REQUIRE(d.shape[k] <= 1 || d.strides[0][k] != 0, "twg_dropout: out must not be broadcast (dimension %d has stride 0)", k);
  if (int rc = twg_iter_coalesce(&d)) return rc;
  DropoutArgs a;
  a.x = x; a.residual = residual; a.out = out;
  a.seed = seed; a.offset = offset; a.state = reinterpret_cast<const u64*>(state);
  const double limit = nearbyint(p * 4294967296.0);
  a.drop_all = limit >= 4294967296.0;
  a.threshold = a.drop_all ? 0xffffffffu : (u32)limit;
  a.scale = a.drop_all ? 0.0f : (float)(1.0 / (1.0 - p));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dispatch_float(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return residual ? launch_dropout<T, true>(a, d, s) : launch_dropout<T, false>(a, d, s);
  });
}
