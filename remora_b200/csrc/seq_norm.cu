// seq_norm.cu — root-mean-square norm of the last axis with the residual's
// addition before it, an e4m3 output with scales, and its gradients.
//
//   s = x + r;  y = s * rstd * w,  rstd = 1 / sqrt(mean(s^2) + eps)
//   dx = rstd * (w dy - xh * mean(w dy xh)) + dsum,  xh = s * rstd
//   dw = sum over rows of dy * xh
//
// Everything here is bound by HBM: each element is read once into registers,
// where it stays between the row's sum and the outputs that need it.  A row is
// held by blockDim.x threads, V groups of VEC consecutive elements each: 16-byte
// accesses (VEC 4) where the row length, every row stride and every address
// allow it, else 4-byte ones.  Rows that are too long for that, or whose elements
// are not consecutive, are read again from L2.
//
// Measured on B200 over buffers past the L2's 126 MB, back to back (a copy runs at
// 6.46 TB/s): forward with a residual of 16384 x 2048 83 us, 6.5 TB/s; to e4m3 with
// a scale per 128 columns, 8192 x 4096, 78 us, 5.6 TB/s; backward of 16384 x 2048
// with the residual's gradient 94 us with the join of dw, 5.7 TB/s.  A launch by
// itself ends 5 to 15 us earlier, with the last of its output still in the L2.  Rows
// past the register kernels' backward, 4096 x 16384: 485 us, 1.7 TB/s.
#include <cuda_fp8.h>

#include <algorithm>

#include "seq.cuh"

namespace remora {
namespace seq {
namespace {

constexpr float kE4M3Max = 448.0f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: the least normal f32

enum { kPlain = 0, kQuantRow = 1, kQuantGroup = 2 };

// One operand of [rows, dim]: the leading axes (up to three) of a row index.
struct Rows {
  char *base;
  int64_t stride[3];  // in elements
  int64_t inner;
};

// Sizes of the leading axes, the slowest first, shared by all operands.
struct Lead {
  int64_t n1, n2;  // sizes of the second and third of three axes
  int one;         // all operands have one row stride (in stride[2])
};

struct NormArgs {
  Rows x, r, y, s, scales;
  const float *w;
  int64_t w_stride;
  Lead lead;
  int64_t rows, dim;
  float eps;
  int group;  // columns per scale
  int has_r, has_s;
};

__device__ __forceinline__ int64_t row_offset(const Rows &v, const Lead &l, int64_t row) {
  if (l.one) return row * v.stride[2];
  const int64_t c = row % l.n2, q = row / l.n2;
  return (q / l.n1) * v.stride[0] + (q % l.n1) * v.stride[1] + c * v.stride[2];
}

template <int VEC>
struct Pack {
  float v[VEC];
};

template <int VEC>
__device__ __forceinline__ Pack<VEC> load(const float *p) {
  Pack<VEC> o;
  if constexpr (VEC == 4) {
    const float4 q = *reinterpret_cast<const float4 *>(p);
    o.v[0] = q.x, o.v[1] = q.y, o.v[2] = q.z, o.v[3] = q.w;
  } else {
    o.v[0] = *p;
  }
  return o;
}

template <int VEC>
__device__ __forceinline__ void store(float *p, const Pack<VEC> &o) {
  if constexpr (VEC == 4)
    *reinterpret_cast<float4 *>(p) = make_float4(o.v[0], o.v[1], o.v[2], o.v[3]);
  else
    *p = o.v[0];
}

// The quotient is IEEE's: multiplied by 1 / scale instead, with two roundings, one
// value in a million, next to a tie, became its other neighbour.  Costs 4 us of
// 78 (8192 x 4096 by 128); the product corrected by two fma 84 us, divisions next
// to a tie only 90.
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t *p, const Pack<VEC> &o, float scale) {
  if constexpr (VEC == 4) {
    const float2 lo = make_float2(o.v[0] / scale, o.v[1] / scale), hi = make_float2(o.v[2] / scale, o.v[3] / scale);
    *reinterpret_cast<uint32_t *>(p) = (uint32_t)__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) |
                                       (uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16;
  } else {
    *p = __nv_cvt_float_to_fp8(o.v[0] / scale, __NV_SATFINITE, __NV_E4M3);
  }
}

// The elements c .. c + VEC-1 of a row of `dim`.  SHIFT: the row does not start at
// a 16-byte boundary, its groups of four do: the first and the last may lie
// partly outside the row, are read element by element there, and give zeros for
// what is not in it.
template <int VEC, bool SHIFT>
__device__ __forceinline__ Pack<VEC> load_in(const float *p, int c, int dim) {
  if constexpr (SHIFT) {
    if (c < 0 || c + VEC > dim) {
      Pack<VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) o.v[k] = c + k >= 0 && c + k < dim ? p[c + k] : 0.0f;
      return o;
    }
  }
  return load<VEC>(p + c);
}

// As load_in, for an operand whose row starts at a boundary of its own.
template <int VEC, bool SHIFT>
__device__ __forceinline__ Pack<VEC> load_w(const float *p, int c, int dim) {
  if constexpr (SHIFT) {
    Pack<VEC> o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.v[k] = c + k >= 0 && c + k < dim ? p[c + k] : 0.0f;
    return o;
  }
  return load<VEC>(p + c);
}

template <int VEC, bool SHIFT>
__device__ __forceinline__ void store_in(float *p, int c, int dim, const Pack<VEC> &o) {
  if constexpr (SHIFT) {
    if (c < 0 || c + VEC > dim) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (c + k >= 0 && c + k < dim) p[c + k] = o.v[k];
      return;
    }
  }
  store<VEC>(p + c, o);
}

template <int VEC, bool SHIFT>
__device__ __forceinline__ void store_e4m3_in(uint8_t *p, int c, int dim, const Pack<VEC> &o, float scale) {
  if constexpr (SHIFT) {
    if (c < 0 || c + VEC > dim) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (c + k >= 0 && c + k < dim) p[c + k] = __nv_cvt_float_to_fp8(o.v[k] / scale, __NV_SATFINITE, __NV_E4M3);
      return;
    }
  }
  store_e4m3<VEC>(p + c, o, scale);
}

// Elements of a row ahead of its first 16-byte boundary's group.
template <bool SHIFT>
__device__ __forceinline__ int shift_of(const float *row) {
  return SHIFT ? (int)(reinterpret_cast<uintptr_t>(row) >> 2) & 3 : 0;
}

// max that keeps a NaN of either side
__device__ __forceinline__ float max_nan(float a, float b) {
  float o;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(o) : "f"(a), "f"(b));
  return o;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum (or maximum) over the blockDim.x threads of a row; part holds 32 floats
// per row of the block.  Every thread of the block takes part.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, u) : v + u;
  }
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  __syncthreads();  // the previous reduction's readers are done
  if ((threadIdx.x & 31) == 0) part[threadIdx.y * 32 + (threadIdx.x >> 5)] = v;
  __syncthreads();
  float t = part[threadIdx.y * 32];
  for (int k = 1; k < warps; ++k) t = MAX ? max_nan(t, part[threadIdx.y * 32 + k]) : t + part[threadIdx.y * 32 + k];
  return t;
}

// One row per blockDim.x threads, held in registers.
template <int VEC, bool SHIFT, int V, int MODE>
__global__ void __launch_bounds__(1024) norm_kernel(const NormArgs a) {
  __shared__ float part[32 * 32];
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.rows;
  const int dim = (int)a.dim;
  const float *x = reinterpret_cast<const float *>(a.x.base) + (live ? row_offset(a.x, a.lead, row) : 0);
  const float *r = reinterpret_cast<const float *>(a.r.base) + (live && a.has_r ? row_offset(a.r, a.lead, row) : 0);
  const int shift = shift_of<SHIFT>(x);
  Pack<VEC> s[V];
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
    if (live && c < dim) {
      s[j] = load_in<VEC, SHIFT>(x, c, dim);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[j].v[k] = 0.0f;
    }
  }
  if (a.has_r) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
      if (live && c < dim) {
        const Pack<VEC> q = load_in<VEC, SHIFT>(r, c, dim);
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[j].v[k] += q.v[k];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int k = 0; k < VEC; ++k) ss = fmaf(s[j].v[k], s[j].v[k], ss);
  ss = row_reduce<false>(ss, part);
  // written behind the sum: 82 us ahead of it, 75 behind (8192 x 4096 to e4m3)
  if (a.has_s && live) {
    float *so = reinterpret_cast<float *>(a.s.base) + row_offset(a.s, a.lead, row);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
      if (c < dim) store_in<VEC, SHIFT>(so, c, dim, s[j]);
    }
  }
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
    if (c < dim) {
      const Pack<VEC> w = load_w<VEC, SHIFT>(a.w, c, dim);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        s[j].v[k] = s[j].v[k] * rstd * w.v[k];
        if (MODE == kQuantRow) amax = max_nan(amax, fabsf(s[j].v[k]));
      }
    }
  }
  if (MODE == kPlain) {
    if (!live) return;
    float *y = reinterpret_cast<float *>(a.y.base) + row_offset(a.y, a.lead, row);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
      if (c < dim) store_in<VEC, SHIFT>(y, c, dim, s[j]);
    }
    return;
  }
  uint8_t *q = reinterpret_cast<uint8_t *>(a.y.base) + (live ? row_offset(a.y, a.lead, row) : 0);
  float *sc = reinterpret_cast<float *>(a.scales.base) + (live ? row_offset(a.scales, a.lead, row) : 0);
  if (MODE == kQuantRow) {
    amax = row_reduce<true>(amax, part);
    if (!live) return;
    const float scale = max_nan(amax / kE4M3Max, kMinScale);
    if (threadIdx.x == 0) sc[0] = scale;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
      if (c < dim) store_e4m3_in<VEC, SHIFT>(q, c, dim, s[j], scale);
    }
  } else {
    // a group is group / 4 neighbouring threads of one j: 8, 16 or 32 lanes
    const int lanes = a.group / VEC;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
      float m = 0.0f;
#pragma unroll
      for (int k = 0; k < VEC; ++k) m = max_nan(m, fabsf(s[j].v[k]));
      for (int o = lanes >> 1; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float scale = max_nan(m / kE4M3Max, kMinScale);
      if (live && c < dim) {
        if ((threadIdx.x & (lanes - 1)) == 0) sc[(c / a.group) * a.scales.inner] = scale;
        store_e4m3_in<VEC, SHIFT>(q, c, dim, s[j], scale);
      }
    }
  }
}

// Rows of any length, one block each: the row is read once for the sum and
// again (from L2) for each output.  With `sum` wanted the later reads take it,
// since the residual may have been overwritten by it in place.
template <int MODE>
__global__ void __launch_bounds__(1024) norm_long_kernel(const NormArgs a) {
  __shared__ float part[32];
  const int64_t row = blockIdx.x;
  const float *x = reinterpret_cast<const float *>(a.x.base) + row_offset(a.x, a.lead, row);
  const float *r = reinterpret_cast<const float *>(a.r.base) + (a.has_r ? row_offset(a.r, a.lead, row) : 0);
  float *so = reinterpret_cast<float *>(a.s.base) + (a.has_s ? row_offset(a.s, a.lead, row) : 0);
  float ss = 0.0f;
  for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
    float v = x[c * a.x.inner];
    if (a.has_r) v += r[c * a.r.inner];
    if (a.has_s) so[c * a.s.inner] = v;
    ss = fmaf(v, v, ss);
  }
  ss = row_reduce<false>(ss, part);
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  // a thread reads back what it wrote itself: no barrier is needed
  auto value = [&](int64_t c) {
    const float v = a.has_s ? so[c * a.s.inner] : a.has_r ? x[c * a.x.inner] + r[c * a.r.inner] : x[c * a.x.inner];
    return v * rstd * a.w[c * a.w_stride];
  };
  if (MODE == kPlain) {
    float *y = reinterpret_cast<float *>(a.y.base) + row_offset(a.y, a.lead, row);
    for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) y[c * a.y.inner] = value(c);
    return;
  }
  uint8_t *q = reinterpret_cast<uint8_t *>(a.y.base) + row_offset(a.y, a.lead, row);
  float *sc = reinterpret_cast<float *>(a.scales.base) + row_offset(a.scales, a.lead, row);
  if (MODE == kQuantRow) {
    float amax = 0.0f;
    for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) amax = max_nan(amax, fabsf(value(c)));
    amax = row_reduce<true>(amax, part);
    const float scale = max_nan(amax / kE4M3Max, kMinScale);
    if (threadIdx.x == 0) sc[0] = scale;
    for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
      Pack<1> o;
      o.v[0] = value(c);
      store_e4m3<1>(q + c * a.y.inner, o, scale);
    }
  } else {
    // a warp per group; its lanes' elements were written by other threads
    __syncthreads();
    for (int64_t g = threadIdx.x >> 5; g < a.dim / a.group; g += blockDim.x >> 5) {
      float m = 0.0f;
      for (int k = threadIdx.x & 31; k < a.group; k += 32) m = max_nan(m, fabsf(value(g * a.group + k)));
#pragma unroll
      for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float scale = max_nan(m / kE4M3Max, kMinScale);
      if ((threadIdx.x & 31) == 0) sc[g * a.scales.inner] = scale;
      for (int k = threadIdx.x & 31; k < a.group; k += 32) {
        Pack<1> o;
        o.v[0] = value(g * a.group + k);
        store_e4m3<1>(q + (g * a.group + k) * a.y.inner, o, scale);
      }
    }
  }
}

struct NormBwdArgs {
  Rows s, dy, ds, dx;
  const float *w;
  int64_t w_stride;
  Lead lead;
  int64_t rows, dim;
  float eps;
  int has_ds;
  float *part;  // [gridDim.x * blockDim.y, dim] sums of dy * xh
  float *rstd;  // [rows], long rows only
};

// As norm_kernel, over several rows per thread group: each thread keeps its
// columns' part of dw in registers and writes it once.
template <int VEC, bool SHIFT, int V>
__global__ void __launch_bounds__(512) norm_bwd_kernel(const NormBwdArgs a) {
  __shared__ float part[2 * 32 * 32];
  const int dim = (int)a.dim;
  const int64_t slot = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int64_t slots = (int64_t)gridDim.x * blockDim.y;
  // the rows of a slot are a multiple of four apart: one shift for all of them
  const int shift =
      shift_of<SHIFT>(reinterpret_cast<const float *>(a.s.base) + (slot < a.rows ? row_offset(a.s, a.lead, slot) : 0));
  Pack<VEC> w[V], dw[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[j].v[k] = dw[j].v[k] = 0.0f;
    if (c < dim) w[j] = load_w<VEC, SHIFT>(a.w, c, dim);
  }
  // every thread of the block takes the same number of turns
  for (int64_t base = (int64_t)blockIdx.x * blockDim.y; base < a.rows; base += slots) {
    const int64_t row = base + threadIdx.y;
    const bool live = row < a.rows;
    const float *s = reinterpret_cast<const float *>(a.s.base) + (live ? row_offset(a.s, a.lead, row) : 0);
    const float *dy = reinterpret_cast<const float *>(a.dy.base) + (live ? row_offset(a.dy, a.lead, row) : 0);
    const float *ds =
        reinterpret_cast<const float *>(a.ds.base) + (live && a.has_ds ? row_offset(a.ds, a.lead, row) : 0);
    Pack<VEC> sv[V], gv[V], dv[V];
    float ss = 0.0f, sg = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
#pragma unroll
      for (int k = 0; k < VEC; ++k) sv[j].v[k] = gv[j].v[k] = dv[j].v[k] = 0.0f;
      if (live && c < dim) {
        sv[j] = load_in<VEC, SHIFT>(s, c, dim);
        gv[j] = load_in<VEC, SHIFT>(dy, c, dim);
        if (a.has_ds) dv[j] = load_in<VEC, SHIFT>(ds, c, dim);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        ss = fmaf(sv[j].v[k], sv[j].v[k], ss);
        sg = fmaf(gv[j].v[k] * w[j].v[k], sv[j].v[k], sg);
      }
    ss = warp_sum(ss);
    sg = warp_sum(sg);
    const int warps = blockDim.x >> 5;
    if (warps > 1) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) {
        part[(threadIdx.y * 32 + (threadIdx.x >> 5)) * 2] = ss;
        part[(threadIdx.y * 32 + (threadIdx.x >> 5)) * 2 + 1] = sg;
      }
      __syncthreads();
      ss = sg = 0.0f;
      for (int k = 0; k < warps; ++k) {
        ss += part[(threadIdx.y * 32 + k) * 2];
        sg += part[(threadIdx.y * 32 + k) * 2 + 1];
      }
    }
    const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
    const float coef = sg * rstd / (float)a.dim;  // mean(w dy xh)
    float *dx = reinterpret_cast<float *>(a.dx.base) + (live ? row_offset(a.dx, a.lead, row) : 0);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
      Pack<VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float xh = sv[j].v[k] * rstd;
        o.v[k] = fmaf(rstd, fmaf(-xh, coef, gv[j].v[k] * w[j].v[k]), dv[j].v[k]);
        dw[j].v[k] = fmaf(gv[j].v[k], xh, dw[j].v[k]);
      }
      if (live && c < dim) store_in<VEC, SHIFT>(dx, c, dim, o);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * VEC - shift;
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (c + k >= 0 && c + k < dim) a.part[slot * a.dim + c + k] = dw[j].v[k];
  }
}

// Rows of any length: dx and rstd, one block per row.
__global__ void __launch_bounds__(1024) norm_bwd_long_kernel(const NormBwdArgs a) {
  __shared__ float part[32];
  const int64_t row = blockIdx.x;
  const float *s = reinterpret_cast<const float *>(a.s.base) + row_offset(a.s, a.lead, row);
  const float *dy = reinterpret_cast<const float *>(a.dy.base) + row_offset(a.dy, a.lead, row);
  const float *ds = reinterpret_cast<const float *>(a.ds.base) + (a.has_ds ? row_offset(a.ds, a.lead, row) : 0);
  float *dx = reinterpret_cast<float *>(a.dx.base) + row_offset(a.dx, a.lead, row);
  float ss = 0.0f, sg = 0.0f;
  for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
    const float v = s[c * a.s.inner];
    ss = fmaf(v, v, ss);
    sg = fmaf(dy[c * a.dy.inner] * a.w[c * a.w_stride], v, sg);
  }
  ss = row_reduce<false>(ss, part);
  sg = row_reduce<false>(sg, part);
  const float rstd = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
  const float coef = sg * rstd / (float)a.dim;
  if (threadIdx.x == 0) a.rstd[row] = rstd;
  for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
    const float xh = s[c * a.s.inner] * rstd;
    const float d = a.has_ds ? ds[c * a.ds.inner] : 0.0f;
    dx[c * a.dx.inner] = fmaf(rstd, fmaf(-xh, coef, dy[c * a.dy.inner] * a.w[c * a.w_stride]), d);
  }
}

// Long rows' dw, read before dx may overwrite an input in place: block
// column c, part y sums rows y, y + gridDim.y, ...
__global__ void __launch_bounds__(256) norm_bwd_long_dw_kernel(const NormBwdArgs a) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.dim) return;
  float t = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float *s = reinterpret_cast<const float *>(a.s.base) + row_offset(a.s, a.lead, row);
    const float *dy = reinterpret_cast<const float *>(a.dy.base) + row_offset(a.dy, a.lead, row);
    t = fmaf(dy[c * a.dy.inner], s[c * a.s.inner] * a.rstd[row], t);
  }
  a.part[blockIdx.y * a.dim + c] = t;
}

// rstd alone, one block per row, ahead of norm_bwd_long_dw_kernel
__global__ void __launch_bounds__(1024) norm_rstd_kernel(const NormBwdArgs a) {
  __shared__ float part[32];
  const float *s = reinterpret_cast<const float *>(a.s.base) + row_offset(a.s, a.lead, blockIdx.x);
  float ss = 0.0f;
  for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) ss = fmaf(s[c * a.s.inner], s[c * a.s.inner], ss);
  ss = row_reduce<false>(ss, part);
  if (threadIdx.x == 0) a.rstd[blockIdx.x] = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
}

// Sum over the rows of part [rows, cols]: 32 columns per block, Y threads down
// each, four rows on their way per thread, joined in thread order.
template <int Y>
__global__ void __launch_bounds__(32 * Y) reduce_rows_kernel(const float *__restrict__ part, int64_t rows, int64_t cols,
                                                             const Columns to) {
  __shared__ float t[Y][33];
  reduce_columns<Y>(part, rows, cols, to, blockIdx.x, threadIdx.x, threadIdx.y, t);
}

// ------------------------------------------------------------------ host --
struct NormShape {
  int64_t rows, dim;
  Lead lead;
};

Rows rows_of(const DescView &v, int esize) {
  Rows o = {v.data(esize), {0, 0, 0}, v.strides[v.rank - 1]};
  for (int d = 0; d < v.rank - 1; ++d) o.stride[3 - (v.rank - 1) + d] = v.strides[d];
  return o;
}

NormShape shape_of(const DescView &v) {
  NormShape o = {1, v.sizes[v.rank - 1], {1, 1, 0}};
  for (int d = 0; d < v.rank - 1; ++d) o.rows *= v.sizes[d];
  if (v.rank >= 2) o.lead.n2 = std::max<int64_t>(1, v.sizes[v.rank - 2]);
  if (v.rank >= 3) o.lead.n1 = std::max<int64_t>(1, v.sizes[v.rank - 3]);
  return o;
}

// Whether the leading axes advance by one stride, that of the last of them
// with more than one row; it is then put in stride[2].
bool one_stride(const DescView &v, Rows *r) {
  int64_t unit = 0, expect = 0;
  for (int d = v.rank - 2; d >= 0; --d) {
    if (v.sizes[d] <= 1) continue;
    if (expect == 0)
      unit = v.strides[d], expect = unit * v.sizes[d];
    else if (v.strides[d] == expect)
      expect *= v.sizes[d];
    else
      return false;
    if (expect == 0) return false;
  }
  r->stride[2] = unit;
  return true;
}

// Whether a row's elements are consecutive.
bool unit_rows(const DescView &v) { return v.strides[v.rank - 1] == 1 || v.sizes[v.rank - 1] == 1; }

bool aligned_rows(const DescView &v, int esize, int vec_bytes) {
  if (reinterpret_cast<uintptr_t>(v.data(esize)) % vec_bytes) return false;
  for (int d = 0; d < v.rank - 1; ++d)
    if (v.sizes[d] > 1 && (v.strides[d] * esize) % vec_bytes) return false;
  return true;
}

// How the register kernels read rows: 16 bytes at a time where every row of
// every operand starts at such a boundary; also where the rows do not, but all
// operands' rows start equally far from one (arrays of an odd row length);
// element by element where they differ; not at all where a row's elements are
// not consecutive.  12000 x 2731 with a residual: 109 us shifted, 125 single.
enum class Access { kVector, kShifted, kSingle, kNone };

struct Operand {
  const DescView *v;  // may be null
  int esize;
};

Access access_for(int64_t dim, const DescView &w, std::initializer_list<Operand> operands) {
  bool aligned = dim % 4 == 0, alike = true;
  const DescView *first = nullptr;
  if (!unit_rows(w)) return Access::kNone;
  for (const Operand &o : operands) {
    if (o.v == nullptr) continue;
    if (!unit_rows(*o.v)) return Access::kNone;
    aligned = aligned && aligned_rows(*o.v, o.esize, 4 * o.esize);
    // in elements from a boundary, modulo four
    if (first == nullptr) first = o.v;
    alike = alike && (reinterpret_cast<uintptr_t>(o.v->data(o.esize)) / o.esize) % 4 ==
                         (reinterpret_cast<uintptr_t>(first->data(4)) / 4) % 4;
    for (int d = 0; d < o.v->rank - 1; ++d)
      alike = alike && (o.v->sizes[d] <= 1 || (o.v->strides[d] - first->strides[d]) % 4 == 0);
  }
  if (aligned && reinterpret_cast<uintptr_t>(w.data(4)) % 16 == 0) return Access::kVector;
  return alike ? Access::kShifted : Access::kSingle;
}

int check_rank(int rank) {
  if (rank < 1 || rank > 4) return fail(REMORA_ERR_RANK, "rms_norm: rank %d outside 1..4", rank);
  return REMORA_OK;
}

int same_shape(const DescView &a, const DescView &b, const char *what) {
  for (int d = 0; d < a.rank; ++d)
    if (a.sizes[d] != b.sizes[d])
      return fail(REMORA_ERR_SHAPE, "%s: axis %d has size %lld, the input %lld", what, d, (long long)b.sizes[d],
                  (long long)a.sizes[d]);
  return REMORA_OK;
}

int check_eps(const RemoraNormSpec *spec, const char *what) {
  if (spec == nullptr) return fail(REMORA_ERR_ARG, "%s: null spec", what);
  if (!(spec->eps >= 0.0f)) return fail(REMORA_ERR_ARG, "%s: eps %g is not >= 0", what, (double)spec->eps);
  return REMORA_OK;
}

// Blocks of the backward pass: its dw partials have one row per thread group.
constexpr int kBwdMaxSlots = 148 * 16;
constexpr int kLongParts = 64;
constexpr int kMaxGroups = 8;  // thread groups (rows) of one block

// Threads per row and vectors per thread of the register kernels.
struct Tiling {
  int threads, v, per_block;
  bool fits;
};

// Four vectors (or eight single elements) per thread, 64 (32) bytes of each
// operand in flight, when the rows fill the device; one, over more threads, when
// there are few rows and the call waits for the latency of a single row.  No
// more than a warp's threads leave each something to do.  Rows that are a little
// too long for shifted vectors are read by single elements.
Tiling tile_for(int64_t rows, int64_t dim, Access *access, int max_threads, int max_single) {
  Tiling t = {32, 1, 1, false};
  if (*access == Access::kNone) return t;
  if (*access == Access::kShifted && (dim + 3 + 3) / 4 > (int64_t)max_threads * 4) *access = Access::kSingle;
  const int vec = *access == Access::kSingle ? 1 : 4, max_v = vec == 4 ? 4 : max_single;
  const int64_t vecs = (dim + (*access == Access::kShifted ? 3 : 0) + vec - 1) / vec;
  int v = 1;
  if (rows >= 592)
    while (v < (vec == 4 ? 4 : 8) && vecs > 32 * v) v *= 2;
  for (; v <= max_v; v *= 2) {
    const int64_t threads = ((vecs + v - 1) / v + 31) / 32 * 32;
    if (threads > max_threads) continue;
    t.threads = (int)threads;
    t.v = v;
    t.fits = true;
    break;
  }
  t.per_block = std::max(1, kMaxGroups * 32 / t.threads);
  while (t.per_block > 1 && rows < (int64_t)t.per_block * 148) t.per_block /= 2;
  return t;
}

template <int VEC, bool SHIFT, int MODE>
int launch_norm(const NormArgs &a, const Tiling &t, cudaStream_t stream) {
  const dim3 block(t.threads, t.per_block);
  const unsigned grid = (unsigned)((a.rows + t.per_block - 1) / t.per_block);
  note_launch();
  switch (t.v) {
  case 1: norm_kernel<VEC, SHIFT, 1, MODE><<<grid, block, 0, stream>>>(a); break;
  case 2: norm_kernel<VEC, SHIFT, 2, MODE><<<grid, block, 0, stream>>>(a); break;
  case 4: norm_kernel<VEC, SHIFT, 4, MODE><<<grid, block, 0, stream>>>(a); break;
  default:
    if constexpr (VEC == 1) norm_kernel<VEC, SHIFT, 8, MODE><<<grid, block, 0, stream>>>(a);
    break;
  }
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

template <int MODE>
int launch_norm(Access access, const NormArgs &a, const Tiling &t, cudaStream_t stream) {
  if (access == Access::kVector) return launch_norm<4, false, MODE>(a, t, stream);
  if constexpr (MODE != kQuantGroup) {
    if (access == Access::kShifted) return launch_norm<4, true, MODE>(a, t, stream);
    return launch_norm<1, false, MODE>(a, t, stream);
  }
  return REMORA_OK;  // not reached: groups are vectors or go to norm_long_kernel
}

int norm_forward(RemoraB200Ctx *ctx, const RemoraNormSpec *spec, const void *x, const void *residual,
                 const RemoraMemRef1 *w, void *y, void *scales, void *sum, int rank, bool quant, cudaStream_t stream) {
  if (ctx == nullptr) return fail(REMORA_ERR_ARG, "null context");
  const char *name = quant ? "rms_norm_quant" : "rms_norm_fwd";
  REMORA_TRY(check_eps(spec, name));
  REMORA_TRY(check_rank(rank));
  DescView xv, rv, wv, yv, sv, cv;
  bool has_r = false, has_s = false;
  REMORA_TRY(read_f32(x, rank, &xv, "rms_norm x"));
  REMORA_TRY(read_optional(residual, rank, &rv, &has_r, "rms_norm residual"));
  REMORA_TRY(read_f32(w, 1, &wv, "rms_norm w"));
  REMORA_TRY(quant ? read_desc(y, rank, &yv, "rms_norm q") : read_f32(y, rank, &yv, "rms_norm y"));
  REMORA_TRY(read_optional(sum, rank, &sv, &has_s, "rms_norm sum"));
  REMORA_TRY(same_shape(xv, yv, quant ? "rms_norm q" : "rms_norm y"));
  if (has_r) REMORA_TRY(same_shape(xv, rv, "rms_norm residual"));
  if (has_s) REMORA_TRY(same_shape(xv, sv, "rms_norm sum"));
  if (has_s && !has_r) return fail(REMORA_ERR_ARG, "%s: sum is the input itself without a residual", name);
  const NormShape sh = shape_of(xv);
  if (sh.dim < 1) return fail(REMORA_ERR_SHAPE, "%s: the normalised axis is empty", name);
  REMORA_TRY(want_shape(wv, {sh.dim}, "rms_norm w"));
  int64_t group = sh.dim;
  if (quant) {
    if (spec->group != 0) {
      if (spec->group != 32 && spec->group != 64 && spec->group != 128)
        return fail(REMORA_ERR_UNSUPPORTED, "%s: group %d (0, 32, 64 or 128)", name, spec->group);
      if (sh.dim % spec->group)
        return fail(REMORA_ERR_SHAPE, "%s: rows of %lld are not groups of %d", name, (long long)sh.dim, spec->group);
      group = spec->group;
    }
    REMORA_TRY(read_f32(scales, rank, &cv, "rms_norm scales"));
    for (int d = 0; d < rank; ++d) {
      const int64_t expect = d == rank - 1 ? sh.dim / group : xv.sizes[d];
      if (cv.sizes[d] != expect)
        return fail(REMORA_ERR_SHAPE, "rms_norm scales: axis %d has size %lld, expected %lld", d,
                    (long long)cv.sizes[d], (long long)expect);
    }
  }
  if (sh.rows == 0) return REMORA_OK;
  if (sh.rows > 0x7fffffff) return fail(REMORA_ERR_LIMIT, "%s: more than 2^31 - 1 rows", name);
  const DescView *rp = has_r ? &rv : nullptr, *sp = has_s ? &sv : nullptr, *cp = quant ? &cv : nullptr;
  REMORA_TRY(want_apart({{&yv, "the output", quant ? 1 : 4}, {sp, "sum", 4}, {cp, "scales", 4}},
                        {{&xv, "x", 4}, {rp, "residual", 4}, {&wv, "w", 4}},
                        {{&yv, &xv}, {&yv, rp}, {sp, &xv}, {sp, rp}}));
  REMORA_TRY(want_own_elements({{&yv, "the output", 1}, {sp, "sum", 4}, {cp, "scales", 4}}));
  NormArgs a = {};
  a.x = rows_of(xv, 4);
  a.y = rows_of(yv, quant ? 1 : 4);
  a.lead = sh.lead;
  bool one = one_stride(xv, &a.x) & one_stride(yv, &a.y);
  Access access = access_for(sh.dim, wv, {{&xv, 4}, {&yv, quant ? 1 : 4}, {rp, 4}, {sp, 4}});
  if (has_r) a.r = rows_of(rv, 4), one = one_stride(rv, &a.r) && one;
  if (has_s) a.s = rows_of(sv, 4), one = one_stride(sv, &a.s) && one;
  if (quant) a.scales = rows_of(cv, 4), one = one_stride(cv, &a.scales) && one;
  if (!one) {  // back to the strides of three axes
    a.x = rows_of(xv, 4), a.y = rows_of(yv, quant ? 1 : 4);
    if (has_r) a.r = rows_of(rv, 4);
    if (has_s) a.s = rows_of(sv, 4);
    if (quant) a.scales = rows_of(cv, 4);
  }
  a.lead.one = one;
  a.w = reinterpret_cast<const float *>(wv.data(4));
  a.w_stride = wv.strides[0];
  a.rows = sh.rows, a.dim = sh.dim, a.eps = spec->eps, a.group = (int)std::min<int64_t>(group, 1 << 30);
  a.has_r = has_r, a.has_s = has_s;
  const int mode = !quant ? kPlain : group == sh.dim && spec->group == 0 ? kQuantRow : kQuantGroup;
  const Tiling t = tile_for(sh.rows, sh.dim, &access, 1024, 8);
  DeviceGuard guard;
  REMORA_TRY(guard.enter(ctx));
  if (!t.fits || (mode == kQuantGroup && access != Access::kVector)) {
    const unsigned threads = (unsigned)std::min<int64_t>(1024, (sh.dim + 31) / 32 * 32);
    note_launch();
    if (mode == kPlain)
      norm_long_kernel<kPlain><<<(unsigned)sh.rows, threads, 0, stream>>>(a);
    else if (mode == kQuantRow)
      norm_long_kernel<kQuantRow><<<(unsigned)sh.rows, threads, 0, stream>>>(a);
    else
      norm_long_kernel<kQuantGroup><<<(unsigned)sh.rows, threads, 0, stream>>>(a);
    REMORA_CUDA_TRY(cudaGetLastError());
    return REMORA_OK;
  }
  if (mode == kPlain) return launch_norm<kPlain>(access, a, t, stream);
  if (mode == kQuantRow) return launch_norm<kQuantRow>(access, a, t, stream);
  return launch_norm<kQuantGroup>(access, a, t, stream);
}

// The last block's thread groups past the rows write a (zero) part too.
int64_t bwd_slots(int64_t rows) {
  return std::max<int64_t>(std::min<int64_t>(rows + kMaxGroups - 1, kBwdMaxSlots), kLongParts);
}

size_t bwd_scratch(int64_t rows, int64_t dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return ((size_t)bwd_slots(rows) * dim + (size_t)rows) * 4;
}

template <int VEC, bool SHIFT>
int launch_bwd(const NormBwdArgs &a, const Tiling &t, unsigned grid, cudaStream_t stream) {
  const dim3 block(t.threads, t.per_block);
  note_launch();
  switch (t.v) {
  case 1: norm_bwd_kernel<VEC, SHIFT, 1><<<grid, block, 0, stream>>>(a); break;
  case 2: norm_bwd_kernel<VEC, SHIFT, 2><<<grid, block, 0, stream>>>(a); break;
  case 4: norm_bwd_kernel<VEC, SHIFT, 4><<<grid, block, 0, stream>>>(a); break;
  default:
    if constexpr (VEC == 1) {
      if (t.v == 8)
        norm_bwd_kernel<VEC, SHIFT, 8><<<grid, block, 0, stream>>>(a);
      else
        norm_bwd_kernel<VEC, SHIFT, 16><<<grid, block, 0, stream>>>(a);
    }
    break;
  }
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

}  // namespace

int reduce_rows(const float *part, int64_t rows, int64_t cols, const Columns &to, cudaStream_t stream) {
  if (cols == 0) return REMORA_OK;
  note_launch();
  const unsigned grid = (unsigned)((cols + 31) / 32);
  if (tall(rows))
    reduce_rows_kernel<32><<<grid, dim3(32, 32), 0, stream>>>(part, rows, cols, to);
  else
    reduce_rows_kernel<8><<<grid, dim3(32, 8), 0, stream>>>(part, rows, cols, to);
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

}  // namespace seq
}  // namespace remora

using namespace remora;
using namespace remora::seq;

extern "C" {

int remora_b200_rms_norm_fwd(RemoraB200Ctx *ctx, const RemoraNormSpec *spec, const void *x, const void *residual,
                             const RemoraMemRef1 *w, void *y, void *sum, int32_t rank, remora_stream_t stream) {
  return norm_forward(ctx, spec, x, residual, w, y, nullptr, sum, rank, false, (cudaStream_t)stream);
}

int remora_b200_rms_norm_quant(RemoraB200Ctx *ctx, const RemoraNormSpec *spec, const void *x, const void *residual,
                               const RemoraMemRef1 *w, void *q, void *scales, void *sum, int32_t rank,
                               remora_stream_t stream) {
  return norm_forward(ctx, spec, x, residual, w, q, scales, sum, rank, true, (cudaStream_t)stream);
}

int remora_b200_rms_norm_bwd_scratch(RemoraB200Ctx *ctx, int64_t rows, int64_t dim, size_t *bytes) {
  if (ctx == nullptr || bytes == nullptr) return fail(REMORA_ERR_ARG, "rms_norm_bwd_scratch: null pointer");
  if (rows < 0 || dim < 0) return fail(REMORA_ERR_ARG, "rms_norm_bwd_scratch: negative size");
  *bytes = bwd_scratch(rows, dim);
  return REMORA_OK;
}

int remora_b200_rms_norm_bwd(RemoraB200Ctx *ctx, const RemoraNormSpec *spec, const void *s, const RemoraMemRef1 *w,
                             const void *dy, const void *dsum, void *dx, RemoraMemRef1 *dw, int32_t rank,
                             void *scratch, size_t scratch_bytes, remora_stream_t stream_) {
  if (ctx == nullptr) return fail(REMORA_ERR_ARG, "null context");
  cudaStream_t stream = (cudaStream_t)stream_;
  REMORA_TRY(check_eps(spec, "rms_norm_bwd"));
  REMORA_TRY(check_rank(rank));
  DescView sv, wv, gv, dv, xv, dwv;
  bool has_ds = false;
  REMORA_TRY(read_f32(s, rank, &sv, "rms_norm_bwd s"));
  REMORA_TRY(read_f32(w, 1, &wv, "rms_norm_bwd w"));
  REMORA_TRY(read_f32(dy, rank, &gv, "rms_norm_bwd dy"));
  REMORA_TRY(read_optional(dsum, rank, &dv, &has_ds, "rms_norm_bwd dsum"));
  REMORA_TRY(read_f32(dx, rank, &xv, "rms_norm_bwd dx"));
  REMORA_TRY(read_f32(dw, 1, &dwv, "rms_norm_bwd dw"));
  REMORA_TRY(same_shape(sv, gv, "rms_norm_bwd dy"));
  REMORA_TRY(same_shape(sv, xv, "rms_norm_bwd dx"));
  if (has_ds) REMORA_TRY(same_shape(sv, dv, "rms_norm_bwd dsum"));
  const NormShape sh = shape_of(sv);
  if (sh.dim < 1) return fail(REMORA_ERR_SHAPE, "rms_norm_bwd: the normalised axis is empty");
  REMORA_TRY(want_shape(wv, {sh.dim}, "rms_norm_bwd w"));
  REMORA_TRY(want_shape(dwv, {sh.dim}, "rms_norm_bwd dw"));
  if (sh.rows > 0x7fffffff) return fail(REMORA_ERR_LIMIT, "rms_norm_bwd: more than 2^31 - 1 rows");
  const DescView *dp = has_ds ? &dv : nullptr;
  REMORA_TRY(want_apart({{&xv, "dx", 4}, {&dwv, "dw", 4}},
                        {{&sv, "s", 4}, {&wv, "w", 4}, {&gv, "dy", 4}, {dp, "dsum", 4}},
                        {{&xv, &sv}, {&xv, &gv}, {&xv, dp}}));
  REMORA_TRY(want_scratch(scratch, scratch_bytes, bwd_scratch(sh.rows, sh.dim), "rms_norm_bwd"));
  REMORA_TRY(want_own_elements({{&xv, "dx", 4}, {&dwv, "dw", 4}}));
  NormBwdArgs a = {};
  a.s = rows_of(sv, 4), a.dy = rows_of(gv, 4), a.dx = rows_of(xv, 4);
  if (has_ds) a.ds = rows_of(dv, 4);
  a.lead = sh.lead;
  NormBwdArgs b = a;
  a.lead.one = one_stride(sv, &b.s) & one_stride(gv, &b.dy) & one_stride(xv, &b.dx);
  if (has_ds) a.lead.one = one_stride(dv, &b.ds) && a.lead.one;
  if (a.lead.one) a.s = b.s, a.dy = b.dy, a.dx = b.dx, a.ds = b.ds;
  Access access = access_for(sh.dim, wv, {{&sv, 4}, {&gv, 4}, {&xv, 4}, {dp, 4}});
  if (access == Access::kShifted && !a.lead.one) access = Access::kSingle;  // a slot's rows share one shift
  a.w = reinterpret_cast<const float *>(wv.data(4)), a.w_stride = wv.strides[0];
  a.rows = sh.rows, a.dim = sh.dim, a.eps = spec->eps, a.has_ds = has_ds;
  a.part = static_cast<float *>(scratch);
  int64_t parts = 0;
  DeviceGuard guard;
  REMORA_TRY(guard.enter(ctx));
  if (sh.rows > 0) {
    const Tiling t = tile_for(sh.rows, sh.dim, &access, 512, 16);
    if (t.fits) {
      const int64_t per_sm = std::max(1, 512 / (t.threads * t.per_block));
      int64_t grid = std::min<int64_t>((sh.rows + t.per_block - 1) / t.per_block,
                                       std::min<int64_t>(ctx->sm_count * per_sm, kBwdMaxSlots / t.per_block));
      // where a slot has several rows (an SM's worth of blocks and more), they are
      // a multiple of four apart
      if (grid * t.per_block < sh.rows) grid -= grid % 4;
      parts = grid * t.per_block;
      if (access == Access::kVector)
        REMORA_TRY((launch_bwd<4, false>(a, t, (unsigned)grid, stream)));
      else if (access == Access::kShifted)
        REMORA_TRY((launch_bwd<4, true>(a, t, (unsigned)grid, stream)));
      else
        REMORA_TRY((launch_bwd<1, false>(a, t, (unsigned)grid, stream)));
    } else {
      parts = std::min<int64_t>(sh.rows, kLongParts);
      a.rstd = a.part + bwd_slots(sh.rows) * sh.dim;
      note_launch();
      norm_rstd_kernel<<<(unsigned)sh.rows, 1024, 0, stream>>>(a);
      note_launch();
      norm_bwd_long_dw_kernel<<<dim3((unsigned)((sh.dim + 255) / 256), (unsigned)parts), 256, 0, stream>>>(a);
      note_launch();
      norm_bwd_long_kernel<<<(unsigned)sh.rows, 1024, 0, stream>>>(a);
      REMORA_CUDA_TRY(cudaGetLastError());
    }
  }
  const Columns to = {reinterpret_cast<float *>(dwv.data(4)), sh.dim, 0, dwv.strides[0], sh.dim, nullptr, 0};
  return reduce_rows(a.part, parts, sh.dim, to, stream);
}

}  // extern "C"
