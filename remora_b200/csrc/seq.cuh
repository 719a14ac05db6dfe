// seq.cuh — what the sequence operators (seq_norm.cu, seq_conv.cu,
// seq_scan*.cu) share: host-side checks of descriptors, the device guard, and
// a few device helpers.
#pragma once

#include <initializer_list>

#include "../../include/remora_b200_seq.h"
#include "common.cuh"

namespace remora {
namespace seq {

// Makes the context's device current and puts the caller's back.  Entered
// once the arguments are checked: a refused call makes no CUDA call.
struct DeviceGuard {
  int prev = -1;
  bool moved = false;
  int enter(RemoraB200Ctx *ctx) {
    REMORA_CUDA_TRY(cudaGetDevice(&prev));
    if (prev != ctx->device) {
      REMORA_CUDA_TRY(cudaSetDevice(ctx->device));
      moved = true;
    }
    return REMORA_OK;
  }
  ~DeviceGuard() {
    if (moved) cudaSetDevice(prev);
  }
};

inline int read_f32(const void *desc, int rank, DescView *out, const char *what) {
  REMORA_TRY(read_desc(desc, rank, out, what));
  if (reinterpret_cast<uintptr_t>(out->aligned) & 3)
    return fail(REMORA_ERR_ARG, "%s: data pointer is not aligned to its 4-byte elements", what);
  return REMORA_OK;
}

// An axis of one element has no stride to speak of: 0, whatever it says, so
// that no check of strides trips over it.
inline int64_t stride_of(const DescView &v, int d) { return v.sizes[d] > 1 ? v.strides[d] : 0; }

// As read_f32, and leaves *have false for a null descriptor.
inline int read_optional(const void *desc, int rank, DescView *out, bool *have, const char *what) {
  *have = desc != nullptr;
  return *have ? read_f32(desc, rank, out, what) : REMORA_OK;
}

inline int want_shape(const DescView &v, std::initializer_list<int64_t> sizes, const char *what) {
  int d = 0;
  for (int64_t s : sizes) {
    if (v.sizes[d] != s)
      return fail(REMORA_ERR_SHAPE, "%s: axis %d has size %lld where the other operands give %lld", what, d,
                  (long long)v.sizes[d], (long long)s);
    ++d;
  }
  return REMORA_OK;
}

inline bool same_view(const DescView &a, const DescView &b) {
  if (a.rank != b.rank || a.aligned + a.offset * 4 != b.aligned + b.offset * 4) return false;
  for (int d = 0; d < a.rank; ++d)
    if (a.sizes[d] != b.sizes[d] || (a.sizes[d] > 1 && a.strides[d] != b.strides[d])) return false;
  return true;
}

// Whether two views share a byte: whether the difference of their addresses is
// a sum of index times stride over the axes of both.  The axes, all made to
// count upwards, are tried from the largest stride down; what those below can
// still add up to leaves one or two indices to try on each of an ordinary
// view's axes.  Views so irregular that this takes long count as overlapping.
struct Overlap {
  struct Axis {
    int64_t stride, size;
  } axes[2 * (REMORA_MAX_RANK + 1)];
  int count = 0;
  int64_t rest[2 * (REMORA_MAX_RANK + 1) + 1];  // the most that axes from here on add up to
  int64_t target;
  int budget = 1 << 14;

  void add(int64_t stride, int64_t size) {
    if (size <= 1 || stride == 0) return;
    if (stride < 0) {  // from the other end
      target -= stride * (size - 1);
      stride = -stride;
    }
    for (int k = 0; k < count; ++k)
      if (axes[k].stride == stride) {
        axes[k].size += size - 1;
        return;
      }
    axes[count++] = {stride, size};
  }

  bool hits(int i, int64_t left) {
    if (left < 0 || left > rest[i]) return false;
    if (i == count || left == 0) return true;
    if (--budget < 0) return true;
    int64_t k = left / axes[i].stride;
    if (k > axes[i].size - 1) k = axes[i].size - 1;
    for (; k >= 0 && left - k * axes[i].stride <= rest[i + 1]; --k)
      if (hits(i + 1, left - k * axes[i].stride)) return true;
    return false;
  }
};

// Byte range of a view's elements.
inline void byte_range(const DescView &v, int esize, char **lo, char **hi) {
  *lo = *hi = v.aligned + v.offset * esize;
  for (int d = 0; d < v.rank; ++d) {
    const int64_t span = (v.sizes[d] - 1) * v.strides[d] * esize;
    (span < 0 ? *lo : *hi) += span;
  }
  *hi += esize;
}

inline bool may_overlap(const DescView &a, int ea, const DescView &b, int eb) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  char *alo, *ahi, *blo, *bhi;
  byte_range(a, ea, &alo, &ahi);
  byte_range(b, eb, &blo, &bhi);
  if (ahi <= blo || bhi <= alo) return false;
  Overlap o;
  o.target = (b.aligned + b.offset * eb) - (a.aligned + a.offset * ea);
  for (int d = 0; d < a.rank; ++d) o.add(a.strides[d] * ea, a.sizes[d]);
  for (int d = 0; d < b.rank; ++d) o.add(-b.strides[d] * eb, b.sizes[d]);
  o.add(1, ea);
  o.add(-1, eb);
  for (int i = 1; i < o.count; ++i)  // the largest stride first
    for (int k = i; k > 0 && o.axes[k - 1].stride < o.axes[k].stride; --k) {
      const Overlap::Axis t = o.axes[k];
      o.axes[k] = o.axes[k - 1], o.axes[k - 1] = t;
    }
  o.rest[o.count] = 0;
  for (int i = o.count - 1; i >= 0; --i) o.rest[i] = o.rest[i + 1] + o.axes[i].stride * (o.axes[i].size - 1);
  return o.hits(0, o.target);
}

// Whether two elements of a view share an address: whether two indices differ by
// steps along its axes that add up to nothing.  Not where each stride is longer
// than all that the smaller ones span; else the steps along every axis are tried
// against those along the axes of smaller strides, with the same limit as above.
inline bool overlaps_itself(const DescView &v) {
  if (v.numel() == 0) return false;
  Overlap o;  // its axes have the differences of two indices, -(size - 1) to size - 1
  for (int d = 0; d < v.rank; ++d) {
    if (v.sizes[d] <= 1) continue;
    if (v.strides[d] == 0) return true;
    const int64_t stride = v.strides[d] < 0 ? -v.strides[d] : v.strides[d];
    int k = o.count++;
    for (; k > 0 && o.axes[k - 1].stride < stride; --k) o.axes[k] = o.axes[k - 1];
    o.axes[k] = {stride, 2 * v.sizes[d] - 1};  // the largest stride first
  }
  o.rest[o.count] = 0;
  for (int i = o.count - 1; i >= 0; --i) {
    const int64_t stride = o.axes[i].stride, most = o.axes[i].size / 2, span = o.rest[i + 1] / 2;
    for (int64_t k = 1; k <= most && k * stride <= span; ++k)
      if (o.hits(i + 1, span - k * stride)) return true;
    o.rest[i] = o.rest[i + 1] + stride * 2 * most;
  }
  return false;
}

struct Named {
  const DescView *v;
  const char *name;
  int esize;
};

// An output that may be exactly this input.
struct InPlace {
  const DescView *out, *in;
};

// Refuses outputs that cannot hold a result, since elements share addresses.
inline int want_own_elements(std::initializer_list<Named> outs) {
  for (const Named &o : outs)
    if (o.v != nullptr && overlaps_itself(*o.v))
      return fail(REMORA_ERR_ARG, "%s: elements of this output share addresses", o.name);
  return REMORA_OK;
}

// Refuses outputs that overlap an input, but for those of in_place, or another
// output.
inline int want_apart(std::initializer_list<Named> outs, std::initializer_list<Named> ins,
                      std::initializer_list<InPlace> in_place = {}) {
  for (const Named &o : outs) {
    if (o.v == nullptr) continue;
    for (const Named &i : ins) {
      if (i.v == nullptr || !may_overlap(*o.v, o.esize, *i.v, i.esize)) continue;
      bool allowed = false;
      for (const InPlace &p : in_place)
        allowed |= p.out == o.v && p.in == i.v && o.esize == i.esize && same_view(*o.v, *i.v);
      if (!allowed) return fail(REMORA_ERR_ARG, "%s overlaps %s", o.name, i.name);
    }
    for (const Named &p : outs)
      if (p.v != nullptr && p.v < o.v && may_overlap(*o.v, o.esize, *p.v, p.esize))
        return fail(REMORA_ERR_ARG, "%s overlaps %s", o.name, p.name);
  }
  return REMORA_OK;
}

inline int want_scratch(const void *scratch, size_t have, size_t need, const char *what) {
  if (need == 0) return REMORA_OK;
  if (scratch == nullptr || have < need)
    return fail(REMORA_ERR_LIMIT, "%s: needs %zu bytes of scratch, got %zu", what, need, scratch ? have : (size_t)0);
  if (reinterpret_cast<uintptr_t>(scratch) & 15)
    return fail(REMORA_ERR_ARG, "%s: scratch is not 16-byte aligned", what);
  return REMORA_OK;
}

// Where reduce_rows puts column c: out[(c / inner) * outer_stride + (c % inner)
// * inner_stride], or from column `split` on tail[(c - split) * tail_stride]
// (columns whose target is null are left out).
struct Columns {
  float *out;
  int64_t inner, outer_stride, inner_stride;
  int64_t split;
  float *tail;
  int64_t tail_stride;
};

// The sum over the rows of part [rows, cols], in a fixed order.
int reduce_rows(const float *part, int64_t rows, int64_t cols, const Columns &to, cudaStream_t stream);

// More threads down a column where rows are many (592 x 2048: 4.1 us with 32, 6.6
// with 8; 64 x 20480: 8.5 with 32, 5.1 with 8).
inline bool tall(int64_t rows) { return rows > 256; }

#ifdef __CUDACC__
// 32 of those columns by a block of Y rows of 32 threads, x and y its thread.
template <int Y>
__device__ __forceinline__ void reduce_columns(const float *__restrict__ part, int64_t rows, int64_t cols,
                                               const Columns &to, int64_t block, int x, int y, float (&t)[Y][33]) {
  const int64_t c = block * 32 + x;
  float v = 0.0f;
  if (c < cols) {
    int64_t p = y;
    for (; p + 3 * Y < rows; p += 4 * Y) {
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = part[(p + k * Y) * cols + c];
      v += (w[0] + w[1]) + (w[2] + w[3]);
    }
    for (; p < rows; p += Y) v += part[p * cols + c];
  }
  t[y][x] = v;
  __syncthreads();
  if (y == 0 && c < cols) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < Y; ++k) s += t[k][x];
    if (c < to.split && to.out != nullptr)
      to.out[(c / to.inner) * to.outer_stride + (c % to.inner) * to.inner_stride] = s;
    else if (c >= to.split && to.tail != nullptr)
      to.tail[(c - to.split) * to.tail_stride] = s;
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp(v): v log2(e) in two parts, so that its rounding (|v| 2^-24) does not
// show; within ex2.approx's 2^-22.
__device__ __forceinline__ float exp_fast(float v) {
  const float t = v * 1.4426950408889634f;
  // log2(e) is the constant above plus 1.926e-8
  const float r = fmaf(v, 1.4426950408889634f, -t) + v * 1.925963033500e-08f;
  const float e = ex2(t);
  // from 2^128 on e is inf, below 2^-128 zero, and r may be inf: nothing to correct
  return fabsf(t) < 128.0f ? fmaf(e, r * 0.6931471805599453f, e) : e;
}

// 1 / (1 + exp(-v)): within (6 + |v|) 2^-24 of its value for v > -87, within
// 2^-126 below, where it becomes 0 as soon as it is no normal number.  exp_fast's
// second part would leave 8 2^-24 of it for every v, but costs a convolution 5 %
// (1 x 8192 x 4096: 47.2 and 49.5 us); without it the value at v = -80, 2e-35, is
// off by 5e-6 of itself.
__device__ __forceinline__ float sigmoid(float v) { return rcp(1.0f + ex2(v * -1.4426950408889634f)); }

// log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|) in (0, 1].  With
// s = e / (2 + e) <= 1/3, log1p(e) = 2 atanh(s) = 2 s (1 + s^2/3 + s^4/5 + ..):
// seven terms leave a relative remainder below 9^-7 / 15 = 1.4e-8.  *sig gets
// the derivative 1 / (1 + exp(-v)).
__device__ __forceinline__ float softplus(float v, float *sig) {
  const float e = exp_fast(-fabsf(v));
  const float r = rcp(1.0f + e);
  *sig = v >= 0.0f ? r : e * r;
  const float s = e * rcp(2.0f + e);
  const float q = s * s;
  float p = fmaf(q, 1.0f / 13, 1.0f / 11);
  p = fmaf(q, p, 1.0f / 9);
  p = fmaf(q, p, 1.0f / 7);
  p = fmaf(q, p, 1.0f / 5);
  p = fmaf(q, p, 1.0f / 3);
  p = fmaf(q, p, 1.0f);
  return fmaxf(v, 0.0f) + 2.0f * s * p;
}

// Two f32 in a register pair, and the instructions on both at once.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pair(float lo, float hi) {
  f2 o;
  asm("mov.b64 %0, {%1, %2};" : "=l"(o) : "f"(lo), "f"(hi));
  return o;
}
__device__ __forceinline__ f2 both(float v) { return pair(v, v); }
__device__ __forceinline__ float lo(f2 v) { return __uint_as_float((unsigned)v); }
__device__ __forceinline__ float hi(f2 v) { return __uint_as_float((unsigned)(v >> 32)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 o;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(o) : "l"(a), "l"(b));
  return o;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 o;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(o) : "l"(a), "l"(b));
  return o;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 o;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(o) : "l"(a), "l"(b), "l"(c));
  return o;
}

// The decay 2^(s a) of one step, a = A log2(e).  ex2.approx returns a little
// too little (measured on B200: 2e-8 for arguments from -0.25 to -0.004, 5e-9
// nearer to 0, 5e-8 below -0.25), which the product of a long memory's decays
// adds up; the lift of the argument halves it there.  At s = 0 it is lost and
// the decay is 1.  The sum with the lift costs nothing: it is the product's fma.
constexpr float kLift = 1.0e-8f * 1.4426950408889634f;
__device__ __forceinline__ float decay(float s, float a) { return ex2(fmaf(s, a, kLift)); }
__device__ __forceinline__ f2 decay2(f2 s, f2 a) {
  const f2 v = fma2(s, a, both(kLift));
  return pair(ex2(lo(v)), ex2(hi(v)));
}
#endif

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace seq
}  // namespace remora
