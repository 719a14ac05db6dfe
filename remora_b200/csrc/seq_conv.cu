// seq_conv.cu — depthwise causal convolution along time with an optional SiLU,
// its gradients, and its single-token form.
//
//   p[t] = bias + sum_k w[k] x[t - (W-1) + k],  y = p or p * sigmoid(p)
//   g = dy * dy/dp;  dx[s] = sum_k w[k] g[s + W-1 - k];  dw[k] = sum_t g[t] x[t - (W-1) + k]
//
// Two products per tap and element against 8 bytes of HBM: bound by HBM.  A
// thread walks a run of time steps of VEC channels (8-byte accesses where
// every address and stride allows it, 256 bytes per warp and row) with the last
// W rows in registers, so each row is read once but for the W-1 rows ahead of
// a run, which its neighbour in the block has just brought into L1.
//
// Measured on B200 over buffers past the L2's 126 MB, back to back (a copy runs at
// 6.46 TB/s): forward with SiLU of 8 x 2048 x 4096 88 us, 6.1 TB/s, of 1 x 8192 x
// 4096 47.5 us, 5.7 TB/s; backward of 8 x 2048 x 4096 161 us with the join of dw and
// dbias, 5.0 TB/s, where the instructions (recomputed pre-activations, 4 W products
// per element) begin to count.  Times below are of single launches, whose last
// output is still in the L2.
#include <algorithm>
#include <type_traits>

#include "seq.cuh"

namespace remora {
namespace seq {
namespace {

constexpr int kMinWidth = 2, kMaxWidth = 8;
constexpr int kLanes = 32;  // threads along the channels
constexpr int kRuns = 4;    // runs of time steps per block
// Rows that a thread loads together while it works on as many, and channels of
// a thread where rows are aligned for it.  Forward of 1 x 8192 x 4096: 47 us
// with 8 rows of 2 channels, 55 with 4 of 4, 54 with 4 of 2.  Backward of 8 x
// 2048 x 4096: 165 us with 4 of 2 at 6 blocks per SM, 180 with 2 of 4, 191 with
// 4 of 1.
constexpr int kFwdRows = 8, kBwdRows = 4;
constexpr int kVec = 2;

struct Op3 {  // [B, time, D]
  float *p;
  int64_t b, t, d;
};

Op3 op3(const DescView &v) {
  return {reinterpret_cast<float *>(v.data(4)), v.strides[0], v.strides[1], v.strides[2]};
}

struct ConvArgs {
  Op3 x, y, state, state_out;
  const float *w, *bias;
  int64_t w_d, w_k, bias_d;
  const int *lengths;
  int64_t lengths_b;
  int64_t batch, length, dim;
  int64_t blocks_d, blocks_t;  // grid: batch x blocks_t x blocks_d, flattened
  int run;                     // time steps per thread
  int silu, zero_rest;
  // backward
  Op3 dy, dx, dstate, dstate_out;
  float *part;  // [batch * blocks_t, (W + 1), dim]
};

template <int VEC>
struct Vec {
  float v[VEC];
};

template <int VEC>
__device__ __forceinline__ Vec<VEC> load(const float *p) {
  Vec<VEC> o;
  if constexpr (VEC == 4) {
    const float4 q = *reinterpret_cast<const float4 *>(p);
    o.v[0] = q.x, o.v[1] = q.y, o.v[2] = q.z, o.v[3] = q.w;
  } else if constexpr (VEC == 2) {
    const float2 q = *reinterpret_cast<const float2 *>(p);
    o.v[0] = q.x, o.v[1] = q.y;
  } else {
    o.v[0] = *p;
  }
  return o;
}

template <int VEC>
__device__ __forceinline__ void store(float *p, const Vec<VEC> &o) {
  if constexpr (VEC == 4)
    *reinterpret_cast<float4 *>(p) = make_float4(o.v[0], o.v[1], o.v[2], o.v[3]);
  else if constexpr (VEC == 2)
    *reinterpret_cast<float2 *>(p) = make_float2(o.v[0], o.v[1]);
  else
    *p = o.v[0];
}

template <int VEC>
__device__ __forceinline__ Vec<VEC> fma(const Vec<VEC> &a, const Vec<VEC> &b, const Vec<VEC> &c) {
  Vec<VEC> o;
#pragma unroll
  for (int j = 0; j < VEC; ++j) o.v[j] = fmaf(a.v[j], b.v[j], c.v[j]);
  return o;
}

template <int VEC>
__device__ __forceinline__ Vec<VEC> zero() {
  Vec<VEC> o;
#pragma unroll
  for (int k = 0; k < VEC; ++k) o.v[k] = 0.0f;
  return o;
}

__device__ __forceinline__ int64_t length_of(const int *lengths, int64_t stride, int64_t b, int64_t length) {
  if (lengths == nullptr) return length;
  const int64_t n = lengths[b * stride];
  return n < 0 ? 0 : n > length ? length : n;
}

template <int VEC>
__device__ __forceinline__ void zero_rows(const Op3 &o, int64_t b, int64_t from, int64_t to, int64_t d) {
  for (int64_t t = from; t < to; ++t) store<VEC>(o.p + b * o.b + t * o.t + d * o.d, zero<VEC>());
}

// Row e of the state followed by the sequence: e < 0 is state row e + W-1.
template <int W, int VEC>
__device__ __forceinline__ Vec<VEC> row_at(const ConvArgs &a, int64_t b, int64_t e, int64_t d) {
  if (e >= 0) return load<VEC>(a.x.p + b * a.x.b + e * a.x.t + d * a.x.d);
  if (a.state.p == nullptr) return zero<VEC>();
  return load<VEC>(a.state.p + b * a.state.b + (e + W - 1) * a.state.t + d * a.state.d);
}

template <int W, int VEC>
__global__ void __launch_bounds__(kLanes *kRuns) conv_fwd_kernel(const ConvArgs a) {
  const int64_t bd = blockIdx.x % a.blocks_d, rest = blockIdx.x / a.blocks_d;
  const int64_t bt = rest % a.blocks_t, b = rest / a.blocks_t;
  const int64_t d = (bd * kLanes + threadIdx.x) * VEC;
  if (d >= a.dim) return;
  const int64_t len = length_of(a.lengths, a.lengths_b, b, a.length);
  const int64_t t0 = (bt * kRuns + threadIdx.y) * a.run;
  if (a.zero_rest) zero_rows<VEC>(a.y, b, max(t0, len), min(t0 + a.run, a.length), d);
  if (t0 >= len && t0 > 0) return;
  const int64_t t1 = min(t0 + a.run, len);
  Vec<VEC> w[W], win[W - 1], bias = zero<VEC>();
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k].v[j] = a.w[(d + j) * a.w_d + k * a.w_k];
    if (a.bias) bias.v[j] = a.bias[(d + j) * a.bias_d];
  }
#pragma unroll
  for (int k = 0; k < W - 1; ++k) win[k] = row_at<W, VEC>(a, b, t0 - (W - 1) + k, d);
  const float *x = a.x.p + b * a.x.b + d * a.x.d + t0 * a.x.t;
  float *y = a.y.p + b * a.y.b + d * a.y.d + t0 * a.y.t;
  auto step = [&](const Vec<VEC> &now) {
    Vec<VEC> o = bias;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) o = fma(w[k], win[k], o);
    o = fma(w[W - 1], now, o);
    if (a.silu) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.v[j] *= sigmoid(o.v[j]);
    }
    store<VEC>(y, o);
    y += a.y.t;
#pragma unroll
    for (int k = 0; k + 1 < W - 1; ++k) win[k] = win[k + 1];
    win[W - 2] = now;
  };
  // the next U rows are on their way while the last U are worked on
  constexpr int U = kFwdRows;
  Vec<VEC> r[U], n[U];
  int64_t t = t0;
  if (t + U <= t1) {
#pragma unroll
    for (int k = 0; k < U; ++k) n[k] = load<VEC>(x + k * a.x.t);
  }
  for (; t + U <= t1; t += U) {
    x += U * a.x.t;
#pragma unroll
    for (int k = 0; k < U; ++k) r[k] = n[k];
    if (t + 2 * U <= t1) {
#pragma unroll
      for (int k = 0; k < U; ++k) n[k] = load<VEC>(x + k * a.x.t);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) step(r[k]);
  }
  for (; t < t1; ++t, x += a.x.t) step(load<VEC>(x));
  // The run at the sequence's start writes the state behind its end.  Row k
  // comes from row len + k, so an update in place reads ahead of its writes.
  if (t0 == 0 && a.state_out.p != nullptr) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
      store<VEC>(a.state_out.p + b * a.state_out.b + k * a.state_out.t + d * a.state_out.d,
                 row_at<W, VEC>(a, b, len - (W - 1) + k, d));
  }
}

// A run of rows s in [t0, t0 + run) of dx needs g[s .. s + W-1]: the walk goes
// W-1 steps past the run, and dw takes the steps inside it only.
template <int W, int VEC>
__global__ void __launch_bounds__(kLanes *kRuns, W <= 4 ? 6 : W <= 6 ? 4 : 3) conv_bwd_kernel(const ConvArgs a) {
  __shared__ float sum[kRuns][kLanes * VEC];
  const int64_t bd = blockIdx.x % a.blocks_d, rest = blockIdx.x / a.blocks_d;
  const int64_t bt = rest % a.blocks_t, b = rest / a.blocks_t;
  const int64_t d = (bd * kLanes + threadIdx.x) * VEC;
  const int64_t len = length_of(a.lengths, a.lengths_b, b, a.length);
  const int64_t t0 = (bt * kRuns + threadIdx.y) * a.run;
  Vec<VEC> dw[W], db = zero<VEC>();
#pragma unroll
  for (int k = 0; k < W; ++k) dw[k] = zero<VEC>();
  if (a.zero_rest && d < a.dim) zero_rows<VEC>(a.dx, b, max(t0, len), min(t0 + a.run, a.length), d);
  if (d < a.dim && (t0 < len || t0 == 0)) {
    const int64_t t1 = min(t0 + a.run, len);  // rows [t0, t1) of dx and of the sums
    Vec<VEC> w[W], win[W], g[W], bias = zero<VEC>();  // win: x rows t-(W-1) .. t; g: g[t-(W-1)] .. g[t]
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
#pragma unroll
      for (int k = 0; k < W; ++k) w[k].v[j] = a.w[(d + j) * a.w_d + k * a.w_k];
      if (a.bias) bias.v[j] = a.bias[(d + j) * a.bias_d];
    }
#pragma unroll
    for (int k = 0; k < W; ++k) g[k] = win[k] = zero<VEC>();
#pragma unroll
    for (int k = 0; k < W - 1; ++k) win[k + 1] = row_at<W, VEC>(a, b, t0 - (W - 1) + k, d);
    const float *x = a.x.p + b * a.x.b + d * a.x.d;
    const float *dy = a.dy.p + b * a.dy.b + d * a.dy.d;
    float *dxp = a.dx.p + b * a.dx.b + d * a.dx.d + (t0 - (W - 1)) * a.dx.t;  // row t - (W-1)
    // One step.  INNER: t lies in the run, W-1 steps or more behind its start;
    // otherwise the step may lie past the run's or the sequence's end, and its
    // row of dx ahead of the run, in the state or in state_out.
    auto step = [&](auto inner, int64_t t, const Vec<VEC> &xr, const Vec<VEC> &gr) {
      constexpr bool INNER = decltype(inner)::value;
#pragma unroll
      for (int k = 0; k + 1 < W; ++k) win[k] = win[k + 1], g[k] = g[k + 1];
      win[W - 1] = xr;
      Vec<VEC> now = gr, o = zero<VEC>();
      if (a.silu) {
        Vec<VEC> p = bias;
#pragma unroll
        for (int k = 0; k < W; ++k) p = fma(w[k], win[k], p);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float s = sigmoid(p.v[j]);
          now.v[j] *= s * fmaf(p.v[j], 1.0f - s, 1.0f);
        }
      }
      if (!INNER && t >= len) now = zero<VEC>();  // whatever a NaN in the window made of it
      if (INNER || t < t1) {
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k] = fma(now, win[k], dw[k]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) db.v[j] += now.v[j];
      }
      g[W - 1] = now;
      const int64_t s = t - (W - 1);
      // rows ahead of the run belong to the run before, or to the state
      if (INNER || s >= t0 || (t0 == 0 && a.dstate.p != nullptr)) {
#pragma unroll
        for (int k = 0; k < W; ++k) o = fma(w[k], g[W - 1 - k], o);
        if (!INNER && a.dstate_out.p != nullptr && t >= len) {  // this row is row t - len of state_out
          const Vec<VEC> e =
              load<VEC>(a.dstate_out.p + b * a.dstate_out.b + (t - len) * a.dstate_out.t + d * a.dstate_out.d);
#pragma unroll
          for (int j = 0; j < VEC; ++j) o.v[j] += e.v[j];
        }
        if (INNER || s >= 0)
          store<VEC>(dxp, o);
        else
          store<VEC>(a.dstate.p + b * a.dstate.b + (s + W - 1) * a.dstate.t + d * a.dstate.d, o);
      }
      dxp += a.dx.t;
    };
    using Inner = std::true_type;
    using Edge = std::false_type;
    const int64_t end = t1 + W - 1, full = min(end, len);
    int64_t t = t0;
    for (; t < min(t0 + W - 1, full); ++t) step(Edge{}, t, load<VEC>(x + t * a.x.t), load<VEC>(dy + t * a.dy.t));
    constexpr int U = kBwdRows;
    Vec<VEC> xr[U], gr[U], xn[U], gn[U];
    auto fetch = [&](int64_t at) {
#pragma unroll
      for (int k = 0; k < U; ++k) xn[k] = load<VEC>(x + (at + k) * a.x.t), gn[k] = load<VEC>(dy + (at + k) * a.dy.t);
    };
    if (t + U <= t1) fetch(t);
    for (; t + U <= t1; t += U) {
#pragma unroll
      for (int k = 0; k < U; ++k) xr[k] = xn[k], gr[k] = gn[k];
      if (t + 2 * U <= t1) fetch(t + U);
#pragma unroll
      for (int k = 0; k < U; ++k) step(Inner{}, t + k, xr[k], gr[k]);
    }
    for (; t < full; ++t) step(Edge{}, t, load<VEC>(x + t * a.x.t), load<VEC>(dy + t * a.dy.t));
    for (; t < end; ++t) step(Edge{}, t, zero<VEC>(), zero<VEC>());
  }
  // the block's runs, joined in their order
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[threadIdx.y][threadIdx.x * VEC + j] = k < W ? dw[k < W ? k : 0].v[j] : db.v[j];
    __syncthreads();
    const int i = threadIdx.y * kLanes + threadIdx.x;
    if (i < kLanes * VEC) {
      float s = 0.0f;
#pragma unroll
      for (int r = 0; r < kRuns; ++r) s += sum[r][i];
      const int64_t c = bd * kLanes * VEC + i;
      if (c < a.dim) a.part[((b * a.blocks_t + bt) * (W + 1) + k) * a.dim + c] = s;
    }
  }
}

struct StepArgs {
  Op3 state, state_out;
  const float *x;
  float *y;
  int64_t x_b, x_d, y_b, y_d;
  const float *w, *bias;
  int64_t w_d, w_k, bias_d;
  const int *slots;
  int64_t slots_b;
  int64_t rows, dim;
  int silu, zero_rest;
};

template <int W, int VEC>
__global__ void __launch_bounds__(128) conv_step_kernel(const StepArgs a) {
  const int64_t i = blockIdx.y;
  int64_t slot = i;
  bool live = true;
  if (a.slots != nullptr) {
    slot = a.slots[i * a.slots_b];
    bool again = false;
    for (int64_t k = threadIdx.x; k < i; k += blockDim.x) again |= a.slots[k * a.slots_b] == slot;
    live = !__syncthreads_or(again) && slot >= 0 && slot < a.rows;
  }
  const int64_t d = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * VEC;
  if (d >= a.dim) return;
  if (!live) {
    if (a.zero_rest) store<VEC>(a.y + i * a.y_b + d * a.y_d, zero<VEC>());
    return;
  }
  const float *s = a.state.p + slot * a.state.b + d * a.state.d;
  float *so = a.state_out.p + slot * a.state_out.b + d * a.state_out.d;
  Vec<VEC> win[W], o = zero<VEC>();
#pragma unroll
  for (int k = 0; k < W - 1; ++k) win[k] = load<VEC>(s + k * a.state.t);
  win[W - 1] = load<VEC>(a.x + i * a.x_b + d * a.x_d);
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    if (a.bias) o.v[j] = a.bias[(d + j) * a.bias_d];
#pragma unroll
    for (int k = 0; k < W; ++k) o.v[j] = fmaf(a.w[(d + j) * a.w_d + k * a.w_k], win[k].v[j], o.v[j]);
    if (a.silu) o.v[j] *= sigmoid(o.v[j]);
  }
  store<VEC>(a.y + i * a.y_b + d * a.y_d, o);
#pragma unroll
  for (int k = 0; k < W - 1; ++k) store<VEC>(so + k * a.state_out.t, win[k + 1]);
}

// ------------------------------------------------------------------ host --
// Time steps per thread, `most` at most: longer runs read fewer rows twice
// ((W-1) / run), shorter ones keep the device full when there are few rows.
// On 8 x 2048 x 4096: forward 83 us with 32 steps and 84 with 64, backward
// 165 with 32 and 152 with 64 or 128.
constexpr int kFwdRun = 32, kBwdRun = 64;

int run_for(int most, int64_t batch, int64_t length, int64_t dim, int vec) {
  int run = most;
  while (run > 8 && batch * ((length + run - 1) / run) * ((dim + vec - 1) / vec) < 148 * 1024) run /= 2;
  return run;
}

// Whether every row can be read `vec` channels at a time.
bool vec_rows(const DescView &v, int vec) {
  if (v.sizes[v.rank - 1] > 1 && v.strides[v.rank - 1] != 1) return false;
  if (reinterpret_cast<uintptr_t>(v.data(4)) % (4 * vec)) return false;
  for (int d = 0; d < v.rank - 1; ++d)
    if (v.sizes[d] > 1 && v.strides[d] % vec) return false;
  return true;
}

template <int VEC, bool BWD>
int launch_conv(int width, const ConvArgs &a, cudaStream_t stream) {
  const unsigned grid = (unsigned)(a.batch * a.blocks_t * a.blocks_d);
  const dim3 block(kLanes, kRuns);
  note_launch();
#define REMORA_CONV_CASE(W)                                    \
  case W:                                                      \
    if constexpr (BWD)                                         \
      conv_bwd_kernel<W, VEC><<<grid, block, 0, stream>>>(a);  \
    else                                                       \
      conv_fwd_kernel<W, VEC><<<grid, block, 0, stream>>>(a);  \
    break;
  switch (width) {
    REMORA_CONV_CASE(2)
    REMORA_CONV_CASE(3)
    REMORA_CONV_CASE(4)
    REMORA_CONV_CASE(5)
    REMORA_CONV_CASE(6)
    REMORA_CONV_CASE(7)
    REMORA_CONV_CASE(8)
  }
#undef REMORA_CONV_CASE
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

template <int VEC>
int launch_step(int width, int64_t batch, const StepArgs &a, cudaStream_t stream) {
  const dim3 grid((unsigned)((a.dim + 128 * VEC - 1) / (128 * VEC)), (unsigned)batch);
  note_launch();
#define REMORA_CONV_CASE(W) \
  case W: conv_step_kernel<W, VEC><<<grid, 128, 0, stream>>>(a); break;
  switch (width) {
    REMORA_CONV_CASE(2)
    REMORA_CONV_CASE(3)
    REMORA_CONV_CASE(4)
    REMORA_CONV_CASE(5)
    REMORA_CONV_CASE(6)
    REMORA_CONV_CASE(7)
    REMORA_CONV_CASE(8)
  }
#undef REMORA_CONV_CASE
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

int check_width(int64_t width, const char *what) {
  if (width < kMinWidth || width > kMaxWidth)
    return fail(REMORA_ERR_UNSUPPORTED, "%s: %lld taps (%d..%d)", what, (long long)width, kMinWidth, kMaxWidth);
  return REMORA_OK;
}

// The grid is sized for the shorter runs, so the size does not depend on the
// alignment of the operands.
int64_t bwd_parts(int64_t batch, int64_t length, int64_t dim) {
  const int run = std::min(run_for(kBwdRun, batch, length, dim, 1), run_for(kBwdRun, batch, length, dim, kVec));
  return batch * std::max<int64_t>(1, (length + (int64_t)run * kRuns - 1) / ((int64_t)run * kRuns));
}

int set_grid(ConvArgs &a, int most, int vec, const char *what) {
  a.run = run_for(most, a.batch, a.length, a.dim, vec);
  a.blocks_d = (a.dim + kLanes * vec - 1) / (kLanes * vec);
  a.blocks_t = std::max<int64_t>(1, (a.length + (int64_t)a.run * kRuns - 1) / ((int64_t)a.run * kRuns));
  if (a.batch * a.blocks_t * a.blocks_d > 0x7fffffff) return fail(REMORA_ERR_LIMIT, "%s: too many blocks", what);
  return REMORA_OK;
}

}  // namespace
}  // namespace seq
}  // namespace remora

using namespace remora;
using namespace remora::seq;

extern "C" {

int remora_b200_causal_conv_fwd(RemoraB200Ctx *ctx, const RemoraCausalConvSpec *spec, const RemoraMemRef3 *x,
                                const RemoraMemRef2 *w, const RemoraMemRef1 *bias, const RemoraMemRef3 *state,
                                const RemoraMemRef1 *lengths, RemoraMemRef3 *y, RemoraMemRef3 *state_out,
                                remora_stream_t stream) {
  if (ctx == nullptr) return fail(REMORA_ERR_ARG, "null context");
  if (spec == nullptr) return fail(REMORA_ERR_ARG, "causal_conv_fwd: null spec");
  DescView xv, wv, bv, sv, lv, yv, ov;
  bool has_b, has_s, has_l, has_o;
  REMORA_TRY(read_f32(x, 3, &xv, "causal_conv x"));
  REMORA_TRY(read_f32(w, 2, &wv, "causal_conv w"));
  REMORA_TRY(read_optional(bias, 1, &bv, &has_b, "causal_conv bias"));
  REMORA_TRY(read_optional(state, 3, &sv, &has_s, "causal_conv state"));
  REMORA_TRY(read_optional(lengths, 1, &lv, &has_l, "causal_conv lengths"));
  REMORA_TRY(read_f32(y, 3, &yv, "causal_conv y"));
  REMORA_TRY(read_optional(state_out, 3, &ov, &has_o, "causal_conv state_out"));
  const int64_t B = xv.sizes[0], L = xv.sizes[1], D = xv.sizes[2], W = wv.sizes[1];
  REMORA_TRY(check_width(W, "causal_conv_fwd"));
  REMORA_TRY(want_shape(wv, {D, W}, "causal_conv w"));
  REMORA_TRY(want_shape(yv, {B, L, D}, "causal_conv y"));
  if (has_b) REMORA_TRY(want_shape(bv, {D}, "causal_conv bias"));
  if (has_s) REMORA_TRY(want_shape(sv, {B, W - 1, D}, "causal_conv state"));
  if (has_l) REMORA_TRY(want_shape(lv, {B}, "causal_conv lengths"));
  if (has_o) REMORA_TRY(want_shape(ov, {B, W - 1, D}, "causal_conv state_out"));
  const DescView *bp = has_b ? &bv : nullptr, *sp = has_s ? &sv : nullptr, *lp = has_l ? &lv : nullptr;
  REMORA_TRY(want_apart({{&yv, "y", 4}}, {{&xv, "x", 4}, {&wv, "w", 4}, {bp, "bias", 4}, {sp, "state", 4},
                                          {lp, "lengths", 4}, {has_o ? &ov : nullptr, "state_out", 4}}));
  if (has_o)
    REMORA_TRY(want_apart({{&ov, "state_out", 4}},
                          {{&xv, "x", 4}, {&wv, "w", 4}, {bp, "bias", 4}, {sp, "state", 4}, {lp, "lengths", 4}},
                          {{&ov, sp}}));
  REMORA_TRY(want_own_elements({{&yv, "y", 4}, {has_o ? &ov : nullptr, "state_out", 4}}));
  if (B == 0 || D == 0 || (L == 0 && !has_o)) return REMORA_OK;
  ConvArgs a = {};
  a.x = op3(xv), a.y = op3(yv);
  if (has_s) a.state = op3(sv);
  if (has_o) a.state_out = op3(ov);
  a.w = reinterpret_cast<const float *>(wv.data(4)), a.w_d = wv.strides[0], a.w_k = wv.strides[1];
  if (has_b) a.bias = reinterpret_cast<const float *>(bv.data(4)), a.bias_d = bv.strides[0];
  if (has_l) a.lengths = reinterpret_cast<const int *>(lv.data(4)), a.lengths_b = lv.strides[0];
  a.batch = B, a.length = L, a.dim = D, a.silu = spec->silu != 0, a.zero_rest = spec->zero_rest != 0;
  constexpr int V = kVec;
  const bool vec = D % V == 0 && vec_rows(xv, V) && vec_rows(yv, V) && (!has_s || vec_rows(sv, V)) &&
                   (!has_o || vec_rows(ov, V));
  REMORA_TRY(set_grid(a, kFwdRun, vec ? V : 1, "causal_conv_fwd"));
  DeviceGuard guard;
  REMORA_TRY(guard.enter(ctx));
  return vec ? launch_conv<V, false>((int)W, a, (cudaStream_t)stream)
             : launch_conv<1, false>((int)W, a, (cudaStream_t)stream);
}

int remora_b200_causal_conv_bwd_scratch(RemoraB200Ctx *ctx, int64_t batch, int64_t length, int64_t dim, int64_t width,
                                        size_t *bytes) {
  if (ctx == nullptr || bytes == nullptr) return fail(REMORA_ERR_ARG, "causal_conv_bwd_scratch: null pointer");
  if (batch < 0 || length < 0 || dim < 0) return fail(REMORA_ERR_ARG, "causal_conv_bwd_scratch: negative size");
  REMORA_TRY(check_width(width, "causal_conv_bwd_scratch"));
  *bytes = (size_t)bwd_parts(batch, length, dim) * (size_t)(width + 1) * (size_t)dim * 4;
  return REMORA_OK;
}

int remora_b200_causal_conv_bwd(RemoraB200Ctx *ctx, const RemoraCausalConvSpec *spec, const RemoraMemRef3 *x,
                                const RemoraMemRef2 *w, const RemoraMemRef1 *bias, const RemoraMemRef3 *state,
                                const RemoraMemRef1 *lengths, const RemoraMemRef3 *dy, const RemoraMemRef3 *dstate_out,
                                RemoraMemRef3 *dx, RemoraMemRef2 *dw, RemoraMemRef1 *dbias, RemoraMemRef3 *dstate,
                                void *scratch, size_t scratch_bytes, remora_stream_t stream_) {
  if (ctx == nullptr) return fail(REMORA_ERR_ARG, "null context");
  cudaStream_t stream = (cudaStream_t)stream_;
  if (spec == nullptr) return fail(REMORA_ERR_ARG, "causal_conv_bwd: null spec");
  DescView xv, wv, bv, sv, lv, gv, ev, dxv, dwv, dbv, dsv;
  bool has_b, has_s, has_l, has_e, has_db, has_ds;
  REMORA_TRY(read_f32(x, 3, &xv, "causal_conv x"));
  REMORA_TRY(read_f32(w, 2, &wv, "causal_conv w"));
  REMORA_TRY(read_optional(bias, 1, &bv, &has_b, "causal_conv bias"));
  REMORA_TRY(read_optional(state, 3, &sv, &has_s, "causal_conv state"));
  REMORA_TRY(read_optional(lengths, 1, &lv, &has_l, "causal_conv lengths"));
  REMORA_TRY(read_f32(dy, 3, &gv, "causal_conv dy"));
  REMORA_TRY(read_optional(dstate_out, 3, &ev, &has_e, "causal_conv dstate_out"));
  REMORA_TRY(read_f32(dx, 3, &dxv, "causal_conv dx"));
  REMORA_TRY(read_f32(dw, 2, &dwv, "causal_conv dw"));
  REMORA_TRY(read_optional(dbias, 1, &dbv, &has_db, "causal_conv dbias"));
  REMORA_TRY(read_optional(dstate, 3, &dsv, &has_ds, "causal_conv dstate"));
  const int64_t B = xv.sizes[0], L = xv.sizes[1], D = xv.sizes[2], W = wv.sizes[1];
  REMORA_TRY(check_width(W, "causal_conv_bwd"));
  REMORA_TRY(want_shape(wv, {D, W}, "causal_conv w"));
  REMORA_TRY(want_shape(gv, {B, L, D}, "causal_conv dy"));
  REMORA_TRY(want_shape(dxv, {B, L, D}, "causal_conv dx"));
  REMORA_TRY(want_shape(dwv, {D, W}, "causal_conv dw"));
  if (has_b) REMORA_TRY(want_shape(bv, {D}, "causal_conv bias"));
  if (has_db) REMORA_TRY(want_shape(dbv, {D}, "causal_conv dbias"));
  if (has_s) REMORA_TRY(want_shape(sv, {B, W - 1, D}, "causal_conv state"));
  if (has_e) REMORA_TRY(want_shape(ev, {B, W - 1, D}, "causal_conv dstate_out"));
  if (has_ds) REMORA_TRY(want_shape(dsv, {B, W - 1, D}, "causal_conv dstate"));
  if (has_l) REMORA_TRY(want_shape(lv, {B}, "causal_conv lengths"));
  REMORA_TRY(want_apart({{&dxv, "dx", 4}, {&dwv, "dw", 4}, {has_db ? &dbv : nullptr, "dbias", 4},
                         {has_ds ? &dsv : nullptr, "dstate", 4}},
                        {{&xv, "x", 4}, {&wv, "w", 4}, {&gv, "dy", 4}, {has_b ? &bv : nullptr, "bias", 4},
                         {has_s ? &sv : nullptr, "state", 4}, {has_l ? &lv : nullptr, "lengths", 4},
                         {has_e ? &ev : nullptr, "dstate_out", 4}}));
  REMORA_TRY(want_own_elements({{&dxv, "dx", 4}, {&dwv, "dw", 4}, {has_db ? &dbv : nullptr, "dbias", 4},
                                {has_ds ? &dsv : nullptr, "dstate", 4}}));
  const int64_t parts = bwd_parts(B, L, D);
  REMORA_TRY(want_scratch(scratch, scratch_bytes, (size_t)parts * (size_t)(W + 1) * (size_t)D * 4, "causal_conv_bwd"));
  if (D == 0) return REMORA_OK;
  ConvArgs a = {};
  a.x = op3(xv), a.dy = op3(gv), a.dx = op3(dxv);
  if (has_s) a.state = op3(sv);
  if (has_e) a.dstate_out = op3(ev);
  if (has_ds) a.dstate = op3(dsv);
  a.w = reinterpret_cast<const float *>(wv.data(4)), a.w_d = wv.strides[0], a.w_k = wv.strides[1];
  if (has_b) a.bias = reinterpret_cast<const float *>(bv.data(4)), a.bias_d = bv.strides[0];
  if (has_l) a.lengths = reinterpret_cast<const int *>(lv.data(4)), a.lengths_b = lv.strides[0];
  a.batch = B, a.length = L, a.dim = D, a.silu = spec->silu != 0, a.zero_rest = spec->zero_rest != 0;
  a.part = static_cast<float *>(scratch);
  constexpr int V = kVec;
  const bool vec = D % V == 0 && vec_rows(xv, V) && vec_rows(gv, V) && vec_rows(dxv, V) &&
                   (!has_s || vec_rows(sv, V)) && (!has_e || vec_rows(ev, V)) && (!has_ds || vec_rows(dsv, V));
  REMORA_TRY(set_grid(a, kBwdRun, vec ? V : 1, "causal_conv_bwd"));
  DeviceGuard guard;
  REMORA_TRY(guard.enter(ctx));
  if (B > 0)
    REMORA_TRY((vec ? launch_conv<V, true>((int)W, a, stream) : launch_conv<1, true>((int)W, a, stream)));
  // a row of part: W rows of dw and one of dbias, each over the channels
  const Columns to = {reinterpret_cast<float *>(dwv.data(4)), D, dwv.strides[1], dwv.strides[0], W * D,
                      has_db ? reinterpret_cast<float *>(dbv.data(4)) : nullptr, has_db ? dbv.strides[0] : 0};
  return reduce_rows(a.part, B * a.blocks_t, (W + 1) * D, to, stream);
}

int remora_b200_causal_conv_step(RemoraB200Ctx *ctx, const RemoraCausalConvSpec *spec, const RemoraMemRef2 *x,
                                 const RemoraMemRef3 *state, const RemoraMemRef2 *w, const RemoraMemRef1 *bias,
                                 const RemoraMemRef1 *slots, RemoraMemRef2 *y, RemoraMemRef3 *state_out,
                                 remora_stream_t stream) {
  if (ctx == nullptr) return fail(REMORA_ERR_ARG, "null context");
  if (spec == nullptr) return fail(REMORA_ERR_ARG, "causal_conv_step: null spec");
  DescView xv, sv, wv, bv, lv, yv, ov;
  bool has_b, has_l;
  REMORA_TRY(read_f32(x, 2, &xv, "causal_conv_step x"));
  REMORA_TRY(read_f32(state, 3, &sv, "causal_conv_step state"));
  REMORA_TRY(read_f32(w, 2, &wv, "causal_conv_step w"));
  REMORA_TRY(read_optional(bias, 1, &bv, &has_b, "causal_conv_step bias"));
  REMORA_TRY(read_optional(slots, 1, &lv, &has_l, "causal_conv_step slots"));
  REMORA_TRY(read_f32(y, 2, &yv, "causal_conv_step y"));
  REMORA_TRY(read_f32(state_out, 3, &ov, "causal_conv_step state_out"));
  const int64_t B = xv.sizes[0], D = xv.sizes[1], W = wv.sizes[1], S = sv.sizes[0];
  REMORA_TRY(check_width(W, "causal_conv_step"));
  REMORA_TRY(want_shape(wv, {D, W}, "causal_conv_step w"));
  REMORA_TRY(want_shape(yv, {B, D}, "causal_conv_step y"));
  REMORA_TRY(want_shape(sv, {S, W - 1, D}, "causal_conv_step state"));
  REMORA_TRY(want_shape(ov, {S, W - 1, D}, "causal_conv_step state_out"));
  if (has_b) REMORA_TRY(want_shape(bv, {D}, "causal_conv_step bias"));
  if (has_l) REMORA_TRY(want_shape(lv, {B}, "causal_conv_step slots"));
  if (!has_l && B > S)
    return fail(REMORA_ERR_SHAPE, "causal_conv_step: %lld rows and %lld states", (long long)B, (long long)S);
  if (B > 65535) return fail(REMORA_ERR_LIMIT, "causal_conv_step: more than 65535 rows");
  REMORA_TRY(want_apart({{&yv, "y", 4}, {&ov, "state_out", 4}},
                        {{&xv, "x", 4}, {&sv, "state", 4}, {&wv, "w", 4}, {has_b ? &bv : nullptr, "bias", 4},
                         {has_l ? &lv : nullptr, "slots", 4}}, {{&ov, &sv}}));
  REMORA_TRY(want_own_elements({{&yv, "y", 4}, {&ov, "state_out", 4}}));
  if (B == 0 || D == 0) return REMORA_OK;
  StepArgs a = {};
  a.state = op3(sv), a.state_out = op3(ov);
  a.x = reinterpret_cast<const float *>(xv.data(4)), a.x_b = xv.strides[0], a.x_d = xv.strides[1];
  a.y = reinterpret_cast<float *>(yv.data(4)), a.y_b = yv.strides[0], a.y_d = yv.strides[1];
  a.w = reinterpret_cast<const float *>(wv.data(4)), a.w_d = wv.strides[0], a.w_k = wv.strides[1];
  if (has_b) a.bias = reinterpret_cast<const float *>(bv.data(4)), a.bias_d = bv.strides[0];
  if (has_l) a.slots = reinterpret_cast<const int *>(lv.data(4)), a.slots_b = lv.strides[0];
  a.rows = S, a.dim = D, a.silu = spec->silu != 0, a.zero_rest = spec->zero_rest != 0;
  const bool vec = D % 4 == 0 && vec_rows(xv, 4) && vec_rows(yv, 4) && vec_rows(sv, 4) && vec_rows(ov, 4);
  DeviceGuard guard;
  REMORA_TRY(guard.enter(ctx));
  return vec ? launch_step<4>((int)W, B, a, (cudaStream_t)stream) : launch_step<1>((int)W, B, a, (cudaStream_t)stream);
}

}  // extern "C"
