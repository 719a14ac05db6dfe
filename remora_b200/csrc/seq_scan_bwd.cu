// seq_scan_bwd.cu — gradients of the selective state space scan.
//
//   dp = dy silu(z);  dz = dy p silu'(z)
//   G_t[n] = c_t[n] dp_t + exp(s_{t+1} a[n]) G_{t+1}[n]          (adjoint of h_t)
//   dc_t[n] = sum_d dp h_t[n];  db_t[n] = sum_d G s u;  da[n] = sum_t G s (exp(s a) h_{t-1})[n]
//   du = s sum_n G b + d dp;  ds = sum_n G a (exp(s a) h_{t-1}) + u sum_n G b;  ddelta = ds f'(delta + bias)
//
// A thread walks time from the end in pieces of kSaveEvery steps.  For each
// it takes the state that the forward kept at the piece's start, runs the
// recurrence forward once, keeping exp(s a) and exp(s a) h of every step in
// registers, then the adjoint backward: one exponential per position, channel
// and state in all.  db and dc sum over the channels of a group: over a warp
// by shuffle, over a block through shared memory, over blocks by partial rows
// in scratch that a second kernel adds in block order.
#include <algorithm>

#include "seq_scan.cuh"

namespace remora {
namespace seq {
namespace {

constexpr int kSteps = kSaveEvery;
constexpr int kWarps = kScanThreads / 32;

// Sums v over the 32 / NL channel lanes of a warp; CNT of the sums end in
// v[0 .. CNT-1] of each lane, the sums FIRST .. FIRST + CNT - 1.
template <int NL>
struct ChannelSum {
  static constexpr int kLanesD = 32 / NL;
  static constexpr int kCount = kLanesD >= 8 ? 1 : 8 / kLanesD;
  __device__ static __forceinline__ void run(float (&v)[8], int lane) {
    int half = 4;
#pragma unroll
    for (int o = 16; o >= NL; o >>= 1) {
      if (half >= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < half) {
            const float send = up ? v[k] : v[k + half];
            const float keep = up ? v[k + half] : v[k];
            v[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
          }
        half >>= 1;
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      }
    }
  }
  __device__ static __forceinline__ int first(int lane) { return lane / (NL > 4 ? NL : 4) * kCount; }
  // of the lanes that hold the same sum, one stores it
  __device__ static __forceinline__ bool stores(int lane) { return NL >= 4 || (lane & 3) < NL; }
};

template <int NL, bool PADDED>
__global__ void __launch_bounds__(kScanThreads) scan_bwd_kernel(const ScanArgs a) {
  constexpr int NP = 4 * NL;
  constexpr int PF = kSteps / NL;
  using Sum = ChannelSum<NL>;
  __shared__ __align__(16) float bs[2][kSteps * NP], cs[2][kSteps * NP];
  __shared__ __align__(16) float red[kWarps][kSteps][2 * NP];  // per step: db[NP], dc[NP]
  const Place<NL> at(a);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t len = scan_length(a, at.b);
  const int64_t t0 = at.chunk * a.chunk, t_end = min(t0 + a.chunk, len);
  const int64_t prow = at.b * a.chunks + at.chunk;
  const int nv = a.states - 4 * at.q;
  float A[4], A2[4], G[4], dA[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool on = at.live && k < nv;
    A[k] = on ? a.a[at.d * a.a_d + (4 * at.q + k) * a.a_n] : 0.0f;
    A2[k] = A[k] * kLog2e;
    G[k] = dA[k] = 0.0f;
    if (on && a.chunks == 1 && a.dh_last.p)
      G[k] = a.dh_last.p[at.b * a.dh_last.s0 + at.d * a.dh_last.s1 + (4 * at.q + k) * a.dh_last.s2];
  }
  if (a.chunks > 1 && (t0 < len || t0 == 0))
    unpack(reinterpret_cast<const float4 *>(a.sum_h)[(prow * a.dim + at.d) * NL + at.q], G);
  const float bias = a.bias ? a.bias[at.d * a.bias_s] : 0.0f;
  const float skip = a.d ? a.d[at.d * a.d_s] : 0.0f;
  const float *up = a.u.p + at.b * a.u.s0 + at.d * a.u.s2;
  const float *dp = a.delta.p + at.b * a.delta.s0 + at.d * a.delta.s2;
  const float *zp = a.z.p + at.b * a.z.s0 + at.d * a.z.s2;
  const float *yp = a.dy.p + at.b * a.dy.s0 + at.d * a.dy.s2;
  float ru[PF], rd[PF], rz[PF], ry[PF];
  float4 rh = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const int64_t kept = (a.length + kSaveEvery - 1) / kSaveEvery;
  auto fetch = [&](int64_t base) {
#pragma unroll
    for (int i = 0; i < PF; ++i) {
      const int64_t t = base + i * NL + at.q;
      const bool on = at.live && t < t_end;
      ru[i] = on ? up[t * a.u.s1] : 0.0f;
      rd[i] = on ? dp[t * a.delta.s1] : 0.0f;
      ry[i] = on ? yp[t * a.dy.s1] : 0.0f;
      if (a.z.p) rz[i] = on ? zp[t * a.z.s1] : 0.0f;
    }
    if (at.live)
      rh = reinterpret_cast<const float4 *>(a.saved)[((at.b * kept + base / kSaveEvery) * a.dim + at.d) * NL + at.q];
  };
  auto stage = [&](int buf, int64_t t) {
    stage_rows<NL, kSteps>(bs[buf], a.b, a.vec_b, at.b, at.g, t, t_end, a.states);
    stage_rows<NL, kSteps>(cs[buf], a.c, a.vec_c, at.b, at.g, t, t_end, a.states);
    copy_commit();
  };
  float sum_d = 0.0f, sum_bias = 0.0f;
  int buf = 0;
  const int64_t last = t_end > t0 ? t0 + (t_end - 1 - t0) / kSteps * kSteps : t0 - kSteps;
  if (last >= t0) {
    stage(0, last);
    fetch(last);
  }
  for (int64_t base = last; base >= t0; base -= kSteps, buf ^= 1) {
    if (base - kSteps >= t0)
      stage(buf ^ 1, base - kSteps);
    else
      copy_commit();
    copy_wait<1>();
    __syncthreads();  // b and c are there; red of the turn before is read
    float s[PF], sig[PF], su[PF], u[PF], dyp[PF], dzf[PF], h[4];
    unpack(rh, h);
#pragma unroll
    for (int i = 0; i < PF; ++i) {
      const float raw = rd[i] + bias;
      sig[i] = 1.0f;
      s[i] = a.softplus ? softplus(raw, &sig[i]) : raw;
      u[i] = ru[i];
      su[i] = s[i] * u[i];
      dyp[i] = ry[i];
      dzf[i] = 0.0f;
      if (a.z.p) {
        const float sz = sigmoid(rz[i]);
        dyp[i] = ry[i] * (rz[i] * sz);
        dzf[i] = ry[i] * (sz * fmaf(rz[i], 1.0f - sz, 1.0f));
      }
    }
    if (base - kSteps >= t0) fetch(base - kSteps);
    float e[kSteps][4], eh[kSteps][4];
    auto piece = [&](auto whole) {
      constexpr bool FULL = decltype(whole)::value;
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        float part[NL];
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const int t = i * NL + j;
          part[j] = 0.0f;
          const float sj = __shfl_sync(0xffffffffu, s[i], j, NL);
          const float suj = __shfl_sync(0xffffffffu, su[i], j, NL);
          if (FULL || base + t < t_end) {
            float b[4], c[4];
            unpack(*reinterpret_cast<const float4 *>(&bs[buf][t * NP + 4 * at.q]), b);
            unpack(*reinterpret_cast<const float4 *>(&cs[buf][t * NP + 4 * at.q]), c);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              e[t][k] = ex2(sj * A2[k]);
              eh[t][k] = e[t][k] * h[k];
              h[k] = eh[t][k] + (PADDED && k >= nv ? 0.0f : suj * b[k]);
              part[j] = fmaf(h[k], c[k], part[j]);
            }
          }
        }
        transpose_sum<NL>(part, at.q);
        const int64_t t = base + i * NL + at.q;
        if (a.dz.p && at.live && t < t_end)
          a.dz.p[at.b * a.dz.s0 + t * a.dz.s1 + at.d * a.dz.s2] = dzf[i] * fmaf(skip, u[i], part[0]);
      }
#pragma unroll
      for (int i = PF - 1; i >= 0; --i) {
        float gb[NL], ga[NL];
#pragma unroll
        for (int j = NL - 1; j >= 0; --j) {
          const int t = i * NL + j;
          gb[j] = ga[j] = 0.0f;
          const float sj = __shfl_sync(0xffffffffu, s[i], j, NL);
          const float suj = __shfl_sync(0xffffffffu, su[i], j, NL);
          const float dj = __shfl_sync(0xffffffffu, dyp[i], j, NL);
          if (FULL || base + t < t_end) {
            float b[4], c[4], v[8];
            unpack(*reinterpret_cast<const float4 *>(&bs[buf][t * NP + 4 * at.q]), b);
            unpack(*reinterpret_cast<const float4 *>(&cs[buf][t * NP + 4 * at.q]), c);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const bool pad = PADDED && k >= nv;
              const float hk = eh[t][k] + (pad ? 0.0f : suj * b[k]);
              G[k] += pad ? 0.0f : c[k] * dj;
              v[k] = G[k] * suj;
              v[4 + k] = dj * hk;
              gb[j] = fmaf(G[k], b[k], gb[j]);
              const float geh = G[k] * eh[t][k];
              dA[k] = fmaf(geh, sj, dA[k]);
              ga[j] = fmaf(geh, A[k], ga[j]);
              G[k] *= e[t][k];
            }
            if (PADDED || !at.live) {
              // lanes without a channel hold zeros already but for b and c
              // that are not finite; states past N are never stored
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (!at.live) v[k] = 0.0f;
            }
            Sum::run(v, lane);
            if (Sum::stores(lane)) {
              const int first = Sum::first(lane);
#pragma unroll
              for (int k = 0; k < Sum::kCount; ++k) {
                const int f = first + k;
                red[warp][t][(f >> 2) * NP + 4 * at.q + (f & 3)] = v[k];
              }
            }
          }
        }
        transpose_sum<NL>(gb, at.q);
        transpose_sum<NL>(ga, at.q);
        const int64_t t = base + i * NL + at.q;
        if (at.live && t < t_end) {
          const float ds = fmaf(u[i], gb[0], ga[0]) * sig[i];
          a.du.p[at.b * a.du.s0 + t * a.du.s1 + at.d * a.du.s2] = fmaf(s[i], gb[0], skip * dyp[i]);
          a.ddelta.p[at.b * a.ddelta.s0 + t * a.ddelta.s1 + at.d * a.ddelta.s2] = ds;
          sum_d = fmaf(dyp[i], u[i], sum_d);
          sum_bias += ds;
        }
      }
    };
    if (base + kSteps <= t_end)
      piece(std::true_type{});
    else
      piece(std::false_type{});
    __syncthreads();
    // join the warps; a row of part_bc is one channel block's share
    const int64_t plane = a.batch * a.length * a.groups * a.states;
    for (int i = threadIdx.x; i < kSteps * 2 * NP; i += kScanThreads) {
      const int t = i / (2 * NP), f = i % (2 * NP), n = f % NP;
      if (base + t >= t_end || n >= a.states) continue;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += red[w][t][f];
      const bool is_c = f >= NP;
      if (a.blocks_d == 1) {
        const Op4 &o = is_c ? a.dc : a.db;
        o.p[at.b * o.s0 + (base + t) * o.s1 + at.g * o.s2 + n * o.s3] = v;
      } else {
        a.part_bc[(at.bd * 2 + is_c) * plane + ((at.b * a.length + base + t) * a.groups + at.g) * a.states + n] = v;
      }
    }
  }
  if (a.dh0.p && at.live && t0 == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < nv) a.dh0.p[at.b * a.dh0.s0 + at.d * a.dh0.s1 + (4 * at.q + k) * a.dh0.s2] = G[k];
  }
#pragma unroll
  for (int o = 1; o < NL; o <<= 1) {
    sum_d += __shfl_xor_sync(0xffffffffu, sum_d, o);
    sum_bias += __shfl_xor_sync(0xffffffffu, sum_bias, o);
  }
  if (at.live) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < nv) a.part_a[(prow * a.dim + at.d) * a.states + 4 * at.q + k] = dA[k];
    if (at.q == 0) {
      a.part_d[prow * 2 * a.dim + at.d] = sum_d;
      a.part_d[(prow * 2 + 1) * a.dim + at.d] = sum_bias;
    }
  }
}

// First pass of a cut time axis: the adjoint that leaves a piece at its start
// when none enters at its end, and the piece's sum of steps.
template <int NL, bool PADDED>
__global__ void __launch_bounds__(kScanThreads) scan_adjoint_kernel(const ScanArgs a) {
  constexpr int NP = 4 * NL;
  constexpr int PF = kSteps / NL;
  __shared__ __align__(16) float cs[2][kSteps * NP];
  const Place<NL> at(a);
  const int64_t len = scan_length(a, at.b);
  const int64_t t0 = at.chunk * a.chunk, t_end = min(t0 + a.chunk, len);
  if (t0 >= len && t0 > 0) return;
  const int nv = a.states - 4 * at.q;
  float A2[4], G[4] = {0.0f, 0.0f, 0.0f, 0.0f}, total = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    A2[k] = at.live && k < nv ? a.a[at.d * a.a_d + (4 * at.q + k) * a.a_n] * kLog2e : 0.0f;
  const float bias = a.bias ? a.bias[at.d * a.bias_s] : 0.0f;
  const float *dp = a.delta.p + at.b * a.delta.s0 + at.d * a.delta.s2;
  const float *zp = a.z.p + at.b * a.z.s0 + at.d * a.z.s2;
  const float *yp = a.dy.p + at.b * a.dy.s0 + at.d * a.dy.s2;
  float rd[PF], rz[PF], ry[PF];
  auto fetch = [&](int64_t base) {
#pragma unroll
    for (int i = 0; i < PF; ++i) {
      const int64_t t = base + i * NL + at.q;
      const bool on = at.live && t < t_end;
      rd[i] = on ? dp[t * a.delta.s1] : 0.0f;
      ry[i] = on ? yp[t * a.dy.s1] : 0.0f;
      if (a.z.p) rz[i] = on ? zp[t * a.z.s1] : 0.0f;
    }
  };
  auto stage = [&](int buf, int64_t t) {
    stage_rows<NL, kSteps>(cs[buf], a.c, a.vec_c, at.b, at.g, t, t_end, a.states);
    copy_commit();
  };
  int buf = 0;
  const int64_t last = t_end > t0 ? t0 + (t_end - 1 - t0) / kSteps * kSteps : t0 - kSteps;
  if (last >= t0) {
    stage(0, last);
    fetch(last);
  }
  for (int64_t base = last; base >= t0; base -= kSteps, buf ^= 1) {
    if (base - kSteps >= t0)
      stage(buf ^ 1, base - kSteps);
    else
      copy_commit();
    copy_wait<1>();
    __syncthreads();
    float s[PF], dyp[PF];
#pragma unroll
    for (int i = 0; i < PF; ++i) {
      const float raw = rd[i] + bias;
      float sig;
      s[i] = a.softplus ? softplus(raw, &sig) : raw;
      dyp[i] = a.z.p ? ry[i] * (rz[i] * sigmoid(rz[i])) : ry[i];
      if (base + i * NL + at.q < t_end) total += s[i];
    }
    if (base - kSteps >= t0) fetch(base - kSteps);
#pragma unroll
    for (int i = PF - 1; i >= 0; --i)
#pragma unroll
      for (int j = NL - 1; j >= 0; --j) {
        const int t = i * NL + j;
        const float sj = __shfl_sync(0xffffffffu, s[i], j, NL);
        const float dj = __shfl_sync(0xffffffffu, dyp[i], j, NL);
        if (base + t < t_end) {
          float c[4];
          unpack(*reinterpret_cast<const float4 *>(&cs[buf][t * NP + 4 * at.q]), c);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            G[k] += PADDED && k >= nv ? 0.0f : c[k] * dj;
            G[k] *= ex2(sj * A2[k]);
          }
        }
      }
    __syncthreads();
  }
#pragma unroll
  for (int o = 1; o < NL; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (at.live) {
    const int64_t i = (at.b * a.chunks + at.chunk) * a.dim + at.d;
    reinterpret_cast<float4 *>(a.sum_h)[i * NL + at.q] = make_float4(G[0], G[1], G[2], G[3]);
    if (at.q == 0) a.sum_dt[i] = total;
  }
}

// db and dc of one position, group and state: the channel blocks' shares.
__global__ void __launch_bounds__(256) join_bc_kernel(const ScanArgs a) {
  const int64_t plane = a.batch * a.length * a.groups * a.states;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= plane) return;
  const int64_t n = i % a.states, g = i / a.states % a.groups, bt = i / a.states / a.groups;
  const int64_t t = bt % a.length, b = bt / a.length;
  if (t >= scan_length(a, b)) return;
  float vb = 0.0f, vc = 0.0f;
  for (int64_t k = 0; k < a.blocks_d; ++k) {
    vb += a.part_bc[2 * k * plane + i];
    vc += a.part_bc[(2 * k + 1) * plane + i];
  }
  a.db.p[b * a.db.s0 + t * a.db.s1 + g * a.db.s2 + n * a.db.s3] = vb;
  a.dc.p[b * a.dc.s0 + t * a.dc.s1 + g * a.dc.s2 + n * a.dc.s3] = vc;
}

// ------------------------------------------------------------------ host --
Op3 op3(const DescView &v) {
  return {reinterpret_cast<float *>(v.data(4)), v.strides[0], v.strides[1], v.strides[2]};
}

// As the forward's: pieces only where the channels give too few warps.
void cut_time(int64_t batch, int64_t length, int64_t dim, int nl, int64_t groups, int64_t *chunks, int64_t *chunk) {
  const int64_t per_block = kScanThreads / nl, per = dim / std::max<int64_t>(groups, 1);
  const int64_t blocks = std::max<int64_t>(1, batch * groups * ((per + per_block - 1) / per_block));
  int64_t n = 1;
  if (blocks < 148) n = std::max<int64_t>(1, std::min<int64_t>(148 * 2 / blocks, length / 64));
  *chunk = std::max<int64_t>(32, ((length + n - 1) / n + 31) / 32 * 32);
  *chunks = std::max<int64_t>(1, (length + *chunk - 1) / *chunk);
}

struct Layout {
  int64_t chunks, chunk;
  size_t sum_h, sum_dt, part_bc, part_a, part_d, total;  // offsets in floats
};

Layout layout_for(int64_t batch, int64_t length, int64_t dim, int states, int64_t groups) {
  Layout l = {};
  const int nl = lanes_for(states);
  cut_time(batch, length, dim, nl, groups, &l.chunks, &l.chunk);
  const int64_t per_block = kScanThreads / nl, per = dim / std::max<int64_t>(groups, 1);
  const int64_t blocks_d = (per + per_block - 1) / per_block;
  size_t at = 0;
  auto take = [&](int64_t n) {
    const size_t o = at;
    at += ((size_t)n + 63) & ~(size_t)63;
    return o;
  };
  l.sum_h = take(l.chunks > 1 ? batch * l.chunks * dim * 4 * nl : 0);
  l.sum_dt = take(l.chunks > 1 ? batch * l.chunks * dim : 0);
  l.part_bc = take(blocks_d > 1 ? blocks_d * 2 * batch * length * groups * states : 0);
  l.part_a = take(batch * l.chunks * dim * states);
  l.part_d = take(batch * l.chunks * 2 * dim);
  l.total = at;
  return l;
}

int launch_bwd(const ScanArgs &a, int nl, bool adjoint, cudaStream_t stream) {
  const unsigned grid = (unsigned)(a.batch * a.chunks * a.groups * a.blocks_d);
  const bool padded = a.states != 4 * nl;
  note_launch();
#define REMORA_SCAN_CASE(NL)                                                        \
  case NL:                                                                          \
    if (adjoint && padded)                                                          \
      scan_adjoint_kernel<NL, true><<<grid, kScanThreads, 0, stream>>>(a);          \
    else if (adjoint)                                                               \
      scan_adjoint_kernel<NL, false><<<grid, kScanThreads, 0, stream>>>(a);         \
    else if (padded)                                                                \
      scan_bwd_kernel<NL, true><<<grid, kScanThreads, 0, stream>>>(a);              \
    else                                                                            \
      scan_bwd_kernel<NL, false><<<grid, kScanThreads, 0, stream>>>(a);             \
    break;
  switch (nl) {
    REMORA_SCAN_CASE(1)
    REMORA_SCAN_CASE(2)
    REMORA_SCAN_CASE(4)
    REMORA_SCAN_CASE(8)
    REMORA_SCAN_CASE(16)
  }
#undef REMORA_SCAN_CASE
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

}  // namespace
}  // namespace seq
}  // namespace remora

using namespace remora;
using namespace remora::seq;

extern "C" {

int remora_b200_selective_scan_bwd_scratch(RemoraB200Ctx *ctx, int64_t batch, int64_t length, int64_t dim,
                                           int64_t states, int64_t groups, size_t *bytes) {
  // the same checks of the sizes as the forward's
  REMORA_TRY(remora_b200_selective_scan_fwd_scratch(ctx, batch, length, dim, states, groups, bytes));
  *bytes = layout_for(batch, length, dim, (int)states, groups).total * 4;
  return REMORA_OK;
}

int remora_b200_selective_scan_bwd(RemoraB200Ctx *ctx, const RemoraSelectiveScanSpec *spec,
                                   const RemoraSelectiveScanIn *in, const RemoraMemRef3 *dy,
                                   const RemoraMemRef3 *dh_last, const void *saved, size_t saved_bytes,
                                   const RemoraSelectiveScanGrads *grads, void *scratch, size_t scratch_bytes,
                                   remora_stream_t stream_) {
  if (ctx == nullptr) return fail(REMORA_ERR_ARG, "null context");
  cudaStream_t stream = (cudaStream_t)stream_;
  ScanArgs a = {};
  DescView v[10], gy, gh, o[9];
  bool has_gh, have[9];
  REMORA_TRY(read_scan_in(spec, in, &a, v, "selective_scan_bwd"));
  if (grads == nullptr) return fail(REMORA_ERR_ARG, "selective_scan_bwd: null gradients");
  REMORA_TRY(read_f32(dy, 3, &gy, "selective_scan dy"));
  REMORA_TRY(read_optional(dh_last, 3, &gh, &has_gh, "selective_scan dh_last"));
  REMORA_TRY(read_f32(grads->du, 3, &o[0], "selective_scan du"));
  REMORA_TRY(read_f32(grads->ddelta, 3, &o[1], "selective_scan ddelta"));
  REMORA_TRY(read_f32(grads->da, 2, &o[2], "selective_scan da"));
  REMORA_TRY(read_f32(grads->db, 4, &o[3], "selective_scan db"));
  REMORA_TRY(read_f32(grads->dc, 4, &o[4], "selective_scan dc"));
  REMORA_TRY(read_optional(grads->dd, 1, &o[5], &have[5], "selective_scan dd"));
  REMORA_TRY(read_optional(grads->dz, 3, &o[6], &have[6], "selective_scan dz"));
  REMORA_TRY(read_optional(grads->ddelta_bias, 1, &o[7], &have[7], "selective_scan ddelta_bias"));
  REMORA_TRY(read_optional(grads->dh0, 3, &o[8], &have[8], "selective_scan dh0"));
  const int64_t B = a.batch, L = a.length, D = a.dim, G = a.groups, N = a.states;
  REMORA_TRY(want_shape(gy, {B, L, D}, "selective_scan dy"));
  if (has_gh) REMORA_TRY(want_shape(gh, {B, D, N}, "selective_scan dh_last"));
  REMORA_TRY(want_shape(o[0], {B, L, D}, "selective_scan du"));
  REMORA_TRY(want_shape(o[1], {B, L, D}, "selective_scan ddelta"));
  REMORA_TRY(want_shape(o[2], {D, N}, "selective_scan da"));
  REMORA_TRY(want_shape(o[3], {B, L, G, N}, "selective_scan db"));
  REMORA_TRY(want_shape(o[4], {B, L, G, N}, "selective_scan dc"));
  if (have[5]) REMORA_TRY(want_shape(o[5], {D}, "selective_scan dd"));
  if (have[6]) REMORA_TRY(want_shape(o[6], {B, L, D}, "selective_scan dz"));
  if (have[7]) REMORA_TRY(want_shape(o[7], {D}, "selective_scan ddelta_bias"));
  if (have[8]) REMORA_TRY(want_shape(o[8], {B, D, N}, "selective_scan dh0"));
  if (have[6] && in->z == nullptr) return fail(REMORA_ERR_ARG, "selective_scan_bwd: dz without z");
  auto out = [&](int k) { return k < 5 || have[k] ? &o[k] : nullptr; };
  auto given = [&](int k) { return v[k].aligned != nullptr ? &v[k] : nullptr; };
  REMORA_TRY(want_apart({{out(0), "du", 4}, {out(1), "ddelta", 4}, {out(2), "da", 4}, {out(3), "db", 4},
                         {out(4), "dc", 4}, {out(5), "dd", 4}, {out(6), "dz", 4}, {out(7), "ddelta_bias", 4},
                         {out(8), "dh0", 4}},
                        {{given(0), "u", 4}, {given(1), "delta", 4}, {given(2), "a", 4}, {given(3), "b", 4},
                         {given(4), "c", 4}, {given(5), "d", 4}, {given(6), "z", 4}, {given(7), "delta_bias", 4},
                         {given(8), "h0", 4}, {given(9), "lengths", 4}, {&gy, "dy", 4},
                         {has_gh ? &gh : nullptr, "dh_last", 4}}));
  const int nl = lanes_for(a.states);
  const Layout l = layout_for(B, L, D, a.states, G);
  size_t need = 0;
  REMORA_TRY(remora_b200_selective_scan_saved(B, L, D, N, &need));
  REMORA_TRY(want_scratch(saved, saved_bytes, need, "selective_scan_bwd (saved)"));
  REMORA_TRY(want_scratch(scratch, scratch_bytes, l.total * 4, "selective_scan_bwd"));
  if (D == 0) return REMORA_OK;
  a.dy = op3(gy);
  if (has_gh) a.dh_last = op3(gh);
  a.du = op3(o[0]), a.ddelta = op3(o[1]);
  a.db = {reinterpret_cast<float *>(o[3].data(4)), o[3].strides[0], o[3].strides[1], o[3].strides[2], o[3].strides[3]};
  a.dc = {reinterpret_cast<float *>(o[4].data(4)), o[4].strides[0], o[4].strides[1], o[4].strides[2], o[4].strides[3]};
  if (have[6]) a.dz = op3(o[6]);
  if (have[8]) a.dh0 = op3(o[8]);
  a.chunks = l.chunks, a.chunk = l.chunk;
  float *base = static_cast<float *>(scratch);
  a.sum_h = base + l.sum_h, a.sum_dt = base + l.sum_dt, a.part_bc = base + l.part_bc;
  a.part_a = base + l.part_a, a.part_d = base + l.part_d;
  a.saved = static_cast<float *>(const_cast<void *>(saved));
  if (B * a.chunks * G * a.blocks_d > 0x7fffffff || B * L * G * N / 256 > 0x7ffffffe || B * D * 4 * nl / 256 > 0x7ffffffe)
    return fail(REMORA_ERR_LIMIT, "selective_scan_bwd: too many blocks");
  DeviceGuard guard;
  REMORA_TRY(guard.enter(ctx));
  if (B > 0) {
    if (a.chunks > 1) {
      REMORA_TRY(launch_bwd(a, nl, true, stream));
      REMORA_TRY(combine_chunks(a, nl, true, stream));
    }
    REMORA_TRY(launch_bwd(a, nl, false, stream));
    if (a.blocks_d > 1 && L > 0) {
      note_launch();
      join_bc_kernel<<<(unsigned)((B * L * G * N + 255) / 256), 256, 0, stream>>>(a);
      REMORA_CUDA_TRY(cudaGetLastError());
    }
  }
  const Columns da = {reinterpret_cast<float *>(o[2].data(4)), N, o[2].strides[0], o[2].strides[1], D * N, nullptr, 0};
  REMORA_TRY(reduce_rows(a.part_a, B * a.chunks, D * N, da, stream));
  if (!have[5] && !have[7]) return REMORA_OK;
  const Columns dd = {have[5] ? reinterpret_cast<float *>(o[5].data(4)) : nullptr, D, 0, have[5] ? o[5].strides[0] : 0, D,
                      have[7] ? reinterpret_cast<float *>(o[7].data(4)) : nullptr, have[7] ? o[7].strides[0] : 0};
  return reduce_rows(a.part_d, B * a.chunks, 2 * D, dd, stream);
}

}  // extern "C"
