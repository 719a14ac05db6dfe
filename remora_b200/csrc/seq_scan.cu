// seq_scan.cu — selective state space scan: forward over prompts and training
// sequences, and one step for single tokens.
//
//   s = f(delta + bias);  h[n] = exp(s a[n]) h[n] + s u b[n];  p = sum_n c[n] h[n] + d u;  y = p silu(z)
//
// Per position and channel: 16 bytes of HBM (u, delta, z, y), N exponentials
// and about 6 N other operations.  At N = 16 the exponentials bound it: the
// special function units give 16 per clock and SM, 4.5e12 a second, and three
// quarters of that is what the first pass reaches.
//
// The recurrence is serial in time.  Where batch x channels give too few
// threads, time is cut into pieces: a first pass gives each piece's end state
// from a zero start and its sum of steps (its decay is exp(a sum s)), a small
// kernel joins them, and the main pass starts each piece from its own state.
// That doubles the exponentials, but a warp alone on its scheduler runs at a
// third of the rate of four.  Cut, 1 x 4096 x 2048 x 16 takes 120 us (49 first pass,
// 5 join, 66 main), 4 x 2048 x 2048 x 16 with the states kept for the backward 229
// (88, 6, 135).  Measured when cut they took 128 and 241: uncut, 522 and 286; decays
// kept in registers between the passes and the pieces exchanged inside a block (one
// exponential per state), 237 for the prompt, at two blocks per SM for want of
// registers; two states of one channel per thread, so that four times the threads
// need no cut, 253 for the second size.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "seq_scan.cuh"

namespace remora {
namespace seq {
namespace {

constexpr int kTile = 32;   // steps of b and c staged at a time
constexpr int64_t kBlocks = 148 * 8;  // blocks of a cut time axis: two rounds of 4 per SM
constexpr int64_t kCutBelow = 148 * 3;

// MAIN: writes y (and h_last, saved).  Otherwise the first pass of a cut time
// axis: sum_h and sum_dt.  PADDED: N is not 4 NL; the states past N must stay
// zero even where s u is not finite.  Four blocks per SM for one lane per channel
// too (4 x 2000 x 2000 x 4: 67 and 46 us, against 85 and 69 with two); three for
// the main pass of two lanes, which spills otherwise (x 8: 77 against 94 us).
template <int NL, bool PADDED, bool MAIN>
__global__ void __launch_bounds__(kScanThreads, MAIN && NL == 2 ? 3 : 4) scan_fwd_kernel(const ScanArgs a) {
  constexpr int NP = 4 * NL;
  constexpr int GROUP = group_steps(NL), SAVE = save_every(NL);
  constexpr int PF = GROUP / NL;  // steps of a group whose inputs a lane loads
  __shared__ __align__(16) float bs[2][kTile * NP];
  __shared__ __align__(16) float cs[2][MAIN ? kTile * NP : 4];
  const Place<NL, kChan> at(a);
  const int64_t len = scan_length(a, at.b);
  const int64_t t0 = at.chunk * a.chunk, t_end = min(t0 + a.chunk, len);
  Lane<NL, kChan> ly(a.y, at, t0);
  if (MAIN && a.zero_rest) zero_rows(ly, at, a, t0, len);
  if (t0 >= len && t0 > 0) return;  // the first piece of an empty sequence hands h0 on
  if (!MAIN && t_end == len) return;  // nothing follows
  const int steps = (int)(t_end - t0);
  const int nv = a.states - 4 * at.q;  // of the four states, those below N
  f2 A[kChan][2], h[kChan][2];
  float bias[kChan], skip[kChan], total[kChan];
  Lane<NL, kChan> lu(a.u, at, t0), ld(a.delta, at, t0), lz(a.z, at, t0);
#pragma unroll
  for (int c = 0; c < kChan; ++c) {
    float av[4], hv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool on = k < nv;
      av[k] = on ? a.a[at.d[c] * a.a_d + (4 * at.q + k) * a.a_n] * kLog2e : kPastN;
      hv[k] = 0.0f;
      if (MAIN && on && a.chunks == 1 && a.h0.p)
        hv[k] = a.h0.p[at.b * a.h0.s0 + at.d[c] * a.h0.s1 + (4 * at.q + k) * a.h0.s2];
    }
    if (MAIN && a.chunks > 1)
      unpack(reinterpret_cast<const float4 *>(a.sum_h)[((at.b * a.chunks + at.chunk) * a.dim + at.d[c]) * NL + at.q], hv);
#pragma unroll
    for (int k = 0; k < 2; ++k) A[c][k] = pair(av[2 * k], av[2 * k + 1]), h[c][k] = pair(hv[2 * k], hv[2 * k + 1]);
    bias[c] = a.bias ? a.bias[at.d[c] * a.bias_s] : 0.0f;
    skip[c] = MAIN && a.d ? a.d[at.d[c] * a.d_s] : 0.0f;
    total[c] = 0.0f;
  }
  const bool gated = MAIN && a.z.p != nullptr;
  float ru[kChan][PF], rd[kChan][PF], rz[kChan][PF];
  // the inputs of steps base .. base + GROUP - 1, zeros past the end, and on to
  // the next
  auto fetch = [&](int base) {
    if (base + GROUP <= steps) {
#pragma unroll
      for (int c = 0; c < kChan; ++c)
#pragma unroll
        for (int i = 0; i < PF; ++i) {
          ru[c][i] = lu(c, i * NL);
          rd[c][i] = ld(c, i * NL);
          if (gated) rz[c][i] = lz(c, i * NL);
        }
    } else {
#pragma unroll
      for (int c = 0; c < kChan; ++c)
#pragma unroll
        for (int i = 0; i < PF; ++i) {
          const bool on = base + i * NL + at.q < steps;
          ru[c][i] = on ? lu(c, i * NL) : 0.0f;
          rd[c][i] = on ? ld(c, i * NL) : 0.0f;
          if (gated) rz[c][i] = on ? lz(c, i * NL) : 0.0f;
        }
    }
    lu.go(GROUP), ld.go(GROUP), lz.go(GROUP);
  };
  auto stage = [&](int buf, int64_t t) {
    stage_rows<NL, kTile>(bs[buf], a.b, a.vec_b, at.b, at.g, t, t_end, a.states);
    if (MAIN) stage_rows<NL, kTile>(cs[buf], a.c, a.vec_c, at.b, at.g, t, t_end, a.states);
    copy_commit();
  };
  // what the steps of the next group need, from the inputs that have arrived
  float s1[kChan][PF], su1[kChan][PF], y1[kChan][PF], w1[kChan][PF];
  auto prepare = [&]() {
#pragma unroll
    for (int c = 0; c < kChan; ++c)
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        const float raw = rd[c][i] + bias[c];
        float sig;
        s1[c][i] = a.softplus ? softplus(raw, &sig) : raw;
        su1[c][i] = s1[c][i] * ru[c][i];
        if (MAIN) y1[c][i] = skip[c] * ru[c][i], w1[c][i] = gated ? rz[c][i] * sigmoid(rz[c][i]) : 1.0f;
      }
  };
  const int64_t kept = (a.length + SAVE - 1) / SAVE;
  // the states kept before every SAVE-th step: [step / SAVE, local channel, q]
  ulonglong2 *keep = reinterpret_cast<ulonglong2 *>(a.saved) + ((at.b * kept + t0 / SAVE) * a.dim + at.first) * NL;
  // GROUP steps from `base` on, whose b and c rows start at bt and ct.  The
  // inputs of the next group are prepared meanwhile, those of the one after
  // it are on their way.
  auto group = [&](auto whole, int base, const float *bt, const float *ct) {
    constexpr bool FULL = decltype(whole)::value;
    float s[kChan][PF], su[kChan][PF], y0[kChan][PF], w[kChan][PF];
#pragma unroll
    for (int c = 0; c < kChan; ++c)
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        s[c][i] = s1[c][i], su[c][i] = su1[c][i];
        if (MAIN) y0[c][i] = y1[c][i], w[c][i] = w1[c][i];
        if (!MAIN && (FULL || base + i * NL + at.q < steps)) total[c] += s[c][i];
      }
    prepare();
    if (base + 2 * GROUP < steps) fetch(base + 2 * GROUP);
#pragma unroll
    for (int i = 0; i < PF; ++i) {
      float part[kChan][NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int t = i * NL + j;
        keep_order();
        float sj[kChan], suj[kChan];
#pragma unroll
        for (int c = 0; c < kChan; ++c) {
          sj[c] = __shfl_sync(0xffffffffu, s[c][i], j, NL);
          suj[c] = __shfl_sync(0xffffffffu, su[c][i], j, NL);
          part[c][j] = 0.0f;
        }
        if (FULL || base + t < steps) {
          if (MAIN && t % SAVE == 0 && a.saved) {
#pragma unroll
            for (int c = 0; c < kChan; ++c)
              if (at.live[c]) keep[(unsigned)(at.local[c] * NL + at.q)] = make_ulonglong2(h[c][0], h[c][1]);
            keep += a.dim * NL;
          }
          const ulonglong2 b = *reinterpret_cast<const ulonglong2 *>(bt + t * NP + 4 * at.q);
          const ulonglong2 cc = MAIN ? *reinterpret_cast<const ulonglong2 *>(ct + t * NP + 4 * at.q) : b;
#pragma unroll
          for (int c = 0; c < kChan; ++c) {
            const f2 sp = both(sj[c]), sup = both(suj[c]);
            f2 in0 = mul2(sup, b.x), in1 = mul2(sup, b.y);
            if (PADDED) {
              in0 = pair(nv > 0 ? lo(in0) : 0.0f, nv > 1 ? hi(in0) : 0.0f);
              in1 = pair(nv > 2 ? lo(in1) : 0.0f, nv > 3 ? hi(in1) : 0.0f);
            }
            h[c][0] = fma2(decay2(sp, A[c][0]), h[c][0], in0);
            h[c][1] = fma2(decay2(sp, A[c][1]), h[c][1], in1);
            if (MAIN) {
              const f2 y = fma2(h[c][1], cc.y, mul2(h[c][0], cc.x));
              part[c][j] = lo(y) + hi(y);
            }
          }
        }
      }
      if (MAIN) {
#pragma unroll
        for (int c = 0; c < kChan; ++c) {
          transpose_sum<NL>(part[c], at.q);
          if (at.live[c] && (FULL || base + i * NL + at.q < steps)) {
            ly(c, i * NL) = (part[c][0] + y0[c][i]) * w[c][i];
          }
        }
      }
    }
  };
  if (steps > 0) {
    stage(0, t0);
    fetch(0);
    prepare();
    fetch(GROUP);
  }
  int buf = 0;
  for (int tile = 0; tile < steps; tile += kTile, buf ^= 1) {
    if (tile + kTile < steps)
      stage(buf ^ 1, t0 + tile + kTile);
    else
      copy_commit();  // an empty group, so that the wait below counts alike
    copy_wait<1>();
    __syncthreads();
#pragma unroll 1
    for (int base = tile; base < min(tile + kTile, steps); base += GROUP) {
      const float *bt = &bs[buf][(base - tile) * NP], *ct = &cs[buf][MAIN ? (base - tile) * NP : 0];
      if (base + GROUP <= steps)
        group(std::true_type{}, base, bt, ct);
      else
        group(std::false_type{}, base, bt, ct);
      if (MAIN) ly.go(GROUP);
    }
    __syncthreads();  // this buffer is filled again in the next turn
  }
#pragma unroll
  for (int c = 0; c < kChan; ++c) {
    const float hv[4] = {lo(h[c][0]), hi(h[c][0]), lo(h[c][1]), hi(h[c][1])};
    if (MAIN) {
      if (a.h_last.p && at.live[c] && t_end == len) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < nv) a.h_last.p[at.b * a.h_last.s0 + at.d[c] * a.h_last.s1 + (4 * at.q + k) * a.h_last.s2] = hv[k];
      }
    } else {
#pragma unroll
      for (int o = 1; o < NL; o <<= 1) total[c] += __shfl_xor_sync(0xffffffffu, total[c], o);
      if (at.live[c]) {
        const int64_t i = (at.b * a.chunks + at.chunk) * a.dim + at.d[c];
        reinterpret_cast<float4 *>(a.sum_h)[i * NL + at.q] = make_float4(hv[0], hv[1], hv[2], hv[3]);
        if (at.q == 0) a.sum_dt[i] = total[c];
      }
    }
  }
}

// Joins the pieces: sum_h of a piece becomes the state it starts from (in
// reverse, the adjoint that reaches its end).
__global__ void __launch_bounds__(256) scan_combine_kernel(const ScanArgs a, int np, int reverse) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.batch * a.dim * np) return;
  const int n = (int)(i % np);
  const int64_t d = i / np % a.dim, b = i / np / a.dim;
  const int64_t len = scan_length(a, b);
  const int64_t used = max((int64_t)1, (len + a.chunk - 1) / a.chunk);
  const Op3 &first = reverse ? a.dh_last : a.h0;
  const bool on = n < a.states;
  const float A = on ? a.a[d * a.a_d + n * a.a_n] * kLog2e : kPastN;
  float h = on && first.p ? first.p[b * first.s0 + d * first.s1 + n * first.s2] : 0.0f;
  constexpr int U = 8;  // pieces whose sums are on their way together
  for (int64_t k0 = 0; k0 < used; k0 += U) {
    float own[U], dt[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t j = (b * a.chunks + (reverse ? used - 1 - k0 - k : k0 + k)) * a.dim + d;
      const bool summed = k0 + k + 1 < used;  // nothing follows the last
      own[k] = summed ? a.sum_h[j * np + n] : 0.0f;
      dt[k] = summed ? a.sum_dt[j] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (k0 + k >= used) break;
      a.sum_h[((b * a.chunks + (reverse ? used - 1 - k0 - k : k0 + k)) * a.dim + d) * np + n] = h;
      h = fmaf(ex2(dt[k] * A), h, own[k]);
    }
  }
}

constexpr int64_t kManyBlocks = 148 * 4;

// An operand of one token per row and its strides along up to three axes.
// They are 32-bit, and four times an index is, so that a stride times an index
// added to an address is one instruction; the host refuses larger ones.  at() is
// what a thread's rows share, row() adds the row's part.
struct Token {
  float *p;
  int s0, s1, s2;
  __device__ __forceinline__ static float *add(float *o, int i, int stride) {
    return reinterpret_cast<float *>(reinterpret_cast<char *>(o) + (int64_t)(4 * i) * stride);
  }
  __device__ __forceinline__ float *at(int j, int k) const { return add(add(p, j, s1), k, s2); }
  __device__ __forceinline__ float *row(float *o, int i) const { return add(o, i, s0); }
  __device__ __forceinline__ float *operator()(int i, int j) const { return row(add(p, j, s1), i); }
};

struct TokenArgs {
  Token state, state_out, b, c, a, u, delta, z, y, d, bias;
  const int *slots;
  int slots_s;
  int batch, rows, dim, per;
  int states, groups, softplus, zero_rest;
};

// Four states of one channel per thread, of R batch rows, R either 1 or the
// smaller of NL and 4.  Bound by the states' bytes: with R > 1 the decay rates
// are read once for R rows, R states are on their way at once, and what belongs
// to a row and channel alone (the step, the gate, y) is worked out by one of the
// NL lanes.  VEC: four states are one aligned load, and none is past N.  Measured
// on B200 for 128 x 4096 x 16: 18.5 us, 4.1 TB/s with what the L2 holds; one row per
// thread 33, indexes multiplied and shifted apart and unpaired arithmetic 22.5.
template <int NL, int R, bool VEC>
__global__ void __launch_bounds__(kScanThreads, 7) scan_step_kernel(const TokenArgs a) {
  const int i0 = (int)blockIdx.y * R;
  const int q = threadIdx.x % NL, d = (int)blockIdx.x * (kScanThreads / NL) + threadIdx.x / NL;
  int slot[R];
  bool on[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = i0 + r;
    slot[r] = i;
    on[r] = i < a.batch;
    if (a.slots != nullptr) {
      slot[r] = on[r] ? a.slots[(int64_t)i * a.slots_s] : -1;
      bool again = false;
      for (int k = threadIdx.x; k < i && on[r]; k += kScanThreads)
        again |= a.slots[(int64_t)k * a.slots_s] == slot[r];
      on[r] = !__syncthreads_or(again) && slot[r] >= 0 && slot[r] < a.rows;
    }
  }
  const int nv = d < a.dim ? a.states - 4 * q : 0;
  const int own = q % R;  // the row whose per-channel values this lane has
  bool mine = false;
#pragma unroll
  for (int r = 0; r < R; ++r) mine = r == own ? on[r] && d < a.dim : mine;
  f2 h[R][2], b[R][2], c[R][2], A[2] = {0, 0};
  auto get = [&](float *p, int stride, f2 (&v)[2]) {
    if (VEC) {
      const ulonglong2 w = *reinterpret_cast<const ulonglong2 *>(p);
      v[0] = w.x, v[1] = w.y;
    } else {
      float w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = k < nv ? *Token::add(p, k, stride) : 0.0f;
      v[0] = pair(w[0], w[1]), v[1] = pair(w[2], w[3]);
    }
  };
  {
    float *p = a.state.at(d, 4 * q);
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (on[r] && nv > 0) get(a.state.row(p, slot[r]), a.state.s2, h[r]);
  }
  float u = 0.0f, s = 0.0f, z = 0.0f, sig;
  if (mine) {
    u = *a.u(i0 + own, d);
    s = *a.delta(i0 + own, d);
    if (a.bias.p) s += *a.bias(0, d);
    if (a.z.p) z = *a.z(i0 + own, d);
  }
  if (nv > 0) get(a.a.at(d, 4 * q), a.a.s2, A);
  {
    const int g = a.groups > 1 ? (int)((unsigned)d / (unsigned)a.per) : 0;
    float *pb = a.b.row(a.b.at(g, 4 * q), i0), *pc = a.c.row(a.c.at(g, 4 * q), i0);
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (on[r] && nv > 0) {
        get(a.b.row(pb, r), a.b.s2, b[r]);
        get(a.c.row(pc, r), a.c.s2, c[r]);
      }
  }
  if (a.softplus) s = softplus(s, &sig);
  const float su = s * u;
  float part[R];
  A[0] = mul2(A[0], both(kLog2e)), A[1] = mul2(A[1], both(kLog2e));
  float *po = a.state_out.at(d, 4 * q);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const f2 sr = both(R > 1 ? __shfl_sync(0xffffffffu, s, r, NL) : s);
    const f2 sur = both(R > 1 ? __shfl_sync(0xffffffffu, su, r, NL) : su);
    part[r] = 0.0f;
    if (on[r] && nv > 0) {
      f2 v[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        v[k] = fma2(decay2(sr, A[k]), h[r][k], mul2(sur, b[r][k]));
        // past N: s u may not be finite
        if (!VEC) v[k] = pair(2 * k < nv ? lo(v[k]) : 0.0f, 2 * k + 1 < nv ? hi(v[k]) : 0.0f);
      }
      const f2 sum = fma2(v[1], c[r][1], mul2(v[0], c[r][0]));
      part[r] = lo(sum) + hi(sum);
      float *o = a.state_out.row(po, slot[r]);
      if (VEC) {
        *reinterpret_cast<ulonglong2 *>(o) = make_ulonglong2(v[0], v[1]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < nv) *Token::add(o, k, a.state_out.s2) = k & 1 ? hi(v[k / 2]) : lo(v[k / 2]);
      }
    }
  }
#pragma unroll
  for (int o = R; o < NL; o <<= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) part[r] += __shfl_xor_sync(0xffffffffu, part[r], o);
  transpose_sum<R>(part, own);
  if (mine && q < R) {
    float y = part[0];
    if (a.d.p) y = fmaf(*a.d(0, d), u, y);
    if (a.z.p) y *= z * sigmoid(z);
    *a.y(i0 + own, d) = y;
  } else if (a.zero_rest && !mine && d < a.dim && i0 + own < a.batch && q < R) {
    *a.y(i0 + own, d) = 0.0f;
  }
}

// ------------------------------------------------------------------ host --
// Rows that 16-byte copies can take: unit stride, a multiple of four states,
// every row 16-byte aligned.
bool vec_states(const DescView &v) {
  const int last = v.rank - 1;
  if (v.sizes[last] % 4 || v.strides[last] != 1 || (reinterpret_cast<uintptr_t>(v.data(4)) & 15)) return false;
  for (int d = 0; d < last; ++d)
    if (v.sizes[d] > 1 && (v.strides[d] & 3)) return false;
  return true;
}

// Pieces of the time axis: one when the channels alone give the device enough
// warps or when the axis is short, else as many as do, of at least 32 steps each.
// 2048 positions of 16 states, whole and in pieces: 128 blocks 266 and 221 us, 256
// 322 and 400, 320 425 and 504, 384 427 and 575, 448 533 and 684, 512 538 and 690.
// So the axis should stay whole from some 200 blocks on rather than from kCutBelow.
// Cutting costs two more launches: 2 x 96 x 300 x 16 takes 15.4 us a call uncut
// (13.6 on the device) and 20.2 (14.2) cut, 2 x 192 x 300 x 16 25.4 and 20.1; 2 x 64 x
// 600 x 4, where a lane has more of a step to itself, 21.5 (19.8) and 25.6 (19.4),
// 2 x 96 x 600 x 4 29.7 and 25.6.
constexpr int64_t cut_beyond(int nl) { return nl < 4 ? 64 : 96; }
void cut_time(int64_t batch, int64_t length, int64_t dim, int states, int groups, int64_t *chunks, int64_t *chunk) {
  const int nl = lanes_for(states);
  const int64_t per_block = block_channels(nl, kChan), per = dim / std::max(groups, 1);
  const int64_t blocks = std::max<int64_t>(1, batch * groups * ((per + per_block - 1) / per_block));
  int64_t n = 1;
  if (blocks < kCutBelow && length > cut_beyond(nl))
    n = std::max<int64_t>(1, std::min<int64_t>(kBlocks / blocks, length / 16));
  *chunk = std::max<int64_t>(kTile, ((length + n - 1) / n + kTile - 1) / kTile * kTile);
  *chunks = std::max<int64_t>(1, (length + *chunk - 1) / *chunk);
}

size_t scratch_for(int64_t batch, int64_t dim, int states, int64_t chunks) {
  if (chunks <= 1) return 0;
  return (size_t)(batch * chunks * dim) * (4 * lanes_for(states) + 4) * 4;
}

int check_sizes(int64_t batch, int64_t length, int64_t dim, int64_t states, int64_t groups, const char *what) {
  if (batch < 0 || length < 0 || dim < 0) return fail(REMORA_ERR_ARG, "%s: negative size", what);
  if (length > kMaxLength) return fail(REMORA_ERR_LIMIT, "%s: more than 2^30 positions", what);
  if (states < 1 || states > kMaxStates)
    return fail(REMORA_ERR_UNSUPPORTED, "%s: %lld states (1..%d)", what, (long long)states, kMaxStates);
  if (groups < 1 || dim % groups)
    return fail(REMORA_ERR_SHAPE, "%s: %lld channels in %lld groups", what, (long long)dim, (long long)groups);
  return REMORA_OK;
}

template <bool MAIN>
int launch_fwd(const ScanArgs &a, int nl, cudaStream_t stream) {
  const unsigned grid = (unsigned)(a.batch * a.chunks * a.groups * a.blocks_d);
  const bool padded = a.states != 4 * nl;
  note_launch();
#define REMORA_SCAN_CASE(NL)                                                            \
  case NL:                                                                              \
    if (padded)                                                                         \
      scan_fwd_kernel<NL, true, MAIN><<<grid, kScanThreads, 0, stream>>>(a);            \
    else                                                                                \
      scan_fwd_kernel<NL, false, MAIN><<<grid, kScanThreads, 0, stream>>>(a);           \
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

// Reads and checks the inputs; views: u, delta, a, b, c, d, z, delta_bias,
// h0, lengths, those not given with a null data pointer and rank 0.
int read_scan_in(const RemoraSelectiveScanSpec *spec, const RemoraSelectiveScanIn *in, ScanArgs *a, DescView views[10],
                 const char *what) {
  if (spec == nullptr || in == nullptr) return fail(REMORA_ERR_ARG, "%s: null spec or inputs", what);
  bool have[10];
  REMORA_TRY(read_f32(in->u, 3, &views[0], "selective_scan u"));
  REMORA_TRY(read_f32(in->delta, 3, &views[1], "selective_scan delta"));
  REMORA_TRY(read_f32(in->a, 2, &views[2], "selective_scan a"));
  REMORA_TRY(read_f32(in->b, 4, &views[3], "selective_scan b"));
  REMORA_TRY(read_f32(in->c, 4, &views[4], "selective_scan c"));
  REMORA_TRY(read_optional(in->d, 1, &views[5], &have[5], "selective_scan d"));
  REMORA_TRY(read_optional(in->z, 3, &views[6], &have[6], "selective_scan z"));
  REMORA_TRY(read_optional(in->delta_bias, 1, &views[7], &have[7], "selective_scan delta_bias"));
  REMORA_TRY(read_optional(in->h0, 3, &views[8], &have[8], "selective_scan h0"));
  REMORA_TRY(read_optional(in->lengths, 1, &views[9], &have[9], "selective_scan lengths"));
  const int64_t B = views[0].sizes[0], L = views[0].sizes[1], D = views[0].sizes[2];
  const int64_t N = views[2].sizes[1], G = views[3].sizes[2];
  REMORA_TRY(check_sizes(B, L, D, N, G, what));
  REMORA_TRY(want_shape(views[1], {B, L, D}, "selective_scan delta"));
  REMORA_TRY(want_shape(views[2], {D, N}, "selective_scan a"));
  REMORA_TRY(want_shape(views[3], {B, L, G, N}, "selective_scan b"));
  REMORA_TRY(want_shape(views[4], {B, L, G, N}, "selective_scan c"));
  if (have[5]) REMORA_TRY(want_shape(views[5], {D}, "selective_scan d"));
  if (have[6]) REMORA_TRY(want_shape(views[6], {B, L, D}, "selective_scan z"));
  if (have[7]) REMORA_TRY(want_shape(views[7], {D}, "selective_scan delta_bias"));
  if (have[8]) REMORA_TRY(want_shape(views[8], {B, D, N}, "selective_scan h0"));
  if (have[9]) REMORA_TRY(want_shape(views[9], {B}, "selective_scan lengths"));
  a->u = op3(views[0]), a->delta = op3(views[1]);
  a->a = reinterpret_cast<const float *>(views[2].data(4)), a->a_d = views[2].strides[0], a->a_n = views[2].strides[1];
  a->b = op4(views[3]), a->c = op4(views[4]);
  a->vec_b = vec_states(views[3]), a->vec_c = vec_states(views[4]);
  if (have[5]) a->d = reinterpret_cast<const float *>(views[5].data(4)), a->d_s = views[5].strides[0];
  if (have[6]) a->z = op3(views[6]);
  if (have[7]) a->bias = reinterpret_cast<const float *>(views[7].data(4)), a->bias_s = views[7].strides[0];
  if (have[8]) a->h0 = op3(views[8]);
  if (have[9]) a->lengths = reinterpret_cast<const int *>(views[9].data(4)), a->lengths_s = views[9].strides[0];
  a->batch = B, a->length = L, a->dim = D, a->states = (int)N, a->groups = (int)G, a->softplus = spec->softplus != 0;
  a->zero_rest = spec->zero_rest != 0;
  a->per = D / G;
  return REMORA_OK;
}

int combine_chunks(const ScanArgs &a, int nl, bool reverse, cudaStream_t stream) {
  const int64_t n = a.batch * a.dim * 4 * nl;
  note_launch();
  scan_combine_kernel<<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(a, 4 * nl, reverse ? 1 : 0);
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

}  // namespace seq
}  // namespace remora

using namespace remora;
using namespace remora::seq;

extern "C" {

int remora_b200_selective_scan_saved(int64_t batch, int64_t length, int64_t dim, int64_t states, size_t *bytes) {
  if (bytes == nullptr) return fail(REMORA_ERR_ARG, "selective_scan_saved: null pointer");
  REMORA_TRY(check_sizes(batch, length, dim, states, 1, "selective_scan_saved"));
  const int nl = lanes_for((int)states), every = save_every(nl);
  *bytes = (size_t)(batch * ((length + every - 1) / every) * dim) * (size_t)(4 * nl) * 4;
  return REMORA_OK;
}

int remora_b200_selective_scan_fwd_scratch(RemoraB200Ctx *ctx, int64_t batch, int64_t length, int64_t dim,
                                           int64_t states, int64_t groups, size_t *bytes) {
  if (ctx == nullptr || bytes == nullptr) return fail(REMORA_ERR_ARG, "selective_scan_fwd_scratch: null pointer");
  REMORA_TRY(check_sizes(batch, length, dim, states, groups, "selective_scan_fwd_scratch"));
  int64_t chunks, chunk;
  cut_time(batch, length, dim, (int)states, (int)groups, &chunks, &chunk);
  *bytes = scratch_for(batch, dim, (int)states, chunks);
  return REMORA_OK;
}

int remora_b200_selective_scan_fwd(RemoraB200Ctx *ctx, const RemoraSelectiveScanSpec *spec,
                                   const RemoraSelectiveScanIn *in, RemoraMemRef3 *y, RemoraMemRef3 *h_last,
                                   void *saved, size_t saved_bytes, void *scratch, size_t scratch_bytes,
                                   remora_stream_t stream_) {
  if (ctx == nullptr) return fail(REMORA_ERR_ARG, "null context");
  cudaStream_t stream = (cudaStream_t)stream_;
  ScanArgs a = {};
  DescView v[10], yv, hv;
  bool has_h;
  REMORA_TRY(read_scan_in(spec, in, &a, v, "selective_scan_fwd"));
  REMORA_TRY(read_f32(y, 3, &yv, "selective_scan y"));
  REMORA_TRY(read_optional(h_last, 3, &hv, &has_h, "selective_scan h_last"));
  REMORA_TRY(want_shape(yv, {a.batch, a.length, a.dim}, "selective_scan y"));
  const int nl = lanes_for(a.states);
  a.blocks_d = (a.per + block_channels(nl, kChan) - 1) / block_channels(nl, kChan);
  if (has_h) REMORA_TRY(want_shape(hv, {a.batch, a.dim, a.states}, "selective_scan h_last"));
  auto given = [&](int k) { return v[k].aligned != nullptr ? &v[k] : nullptr; };
  REMORA_TRY(want_apart({{&yv, "y", 4}, {has_h ? &hv : nullptr, "h_last", 4}},
                        {{given(0), "u", 4}, {given(1), "delta", 4}, {given(2), "a", 4}, {given(3), "b", 4},
                         {given(4), "c", 4}, {given(5), "d", 4}, {given(6), "z", 4}, {given(7), "delta_bias", 4},
                         {given(8), "h0", 4}, {given(9), "lengths", 4}}, {{&hv, &v[8]}}));
  REMORA_TRY(want_own_elements({{&yv, "y", 4}, {has_h ? &hv : nullptr, "h_last", 4}}));
  for (int k : {0, 1, 6})
    if (v[k].aligned) REMORA_TRY(check_reach(v[k], nl, kChan, a.per, "selective_scan_fwd"));
  REMORA_TRY(check_reach(yv, nl, kChan, a.per, "selective_scan_fwd"));
  a.y = op3(yv);
  if (has_h) a.h_last = op3(hv);
  cut_time(a.batch, a.length, a.dim, a.states, a.groups, &a.chunks, &a.chunk);
  if (saved != nullptr) {
    size_t need = 0;
    REMORA_TRY(remora_b200_selective_scan_saved(a.batch, a.length, a.dim, a.states, &need));
    REMORA_TRY(want_scratch(saved, saved_bytes, need, "selective_scan_fwd (saved)"));
    a.saved = static_cast<float *>(saved);
  }
  REMORA_TRY(want_scratch(scratch, scratch_bytes, scratch_for(a.batch, a.dim, a.states, a.chunks),
                          "selective_scan_fwd"));
  if (a.batch == 0 || a.dim == 0 || (a.length == 0 && !has_h)) return REMORA_OK;
  if (a.batch * a.chunks * a.groups * a.blocks_d > 0x7fffffff || a.batch * a.dim * 4 * nl / 256 > 0x7ffffffe)
    return fail(REMORA_ERR_LIMIT, "selective_scan_fwd: too many blocks");
  DeviceGuard guard;
  REMORA_TRY(guard.enter(ctx));
  if (a.chunks > 1) {
    a.sum_h = static_cast<float *>(scratch);
    a.sum_dt = a.sum_h + a.batch * a.chunks * a.dim * 4 * nl;
    REMORA_TRY(launch_fwd<false>(a, nl, stream));
    REMORA_TRY(combine_chunks(a, nl, false, stream));
  }
  return launch_fwd<true>(a, nl, stream);
}

int remora_b200_selective_scan_step(RemoraB200Ctx *ctx, const RemoraSelectiveScanSpec *spec,
                                    const RemoraSelectiveStepIn *in, RemoraMemRef2 *y, RemoraMemRef3 *state_out,
                                    remora_stream_t stream) {
  if (ctx == nullptr) return fail(REMORA_ERR_ARG, "null context");
  if (spec == nullptr || in == nullptr) return fail(REMORA_ERR_ARG, "selective_scan_step: null spec or inputs");
  DescView sv, uv, ev, av, bv, cv, dv, zv, iv, lv, yv, ov;
  bool has_d, has_z, has_i, has_l;
  REMORA_TRY(read_f32(in->state, 3, &sv, "selective_scan_step state"));
  REMORA_TRY(read_f32(in->u, 2, &uv, "selective_scan_step u"));
  REMORA_TRY(read_f32(in->delta, 2, &ev, "selective_scan_step delta"));
  REMORA_TRY(read_f32(in->a, 2, &av, "selective_scan_step a"));
  REMORA_TRY(read_f32(in->b, 3, &bv, "selective_scan_step b"));
  REMORA_TRY(read_f32(in->c, 3, &cv, "selective_scan_step c"));
  REMORA_TRY(read_optional(in->d, 1, &dv, &has_d, "selective_scan_step d"));
  REMORA_TRY(read_optional(in->z, 2, &zv, &has_z, "selective_scan_step z"));
  REMORA_TRY(read_optional(in->delta_bias, 1, &iv, &has_i, "selective_scan_step delta_bias"));
  REMORA_TRY(read_optional(in->slots, 1, &lv, &has_l, "selective_scan_step slots"));
  REMORA_TRY(read_f32(y, 2, &yv, "selective_scan_step y"));
  REMORA_TRY(read_f32(state_out, 3, &ov, "selective_scan_step state_out"));
  const int64_t B = uv.sizes[0], D = uv.sizes[1], N = av.sizes[1], G = bv.sizes[1], S = sv.sizes[0];
  REMORA_TRY(check_sizes(B, 1, D, N, G, "selective_scan_step"));
  REMORA_TRY(want_shape(ev, {B, D}, "selective_scan_step delta"));
  REMORA_TRY(want_shape(av, {D, N}, "selective_scan_step a"));
  REMORA_TRY(want_shape(bv, {B, G, N}, "selective_scan_step b"));
  REMORA_TRY(want_shape(cv, {B, G, N}, "selective_scan_step c"));
  REMORA_TRY(want_shape(sv, {S, D, N}, "selective_scan_step state"));
  REMORA_TRY(want_shape(ov, {S, D, N}, "selective_scan_step state_out"));
  REMORA_TRY(want_shape(yv, {B, D}, "selective_scan_step y"));
  if (has_d) REMORA_TRY(want_shape(dv, {D}, "selective_scan_step d"));
  if (has_z) REMORA_TRY(want_shape(zv, {B, D}, "selective_scan_step z"));
  if (has_i) REMORA_TRY(want_shape(iv, {D}, "selective_scan_step delta_bias"));
  if (has_l) REMORA_TRY(want_shape(lv, {B}, "selective_scan_step slots"));
  if (!has_l && B > S)
    return fail(REMORA_ERR_SHAPE, "selective_scan_step: %lld rows and %lld states", (long long)B, (long long)S);
  if (B > 65535) return fail(REMORA_ERR_LIMIT, "selective_scan_step: more than 65535 rows");
  REMORA_TRY(want_apart({{&yv, "y", 4}, {&ov, "state_out", 4}},
                        {{&sv, "state", 4}, {&uv, "u", 4}, {&ev, "delta", 4}, {&av, "a", 4}, {&bv, "b", 4},
                         {&cv, "c", 4}, {has_d ? &dv : nullptr, "d", 4}, {has_z ? &zv : nullptr, "z", 4},
                         {has_i ? &iv : nullptr, "delta_bias", 4}, {has_l ? &lv : nullptr, "slots", 4}}, {{&ov, &sv}}));
  REMORA_TRY(want_own_elements({{&yv, "y", 4}, {&ov, "state_out", 4}}));
  if (B == 0 || D == 0) return REMORA_OK;
  if (std::max(D, S) > 0x1fffffff)
    return fail(REMORA_ERR_LIMIT, "selective_scan_step: 2^29 channels or rows of state, or more");
  TokenArgs a = {};
  // each operand's place in Token: row, channel (or group), state
  struct {
    const DescView *v;
    int row, channel, state;
    Token *to;
  } const places[] = {{&sv, 0, 1, 2, &a.state}, {&ov, 0, 1, 2, &a.state_out}, {&bv, 0, 1, 2, &a.b}, {&cv, 0, 1, 2, &a.c},
                      {&av, -1, 0, 1, &a.a},    {&uv, 0, 1, -1, &a.u},        {&ev, 0, 1, -1, &a.delta},
                      {&yv, 0, 1, -1, &a.y},    {has_z ? &zv : nullptr, 0, 1, -1, &a.z},
                      {has_d ? &dv : nullptr, -1, 0, -1, &a.d}, {has_i ? &iv : nullptr, -1, 0, -1, &a.bias},
                      {has_l ? &lv : nullptr, 0, -1, -1, nullptr}};
  for (const auto &x : places) {
    if (x.v == nullptr) continue;
    for (int k = 0; k < x.v->rank; ++k)
      if (std::abs(stride_of(*x.v, k)) > 0x7fffffff)
        return fail(REMORA_ERR_LIMIT, "selective_scan_step: a stride of %lld elements (at most 2^31 - 1)",
                    (long long)x.v->strides[k]);
    auto stride = [&](int k) { return k < 0 ? 0 : (int)stride_of(*x.v, k); };
    if (x.to) *x.to = {reinterpret_cast<float *>(x.v->data(4)), stride(x.row), stride(x.channel), stride(x.state)};
  }
  if (has_l) a.slots = reinterpret_cast<const int *>(lv.data(4)), a.slots_s = (int)stride_of(lv, 0);
  a.batch = (int)B, a.rows = (int)S, a.dim = (int)D, a.per = (int)(D / G), a.states = (int)N, a.groups = (int)G;
  a.softplus = spec->softplus != 0, a.zero_rest = spec->zero_rest != 0;
  const bool vec = vec_states(sv) && vec_states(ov) && vec_states(av) && vec_states(bv) && vec_states(cv);
  const int nl = lanes_for(a.states);
  // several rows per thread once that leaves every SM some blocks
  const int64_t blocks = (D + kScanThreads / nl - 1) / (kScanThreads / nl);
  const int rows = nl < 4 ? nl : 4;
  const bool many = nl > 1 && blocks * (B / rows) >= kManyBlocks;
  const dim3 grid((unsigned)blocks, (unsigned)(many ? (B + rows - 1) / rows : B));
  DeviceGuard guard;
  REMORA_TRY(guard.enter(ctx));
  cudaStream_t s = (cudaStream_t)stream;
  note_launch();
#define REMORA_STEP_LAUNCH(NL, R)                                     \
  if (vec)                                                            \
    scan_step_kernel<NL, R, true><<<grid, kScanThreads, 0, s>>>(a);   \
  else                                                                \
    scan_step_kernel<NL, R, false><<<grid, kScanThreads, 0, s>>>(a);
#define REMORA_STEP_CASE(NL)                        \
  case NL:                                          \
    if (many) {                                     \
      REMORA_STEP_LAUNCH(NL, (NL < 4 ? NL : 4))     \
    } else {                                        \
      REMORA_STEP_LAUNCH(NL, 1)                     \
    }                                               \
    break;
  switch (nl) {
  case 1: REMORA_STEP_LAUNCH(1, 1) break;
    REMORA_STEP_CASE(2)
    REMORA_STEP_CASE(4)
    REMORA_STEP_CASE(8)
    REMORA_STEP_CASE(16)
  }
#undef REMORA_STEP_LAUNCH
#undef REMORA_STEP_CASE
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

}  // extern "C"
