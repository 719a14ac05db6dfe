// seq_scan_bwd.cu — gradients of the selective state space scan.
//
//   dp = dy silu(z);  dz = dy p silu'(z)
//   G_t[n] = c_t[n] dp_t + exp(s_{t+1} a[n]) G_{t+1}[n]          (adjoint of h_t)
//   dc_t[n] = sum_d dp h_t[n];  db_t[n] = sum_d G s u;  da[n] = sum_t G s (exp(s a) h_{t-1})[n]
//   du = s sum_n G b + d dp;  ds = sum_n G a (exp(s a) h_{t-1}) + u sum_n G b;  ddelta = ds f'(delta + bias)
//
// A thread walks time from the end in pieces of save_every steps.  For each it
// takes the state that the forward kept at the piece's start, runs the
// recurrence forward once, keeping exp(s a) h_{t-1} of every step in registers,
// then the adjoint backward (the decay's second exponential costs less there
// than the registers to keep it).  db and dc sum over the channels of a group:
// over a thread's channels, over a warp by way of shared memory, over a block
// through shared memory, over blocks by partial rows in scratch that a second
// kernel adds in block order.
//
// Bound by issue and latency: some 220 instructions per warp, step and pair of
// channels (8 states per thread), at 57 % of the issue slots, since the registers
// leave 8 to 16 warps per SM.  Measured on B200 for 4 x 2048 x 2048 x 16:
// 357 us, first pass of the adjoint 90, joins 23.  The sums over channels by
// shuffles: 414 us, with a state kept every eight steps 400; the steps' s, s u and dp
// from shared memory instead of shuffles 432; the next step's shuffles ahead of a
// step, the same time.
#include <algorithm>
#include <type_traits>

#include "seq_scan.cuh"

namespace remora {
namespace seq {
namespace {

constexpr int kWarps = kScanThreads / 32;
constexpr float kLn2 = 0.6931471805599453f;

constexpr int bwd_chan(int nl) { return nl > 8 || nl < 4 ? 1 : 2; }

// Channels of a thread, steps of a piece, steps whose b, c, db and dc are in
// shared memory together.
template <int NL>
struct Bwd {
  static constexpr int kChan = bwd_chan(NL);
  static constexpr int kPiece = save_every(NL);
  static constexpr int kTile = NL > 4 ? 16 : 32;
};

constexpr int64_t kBlocks = 148 * 16;  // blocks of a cut time axis
constexpr int64_t kCutBelow = 148 * 2;
// A shorter axis is not cut: 2 x 48 x 300 x 16 takes 31.1 us a call uncut (25.1 on the
// device) and 36.7 (26.2) cut, 2 x 64 x 300 x 16 35.2 (29.8) and 36.3 (27.2).
constexpr int64_t kCutBeyond = 48;

int64_t bwd_channels(int nl) { return kScanThreads / nl * bwd_chan(nl); }  // of a block

// The sums over a warp's channels: lanes of the same q.  Each lane leaves its four
// states of db and of dc in shared memory, and after kSteps steps each lane adds
// up four states of one step's db or dc over all channels (over a kParts-th of
// them, and the parts by shuffles).  Rows are kRow floats apart, so that eight
// lanes, which read 16 bytes each at once, meet 32 banks.
template <int NL>
struct ChannelSum {
  static constexpr int kSteps = 16 / NL < save_every(NL) ? 16 / NL : save_every(NL);
  static constexpr int kParts = 16 / (NL * kSteps);
  static constexpr int kEach = 32 / NL / kParts;
  static constexpr int kRow = 128 + 4 * NL % 32;
  static constexpr int kFloats = kSteps * 2 * kRow;
  float *to;          // where the lane leaves its states of step 0
  const float *from;  // the first of the values that it adds up
  int out;            // where their sum goes, from a step's row of db and dc
  bool stores;
  __device__ __forceinline__ ChannelSum(float *room, int lane) {
    const int q = lane % NL, which = lane / NL % 2, step = lane / (2 * NL) % kSteps, part = lane / (2 * NL * kSteps);
    to = room + 4 * lane;
    from = room + (step * 2 + which) * kRow + part * kEach * 4 * NL + 4 * q;
    out = (step * 2 + which) * 4 * NL + 4 * q;
    stores = part == 0;
  }
  __device__ __forceinline__ void put(int step, const f2 (&db)[2], const f2 (&dc)[2]) const {
    *reinterpret_cast<ulonglong2 *>(to + step * 2 * kRow) = make_ulonglong2(db[0], db[1]);
    *reinterpret_cast<ulonglong2 *>(to + (step * 2 + 1) * kRow) = make_ulonglong2(dc[0], dc[1]);
  }
  // all lanes of the warp, after the last put of kSteps steps
  __device__ __forceinline__ void add_up(float *row) const {
    __syncwarp();
    ulonglong2 sum = *reinterpret_cast<const ulonglong2 *>(from);
#pragma unroll
    for (int k = 1; k < kEach; ++k) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(from + k * 4 * NL);
      sum.x = add2(sum.x, v.x), sum.y = add2(sum.y, v.y);
    }
    __syncwarp();  // read, before the next step is put there
#pragma unroll
    for (int o = 16; o >= 2 * NL * kSteps; o >>= 1) {
      sum.x = add2(sum.x, __shfl_xor_sync(0xffffffffu, sum.x, o));
      sum.y = add2(sum.y, __shfl_xor_sync(0xffffffffu, sum.y, o));
    }
    if (stores) *reinterpret_cast<ulonglong2 *>(row + out) = sum;
  }
};

// Blocks of an SM that the registers are cut for.  4 x 2048 x 2048 x 16: 357 us with
// three and 363 with two; 4 x 2000 x 2000: x 8, 172 with four and 189 with three of
// two channels per thread; x 4, 147 with three and 153 with four.
constexpr int bwd_blocks(int nl) { return nl > 4 ? 2 : nl == 2 ? 4 : 3; }

template <int NL>
__global__ void __launch_bounds__(kScanThreads, bwd_blocks(NL)) scan_bwd_kernel(const ScanArgs a) {
  constexpr int NP = 4 * NL, C = Bwd<NL>::kChan, T = Bwd<NL>::kPiece, TILE = Bwd<NL>::kTile;
  constexpr int PF = T / NL;
  __shared__ __align__(16) float bs[2][TILE * NP], cs[2][TILE * NP];
  extern __shared__ __align__(16) float red[];  // [kWarps][TILE][2 NP]: per step db, dc; room for ChannelSum
  const Place<NL, C> at(a);
  const int warp = threadIdx.x >> 5;
  const ChannelSum<NL> over(red + kWarps * TILE * 2 * NP + warp * ChannelSum<NL>::kFloats, threadIdx.x & 31);
  const int64_t len = scan_length(a, at.b);
  const int64_t t0 = at.chunk * a.chunk, t_end = min(t0 + a.chunk, len);
  const int steps = t_end > t0 ? (int)(t_end - t0) : 0;
  const int64_t prow = at.b * a.chunks + at.chunk;
  const int64_t kept = (a.length + T - 1) / T;
  const int nv = a.states - 4 * at.q;
  f2 A[C][2], G[C][2], dA[C][2];
  float bias[C], skip[C], sum_d[C], sum_bias[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float av[4], gv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool on = at.live[c] && k < nv;
      av[k] = on ? a.a[at.d[c] * a.a_d + (4 * at.q + k) * a.a_n] * kLog2e : kPastN;
      gv[k] = 0.0f;
      if (on && a.chunks == 1 && a.dh_last.p)
        gv[k] = a.dh_last.p[at.b * a.dh_last.s0 + at.d[c] * a.dh_last.s1 + (4 * at.q + k) * a.dh_last.s2];
    }
    if (a.chunks > 1 && at.live[c] && (t0 < len || t0 == 0))
      unpack(reinterpret_cast<const float4 *>(a.sum_h)[(prow * a.dim + at.d[c]) * NL + at.q], gv);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      A[c][k] = pair(av[2 * k], av[2 * k + 1]);
      G[c][k] = pair(gv[2 * k], gv[2 * k + 1]);
      dA[c][k] = 0;
    }
    bias[c] = a.bias ? a.bias[at.d[c] * a.bias_s] : 0.0f;
    skip[c] = a.d ? a.d[at.d[c] * a.d_s] : 0.0f;
    sum_d[c] = sum_bias[c] = 0.0f;
  }
  const bool gated = a.z.p != nullptr;
  float ru[C][PF], rd[C][PF], rz[C][PF], ry[C][PF];
  ulonglong2 rh[C];
  Lane<NL, C> lu(a.u, at, t0), ld(a.delta, at, t0), lz(a.z, at, t0), ly(a.dy, at, t0);
  Lane<NL, C> ldu(a.du, at, t0), ldd(a.ddelta, at, t0), ldz(a.dz, at, t0);
  if (a.zero_rest) {
    zero_rows(ldu, at, a, t0, len);
    zero_rows(ldd, at, a, t0, len);
    if (a.dz.p) zero_rows(ldz, at, a, t0, len);
    if (a.blocks_d == 1) {  // else by join_kernel
      const int64_t from = max(t0, len), rows = min(t0 + a.chunk, a.length) - from;
      for (int64_t i = threadIdx.x; i < rows * a.states; i += kScanThreads) {
        const int64_t t = from + i / a.states, n = i % a.states;
        a.db.p[at.b * a.db.s0 + t * a.db.s1 + at.g * a.db.s2 + n * a.db.s3] = 0.0f;
        a.dc.p[at.b * a.dc.s0 + t * a.dc.s1 + at.g * a.dc.s2 + n * a.dc.s3] = 0.0f;
      }
    }
  }
  // the states kept at the pieces' starts: [piece, local channel, q]
  const ulonglong2 *hp = reinterpret_cast<const ulonglong2 *>(a.saved) +
                         ((at.b * kept + t0 / T) * a.dim + at.first) * NL;
  const int64_t hstep = a.dim * NL;
  // the inputs of the piece from `base` on, zeros past the end, and back to the
  // piece before it
  auto fetch = [&](int base) {
    const bool full = base + T <= steps;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        const bool on = full || base + i * NL + at.q < steps;
        ru[c][i] = on ? lu(c, i * NL) : 0.0f;
        rd[c][i] = on ? ld(c, i * NL) : 0.0f;
        ry[c][i] = on ? ly(c, i * NL) : 0.0f;
        rz[c][i] = gated && on ? lz(c, i * NL) : 0.0f;
      }
      rh[c] = hp[(unsigned)(at.local[c] * NL + at.q)];
    }
    lu.go(-T), ld.go(-T), ly.go(-T), lz.go(-T);
    hp -= hstep;
  };
  auto stage = [&](int buf, int tile) {
    stage_rows<NL, TILE>(bs[buf], a.b, a.vec_b, at.b, at.g, t0 + tile, t_end, a.states);
    stage_rows<NL, TILE>(cs[buf], a.c, a.vec_c, at.b, at.g, t0 + tile, t_end, a.states);
    copy_commit();
  };
  // the piece from `base` on; its rows of b, c and red start at bt, ct, rt
  auto piece = [&](auto whole, int base, const float *bt, const float *ct, float *rt) {
    constexpr bool FULL = decltype(whole)::value;
    float s[C][PF], sig[C][PF], su[C][PF], u[C][PF], dyp[C][PF], dzf[C][PF];
    f2 h[C][2], eh[T][C][2];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      h[c][0] = rh[c].x, h[c][1] = rh[c].y;
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        const float raw = rd[c][i] + bias[c];
        sig[c][i] = 1.0f;
        s[c][i] = a.softplus ? softplus(raw, &sig[c][i]) : raw;
        u[c][i] = ru[c][i];
        su[c][i] = s[c][i] * u[c][i];
        dyp[c][i] = ry[c][i];
        dzf[c][i] = 0.0f;
        if (gated) {
          const float sz = sigmoid(rz[c][i]);
          dyp[c][i] = ry[c][i] * (rz[c][i] * sz);
          dzf[c][i] = ry[c][i] * (sz * fmaf(rz[c][i], 1.0f - sz, 1.0f));
        }
      }
    }
    if (!at.whole) {  // dead channels must add nothing to the sums over channels
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (at.live[c]) continue;
        h[c][0] = h[c][1] = 0;
#pragma unroll
        for (int i = 0; i < PF; ++i) s[c][i] = su[c][i] = dyp[c][i] = 0.0f;
      }
    }
    if (base >= T) fetch(base - T);
#pragma unroll
    for (int i = 0; i < PF; ++i) {
      float part[C][NL];
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int t = i * NL + j;
        keep_order();
        float sj[C], suj[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          sj[c] = __shfl_sync(0xffffffffu, s[c][i], j, NL);
          suj[c] = __shfl_sync(0xffffffffu, su[c][i], j, NL);
          part[c][j] = 0.0f;
        }
        if (FULL || base + t < steps) {
          const ulonglong2 b = *reinterpret_cast<const ulonglong2 *>(bt + t * NP + 4 * at.q);
          const ulonglong2 cc = *reinterpret_cast<const ulonglong2 *>(ct + t * NP + 4 * at.q);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const f2 sp = both(sj[c]), sup = both(suj[c]);
            eh[t][c][0] = mul2(decay2(sp, A[c][0]), h[c][0]);
            eh[t][c][1] = mul2(decay2(sp, A[c][1]), h[c][1]);
            h[c][0] = fma2(sup, b.x, eh[t][c][0]);
            h[c][1] = fma2(sup, b.y, eh[t][c][1]);
            const f2 y = fma2(h[c][1], cc.y, mul2(h[c][0], cc.x));
            part[c][j] = lo(y) + hi(y);
          }
        }
      }
      if (a.dz.p) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          transpose_sum<NL>(part[c], at.q);
          if (at.live[c] && (FULL || base + i * NL + at.q < steps))
            ldz(c, i * NL) = dzf[c][i] * fmaf(skip[c], u[c][i], part[c][0]);
        }
      }
    }
    // a piece's share of da on its own: long sums in parts
    f2 da[C][2];
#pragma unroll
    for (int c = 0; c < C; ++c) da[c][0] = da[c][1] = 0;
#pragma unroll
    for (int i = PF - 1; i >= 0; --i) {
      float gb[C][NL], ga[C][NL];
#pragma unroll
      for (int j = NL - 1; j >= 0; --j) {
        const int t = i * NL + j;
        keep_order();
        float sj[C], suj[C], dj[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
          sj[c] = __shfl_sync(0xffffffffu, s[c][i], j, NL);
          suj[c] = __shfl_sync(0xffffffffu, su[c][i], j, NL);
          dj[c] = __shfl_sync(0xffffffffu, dyp[c][i], j, NL);
          gb[c][j] = ga[c][j] = 0.0f;
        }
        if (FULL || base + t < steps) {
          const ulonglong2 b = *reinterpret_cast<const ulonglong2 *>(bt + t * NP + 4 * at.q);
          const ulonglong2 cc = *reinterpret_cast<const ulonglong2 *>(ct + t * NP + 4 * at.q);
          f2 db[2], dc[2];
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const f2 sp = both(sj[c]), sup = both(suj[c]), djp = both(dj[c]);
            f2 g2, a2;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const f2 bk = k ? b.y : b.x, ck = k ? cc.y : cc.x, x = eh[t][c][k];
              const f2 hk = fma2(sup, bk, x);
              G[c][k] = fma2(ck, djp, G[c][k]);
              db[k] = c ? fma2(G[c][k], sup, db[k]) : mul2(G[c][k], sup);
              dc[k] = c ? fma2(hk, djp, dc[k]) : mul2(hk, djp);
              const f2 gx = mul2(G[c][k], x);
              g2 = k ? fma2(G[c][k], bk, g2) : mul2(G[c][k], bk);
              a2 = k ? fma2(gx, A[c][k], a2) : mul2(gx, A[c][k]);
              da[c][k] = fma2(gx, sp, da[c][k]);
              G[c][k] = mul2(G[c][k], decay2(sp, A[c][k]));
            }
            gb[c][j] = lo(g2) + hi(g2);
            ga[c][j] = lo(a2) + hi(a2);
          }
          over.put(t % over.kSteps, db, dc);
          if (t % over.kSteps == 0) over.add_up(rt + t * 2 * NP);
        }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        transpose_sum<NL>(gb[c], at.q);
        transpose_sum<NL>(ga[c], at.q);
        if (at.live[c] && (FULL || base + i * NL + at.q < steps)) {
          // A is a log2(e): its log2(e) comes off the sum here
          const float ds = fmaf(u[c][i], gb[c][0], ga[c][0] * kLn2) * sig[c][i];
          ldu(c, i * NL) = fmaf(s[c][i], gb[c][0], skip[c] * dyp[c][i]);
          ldd(c, i * NL) = ds;
          sum_d[c] = fmaf(dyp[c][i], u[c][i], sum_d[c]);
          sum_bias[c] += ds;
        }
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int k = 0; k < 2; ++k) dA[c][k] = add2(dA[c][k], da[c][k]);
    ldu.go(-T), ldd.go(-T), ldz.go(-T);
  };
  // In a tile's join a thread has one column, jf (state jn of db or dc), and every
  // JROWS-th step.
  constexpr int JROWS = kScanThreads / (2 * NP);
  const int jf = threadIdx.x % (2 * NP), jt = threadIdx.x / (2 * NP), jn = jf % NP;
  const bool jc = jf >= NP;
  const Op4 &jo = jc ? a.dc : a.db;
  const int64_t jstep = a.blocks_d == 1 ? jo.s1 : (int64_t)a.groups * 2 * a.states;
  float *jp = a.blocks_d == 1
                  ? jo.p + (at.b * jo.s0 + t0 * jo.s1 + at.g * jo.s2 + jn * jo.s3)
                  : a.part_bc + ((((at.bd * a.batch + at.b) * a.length + t0) * a.groups + at.g) * 2 + jc) * a.states + jn;
  const int last = steps > 0 ? (steps - 1) / TILE * TILE : -TILE;
  if (steps > 0) {
    const int end = (steps - 1) / T * T;
    lu.go(end), ld.go(end), ly.go(end), lz.go(end), ldu.go(end), ldd.go(end), ldz.go(end);
    hp += end / T * hstep;
    stage(0, last);
    fetch(end);
  }
  int buf = 0;
  for (int tile = last; tile >= 0; tile -= TILE, buf ^= 1) {
    if (tile > 0)
      stage(buf ^ 1, tile - TILE);
    else
      copy_commit();  // an empty group, so that the wait below counts alike
    copy_wait<1>();
    __syncthreads();  // b and c are there; red of the turn before is read
    float *rows = red + warp * TILE * 2 * NP;
#pragma unroll 1
    for (int base = (min(tile + TILE, steps) - 1) / T * T; base >= tile; base -= T) {
      const int off = (base - tile) * NP;
      if (base + T <= steps)
        piece(std::true_type{}, base, bs[buf] + off, cs[buf] + off, rows + 2 * off);
      else
        piece(std::false_type{}, base, bs[buf] + off, cs[buf] + off, rows + 2 * off);
    }
    __syncthreads();
    // join the warps; a row of part_bc is one channel block's share
    if (jn < a.states) {
#pragma unroll 4
      for (int t = jt; t < TILE && tile + t < steps; t += JROWS) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += red[w * TILE * 2 * NP + t * 2 * NP + jf];
        jp[(tile + t) * jstep] = v;
      }
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int o = 1; o < NL; o <<= 1) {
      sum_d[c] += __shfl_xor_sync(0xffffffffu, sum_d[c], o);
      sum_bias[c] += __shfl_xor_sync(0xffffffffu, sum_bias[c], o);
    }
    if (!at.live[c]) continue;
    const float gv[4] = {lo(G[c][0]), hi(G[c][0]), lo(G[c][1]), hi(G[c][1])};
    const float dv[4] = {lo(dA[c][0]), hi(dA[c][0]), lo(dA[c][1]), hi(dA[c][1])};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < nv) {
        if (a.dh0.p && t0 == 0) a.dh0.p[at.b * a.dh0.s0 + at.d[c] * a.dh0.s1 + (4 * at.q + k) * a.dh0.s2] = gv[k];
        a.part_a[(prow * a.dim + at.d[c]) * a.states + 4 * at.q + k] = dv[k];
      }
    if (at.q == 0) {
      a.part_d[prow * 2 * a.dim + at.d[c]] = sum_d[c];
      a.part_d[(prow * 2 + 1) * a.dim + at.d[c]] = sum_bias[c];
    }
  }
}

// First pass of a cut time axis: the adjoint that leaves a piece of it at its
// start when none enters at its end, and the piece's sum of steps.
template <int NL>
__global__ void __launch_bounds__(kScanThreads, 4) scan_adjoint_kernel(const ScanArgs a) {
  constexpr int NP = 4 * NL, C = Bwd<NL>::kChan, T = group_steps(NL), TILE = Bwd<NL>::kTile;
  constexpr int PF = T / NL;
  __shared__ __align__(16) float cs[2][TILE * NP];
  const Place<NL, C> at(a);
  const int64_t len = scan_length(a, at.b);
  const int64_t t0 = at.chunk * a.chunk, t_end = min(t0 + a.chunk, len);
  if (t0 == 0 || t0 >= len) return;  // nothing lies ahead of the first
  const int steps = (int)(t_end - t0);
  const int nv = a.states - 4 * at.q;
  f2 A[C][2], G[C][2];
  float bias[C], total[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float av[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      av[k] = k < nv ? a.a[at.d[c] * a.a_d + (4 * at.q + k) * a.a_n] * kLog2e : kPastN;
#pragma unroll
    for (int k = 0; k < 2; ++k) A[c][k] = pair(av[2 * k], av[2 * k + 1]), G[c][k] = 0;
    bias[c] = a.bias ? a.bias[at.d[c] * a.bias_s] : 0.0f;
    total[c] = 0.0f;
  }
  const bool gated = a.z.p != nullptr;
  float rd[C][PF], rz[C][PF], ry[C][PF];
  Lane<NL, C> ld(a.delta, at, t0), lz(a.z, at, t0), ly(a.dy, at, t0);
  auto fetch = [&](int base) {
    const bool full = base + T <= steps;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        const bool on = full || base + i * NL + at.q < steps;
        rd[c][i] = on ? ld(c, i * NL) : 0.0f;
        ry[c][i] = on ? ly(c, i * NL) : 0.0f;
        rz[c][i] = gated && on ? lz(c, i * NL) : 0.0f;
      }
    ld.go(-T), ly.go(-T), lz.go(-T);
  };
  auto stage = [&](int buf, int tile) {
    stage_rows<NL, TILE>(cs[buf], a.c, a.vec_c, at.b, at.g, t0 + tile, t_end, a.states);
    copy_commit();
  };
  auto piece = [&](auto whole, int base, const float *ct) {
    constexpr bool FULL = decltype(whole)::value;
    float s[C][PF], dyp[C][PF];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        const float raw = rd[c][i] + bias[c];
        float sig;
        s[c][i] = a.softplus ? softplus(raw, &sig) : raw;
        dyp[c][i] = gated ? ry[c][i] * (rz[c][i] * sigmoid(rz[c][i])) : ry[c][i];
        if (FULL || base + i * NL + at.q < steps) total[c] += s[c][i];
      }
    if (base >= T) fetch(base - T);
#pragma unroll
    for (int t = T - 1; t >= 0; --t) {
      keep_order();
      float sj[C], dj[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        sj[c] = __shfl_sync(0xffffffffu, s[c][t / NL], t % NL, NL);
        dj[c] = __shfl_sync(0xffffffffu, dyp[c][t / NL], t % NL, NL);
      }
      if (FULL || base + t < steps) {
        const ulonglong2 cc = *reinterpret_cast<const ulonglong2 *>(ct + t * NP + 4 * at.q);
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const f2 sp = both(sj[c]), djp = both(dj[c]);
          G[c][0] = mul2(fma2(cc.x, djp, G[c][0]), decay2(sp, A[c][0]));
          G[c][1] = mul2(fma2(cc.y, djp, G[c][1]), decay2(sp, A[c][1]));
        }
      }
    }
  };
  const int last = (steps - 1) / TILE * TILE;
  const int end = (steps - 1) / T * T;
  ld.go(end), ly.go(end), lz.go(end);
  stage(0, last);
  fetch(end);
  int buf = 0;
  for (int tile = last; tile >= 0; tile -= TILE, buf ^= 1) {
    if (tile > 0)
      stage(buf ^ 1, tile - TILE);
    else
      copy_commit();
    copy_wait<1>();
    __syncthreads();
#pragma unroll 1
    for (int base = (min(tile + TILE, steps) - 1) / T * T; base >= tile; base -= T) {
      if (base + T <= steps)
        piece(std::true_type{}, base, cs[buf] + (base - tile) * NP);
      else
        piece(std::false_type{}, base, cs[buf] + (base - tile) * NP);
    }
    __syncthreads();
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int o = 1; o < NL; o <<= 1) total[c] += __shfl_xor_sync(0xffffffffu, total[c], o);
    if (!at.live[c]) continue;
    const int64_t i = (at.b * a.chunks + at.chunk) * a.dim + at.d[c];
    reinterpret_cast<ulonglong2 *>(a.sum_h)[i * NL + at.q] = make_ulonglong2(G[c][0], G[c][1]);
    if (at.q == 0) a.sum_dt[i] = total[c];
  }
}

// db and dc of one position, group and state: the channel blocks' shares.
__device__ __forceinline__ void join_bc(const ScanArgs &a, int64_t i) {
  const int64_t plane = a.batch * a.length * a.groups * a.states;
  if (i >= plane) return;
  const int64_t n = i % a.states, g = i / a.states % a.groups, bt = i / a.states / a.groups;
  const int64_t t = bt % a.length, b = bt / a.length;
  const bool rest = t >= scan_length(a, b);
  if (rest && !a.zero_rest) return;
  const float *p = a.part_bc + (bt * a.groups + g) * 2 * a.states + n;
  float vb = 0.0f, vc = 0.0f;
#pragma unroll 8
  for (int64_t k = 0; k < a.blocks_d; ++k, p += 2 * plane) {
    vb += p[0];
    vc += p[a.states];
  }
  if (rest) vb = vc = 0.0f;  // their shares were never written
  a.db.p[b * a.db.s0 + t * a.db.s1 + g * a.db.s2 + n * a.db.s3] = vb;
  a.dc.p[b * a.dc.s0 + t * a.dc.s1 + g * a.dc.s2 + n * a.dc.s3] = vc;
}

// The rows of the partial sums and where their columns go.
struct Joins {
  int64_t rows;
  Columns a, d;
  unsigned blocks_a, blocks_d;  // the first blocks of the grid; the others join db and dc
};

// All sums that are left: of da, of dd and ddelta_bias over the pieces of time and
// the batch, of db and dc over the channel blocks.  In one launch: as three, 3 x 509
// x 388 x 13 took 6 us more.
template <int Y>
__global__ void __launch_bounds__(32 * Y) join_kernel(const ScanArgs a, const Joins j) {
  __shared__ float t[Y][33];
  const int x = threadIdx.x % 32, y = threadIdx.x / 32;
  unsigned block = blockIdx.x;
  if (block < j.blocks_a) return reduce_columns<Y>(a.part_a, j.rows, a.dim * a.states, j.a, block, x, y, t);
  block -= j.blocks_a;
  if (block < j.blocks_d) return reduce_columns<Y>(a.part_d, j.rows, 2 * a.dim, j.d, block, x, y, t);
  join_bc(a, (int64_t)(block - j.blocks_d) * (32 * Y) + threadIdx.x);
}

// ------------------------------------------------------------------ host --
// As the forward's: pieces only where the channels give too few warps.  Training
// steps of 2048 positions and 16 states with the backward's axis whole and in pieces,
// the forward alike on both sides: 128 blocks 986 and 717 us, 256 1371 and 1323, 320
// 1751 and 1649, 384 1828 and 1942, 448 2423 and 2148, 512 2428 and 2289, 768 3268 and
// 3408, 1024 3970 and 4180.  444 blocks fit the device at once: a whole axis wins
// where they fill their last round, which kCutBelow alone does not tell.
void cut_time(int64_t batch, int64_t length, int64_t dim, int nl, int64_t groups, int64_t *chunks, int64_t *chunk) {
  const int64_t per_block = bwd_channels(nl), per = dim / std::max<int64_t>(groups, 1);
  const int64_t blocks = std::max<int64_t>(1, batch * groups * ((per + per_block - 1) / per_block));
  int64_t n = 1;
  if (blocks < kCutBelow && length > kCutBeyond)
    n = std::max<int64_t>(1, std::min<int64_t>(kBlocks / blocks, length / 16));
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
  const int64_t per_block = bwd_channels(nl), per = dim / std::max<int64_t>(groups, 1);
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

template <int NL>
int launch_one(const ScanArgs &a, bool adjoint, cudaStream_t stream) {
  const unsigned grid = (unsigned)(a.batch * a.chunks * a.groups * a.blocks_d);
  note_launch();
  if (adjoint) {
    scan_adjoint_kernel<NL><<<grid, kScanThreads, 0, stream>>>(a);
  } else {
    constexpr int kRed = kWarps * (Bwd<NL>::kTile * 8 * NL + ChannelSum<NL>::kFloats) * 4;
    constexpr int kStatic = 4 * Bwd<NL>::kTile * 4 * NL * 4;
    if (kRed + kStatic > 48 * 1024)
      REMORA_CUDA_TRY(cudaFuncSetAttribute(scan_bwd_kernel<NL>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRed));
    scan_bwd_kernel<NL><<<grid, kScanThreads, kRed, stream>>>(a);
  }
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

int launch_bwd(const ScanArgs &a, int nl, bool adjoint, cudaStream_t stream) {
  switch (nl) {
  case 1: return launch_one<1>(a, adjoint, stream);
  case 2: return launch_one<2>(a, adjoint, stream);
  case 4: return launch_one<4>(a, adjoint, stream);
  case 8: return launch_one<8>(a, adjoint, stream);
  default: return launch_one<16>(a, adjoint, stream);
  }
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
  const int nl = lanes_for(a.states);
  a.blocks_d = (a.per + bwd_channels(nl) - 1) / bwd_channels(nl);
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
  for (int k = 0; k < 9; ++k) REMORA_TRY(want_own_elements({{out(k), "a gradient", 4}}));
  const Layout l = layout_for(B, L, D, a.states, G);
  size_t need = 0;
  REMORA_TRY(remora_b200_selective_scan_saved(B, L, D, N, &need));
  REMORA_TRY(want_scratch(saved, saved_bytes, need, "selective_scan_bwd (saved)"));
  REMORA_TRY(want_scratch(scratch, scratch_bytes, l.total * 4, "selective_scan_bwd"));
  const int chan = bwd_chan(nl);
  for (int k : {0, 1, 6})
    if (v[k].aligned) REMORA_TRY(check_reach(v[k], nl, chan, a.per, "selective_scan_bwd"));
  for (const DescView *x : {&gy, &o[0], &o[1], have[6] ? &o[6] : &o[0]})
    REMORA_TRY(check_reach(*x, nl, chan, a.per, "selective_scan_bwd"));
  a.dy = op3(gy);
  if (has_gh) a.dh_last = op3(gh);
  a.du = op3(o[0]), a.ddelta = op3(o[1]);
  a.db = op4(o[3]), a.dc = op4(o[4]);
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
  if (B > 0 && D > 0) {
    if (a.chunks > 1) {
      REMORA_TRY(launch_bwd(a, nl, true, stream));
      REMORA_TRY(combine_chunks(a, nl, true, stream));
    }
    REMORA_TRY(launch_bwd(a, nl, false, stream));
  }
  Joins j = {B * a.chunks};
  j.a = {reinterpret_cast<float *>(o[2].data(4)), N, o[2].strides[0], o[2].strides[1], D * N, nullptr, 0};
  j.d = {have[5] ? reinterpret_cast<float *>(o[5].data(4)) : nullptr, D, 0, have[5] ? o[5].strides[0] : 0, D,
         have[7] ? reinterpret_cast<float *>(o[7].data(4)) : nullptr, have[7] ? o[7].strides[0] : 0};
  const bool wide = tall(j.rows);
  const int threads = wide ? 1024 : 256;
  j.blocks_a = (unsigned)((D * N + 31) / 32);
  j.blocks_d = have[5] || have[7] ? (unsigned)((2 * D + 31) / 32) : 0;
  // without channels db and dc are zeros
  const unsigned blocks =
      j.blocks_a + j.blocks_d + (a.blocks_d != 1 ? (unsigned)((B * L * G * N + threads - 1) / threads) : 0);
  if (blocks == 0) return REMORA_OK;
  note_launch();
  if (wide)
    join_kernel<32><<<blocks, threads, 0, stream>>>(a, j);
  else
    join_kernel<8><<<blocks, threads, 0, stream>>>(a, j);
  REMORA_CUDA_TRY(cudaGetLastError());
  return REMORA_OK;
}

}  // extern "C"
