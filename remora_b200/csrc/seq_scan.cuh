// seq_scan.cuh — what the forward (seq_scan.cu) and backward
// (seq_scan_bwd.cu) selective scans share: the operands as the kernels see
// them, the mapping of channels and states to threads, and the staging of b
// and c in shared memory.
//
// Mapping.  A channel's N states are spread over NL neighbouring lanes of a
// warp, four states each (NP = 4 NL >= N, the states past N are zero).  A
// thread holds kChan channels, 32 / NL apart, so a warp works on 32 kChan / NL:
// b and c of a step, which all channels read from shared memory, cost one
// clock of the SM's shared-memory pipe per register that they fill, and are
// used kChan times.  Time runs serially in a thread.  The per-channel inputs
// are loaded by the lane that a step falls to (lane q of a channel takes steps
// q, q + NL, ...) and broadcast by shuffle; sums over the states go back to
// that lane by a transposed (reduce-scatter) shuffle, so every per-channel
// value is loaded, transformed and stored once.  State arithmetic is done on
// pairs of states (f32x2 instructions, each half rounded as the scalar form).
#pragma once

#include "seq.cuh"

namespace remora {
namespace seq {

constexpr int kScanThreads = 128;
// Steps whose inputs are loaded together.
constexpr int group_steps(int nl) { return nl > 8 ? 16 : nl > 1 ? 8 : 4; }
// Steps between the states that the forward keeps for the backward pass, whose
// threads hold as many in registers: a multiple of nl.  Four instead of eight
// lets three blocks live on an SM instead of two (4 x 2048 x 2048 x 16: 357
// against 400 us) and costs a write and a read of a state twice as often.
constexpr int save_every(int nl) { return nl > 8 ? 16 : nl > 4 ? 8 : 4; }
constexpr int kMaxStates = 64;
constexpr int64_t kMaxLength = 1 << 30;
constexpr int kChan = 2;  // channels per thread
// a of the states past N: their decay is 0 for a step that is inf, where a = 0
// would make it, and through the sums over the states every output, NaN; and it is
// finite for every finite step, of either sign.
constexpr float kPastN = -1.17549435e-38f;

struct Op3 {  // [B, time, D], or [B, D, N]
  float *p;
  int64_t s0, s1, s2;
};

struct Op4 {  // [B, time, G, N]
  float *p;
  int64_t s0, s1, s2, s3;
};

struct ScanArgs {
  Op3 u, delta, z, y, h0, h_last;
  Op4 b, c;
  const float *a, *d, *bias;
  int64_t a_d, a_n, d_s, bias_s;
  const int *lengths;
  int64_t lengths_s;
  int64_t batch, length, dim;
  int states, groups, softplus, zero_rest;
  int64_t per;       // channels per group
  int64_t blocks_d;  // channel blocks per group
  int64_t chunks;    // pieces of the time axis, each by blocks of its own
  int64_t chunk;     // their length, a multiple of 32
  int vec_b, vec_c;  // b, c rows can be copied 16 bytes at a time
  float *saved;      // [B, ceil(L / save_every), D, NP]
  float *sum_h;      // [B, chunks, D, NP]: a piece's own end state, then its start state
  float *sum_dt;     // [B, chunks, D]: a piece's sum of steps
  // backward
  Op3 dy, dh_last, du, ddelta, dz, dh0;
  Op4 db, dc;
  float *part_bc;  // [blocks_d, B, L, G, 2, N]
  float *part_a;   // [B * chunks, D, N]
  float *part_d;   // [B * chunks, 2, D]
};

// Channels of a block whose threads hold `chan` channels each.
inline int64_t block_channels(int nl, int chan) { return (int64_t)kScanThreads / nl * chan; }

// Lane's 32-bit offsets reach the block's channels, of the `per` of a group, and a
// lane group's steps.
inline int check_reach(const DescView &v, int nl, int chan, int64_t per, const char *what) {
  const int64_t most = (int64_t)1 << 30;
  const int64_t s1 = stride_of(v, 1) < 0 ? -stride_of(v, 1) : stride_of(v, 1);
  const int64_t s2 = stride_of(v, 2) < 0 ? -stride_of(v, 2) : stride_of(v, 2);
  const int64_t steps = (v.sizes[1] < nl ? v.sizes[1] : nl) - 1;
  const int64_t channels = (per < block_channels(nl, chan) ? per : block_channels(nl, chan)) - 1;
  if ((steps > 0 && s1 > most / steps) || (channels > 0 && s2 > most / channels) ||
      (steps > 0 ? s1 * steps : 0) + (channels > 0 ? s2 * channels : 0) >= most)
    return fail(REMORA_ERR_LIMIT, "%s: time and channel strides of %lld and %lld elements spread a block over 2^30", what,
                (long long)s1, (long long)s2);
  return REMORA_OK;
}

// Lanes per channel for N states.
inline int lanes_for(int states) {
  int nl = 1;
  while (nl * 4 < states) nl *= 2;
  return nl;
}

inline Op3 op3(const DescView &v) {
  return {reinterpret_cast<float *>(v.data(4)), stride_of(v, 0), stride_of(v, 1), stride_of(v, 2)};
}

inline Op4 op4(const DescView &v) {
  return {reinterpret_cast<float *>(v.data(4)), stride_of(v, 0), stride_of(v, 1), stride_of(v, 2), stride_of(v, 3)};
}

int read_scan_in(const RemoraSelectiveScanSpec *spec, const RemoraSelectiveScanIn *in, ScanArgs *a, DescView views[10],
                 const char *what);
int combine_chunks(const ScanArgs &a, int nl, bool reverse, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ int64_t scan_length(const ScanArgs &a, int64_t b) {
  if (a.lengths == nullptr) return a.length;
  const int64_t n = a.lengths[b * a.lengths_s];
  return n < 0 ? 0 : n > a.length ? a.length : n;
}

// The place of a thread: block = ((b * chunks + chunk) * groups + g) * blocks_d + bd.
// Channels past the group's last stand on the block's first, with live false.
template <int NL, int CHAN>
struct Place {
  static constexpr int kChannels = kScanThreads / NL * CHAN;  // of a block
  int64_t bd, g, chunk, b, d[CHAN];
  int64_t first;    // the block's first channel
  int channels, lanes;  // of a block's channels and a lane group's steps, those that there are anywhere
  int local[CHAN];  // a channel's place in the block
  int q;
  bool live[CHAN], whole;  // whole: the block has no dead channel
  __device__ __forceinline__ explicit Place(const ScanArgs &a) {
    unsigned i = blockIdx.x;
    const unsigned groups = a.groups, blocks_d = (unsigned)a.blocks_d, chunks = (unsigned)a.chunks;
    bd = i % blocks_d, i /= blocks_d;
    g = i % groups, i /= groups;
    chunk = i % chunks, b = i / chunks;
    q = threadIdx.x % NL;
    first = g * a.per + bd * kChannels;
    channels = (int)min(a.per, (int64_t)kChannels);
    lanes = (int)min(a.length, (int64_t)NL);
    const int64_t left = a.per - bd * kChannels;
    whole = left >= kChannels;
#pragma unroll
    for (int c = 0; c < CHAN; ++c) {
      local[c] = (threadIdx.x / 32 * CHAN + c) * (32 / NL) + threadIdx.x % 32 / NL;
      live[c] = local[c] < left;
      if (!live[c]) local[c] = 0;
      d[c] = first + local[c];
    }
  }
};

// A lane's elements of a [B, time, D] operand: a base address that the whole
// block shares, moved along time, and a 32-bit offset per channel.  The offset
// counts from the lowest of the block's addresses, so it is never negative (but for
// lanes past the axis's end, which use none).
template <int NL, int CHAN>
struct Lane {
  char *base;
  int64_t step;  // bytes per time step
  unsigned off[CHAN];
  __device__ __forceinline__ Lane(const Op3 &o, const Place<NL, CHAN> &at, int64_t t0) {
    const int64_t low = (o.s2 < 0 ? o.s2 * (at.channels - 1) : 0) + (o.s1 < 0 ? o.s1 * (at.lanes - 1) : 0);
    base = reinterpret_cast<char *>(o.p + (at.b * o.s0 + t0 * o.s1 + at.first * o.s2 + low));
    step = o.s1 * 4;
#pragma unroll
    for (int c = 0; c < CHAN; ++c)
      off[c] = (unsigned)((at.local[c] * o.s2 + at.q * o.s1 - low) * 4);
  }
  __device__ __forceinline__ void go(int64_t steps) { base += steps * step; }
  // step t + q of channel c, t counted from where the base has got to
  __device__ __forceinline__ float &operator()(int c, int t) const {
    return *reinterpret_cast<float *>(base + t * step + off[c]);
  }
};

// Sets the rows of a chunk that lie behind the sequence's end to zero.
template <int NL, int CHAN>
__device__ __forceinline__ void zero_rows(const Lane<NL, CHAN> &o, const Place<NL, CHAN> &at, const ScanArgs &a,
                                          int64_t t0, int64_t len) {
  const int upto = (int)(min(t0 + a.chunk, a.length) - t0);
  for (int t = (int)(max(t0, len) - t0); t < upto; t += NL)
#pragma unroll
    for (int c = 0; c < CHAN; ++c)
      if (at.live[c] && t + at.q < upto) o(c, t) = 0.0f;
}

__device__ __forceinline__ void copy_async4(float *dst, const float *src, bool on) {
  const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(s), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_async16(float *dst, const float *src, bool on) {
  const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Starts the copy of rows [t0, t0 + STEPS) of one group of b or c to dst
// [STEPS][4 NL]; rows from t_end on and states from N on become zero (and
// their address, that of row t0, is not read).
template <int NL, int STEPS>
__device__ __forceinline__ void stage_rows(float *dst, const Op4 &src, int vec, int64_t b, int64_t g, int64_t t0,
                                           int64_t t_end, int states) {
  constexpr int NP = 4 * NL;
  const float *base = src.p + b * src.s0 + t0 * src.s1 + g * src.s2;
  const int rows = (int)(t_end - t0 < STEPS ? t_end - t0 : STEPS);
  if (vec) {
    for (int i = threadIdx.x; i < STEPS * NL; i += kScanThreads) {
      const int r = i / NL, n = (i % NL) * 4;
      const bool on = r < rows && n < states;
      copy_async16(dst + r * NP + n, on ? base + r * src.s1 + n : base, on);
    }
  } else {
    for (int i = threadIdx.x; i < STEPS * NP; i += kScanThreads) {
      const int r = i / NP, n = i % NP;
      const bool on = r < rows && n < states;
      copy_async4(dst + i, on ? base + r * src.s1 + n * src.s3 : base, on);
    }
  }
}

// Loads are not moved over this.  The steps of a piece are unrolled; with all
// their loads hoisted to its start the registers spill (backward pass of 4 x
// 2048 x 2048 x 16: 739 us without, 466 us with it).
__device__ __forceinline__ void keep_order() { asm volatile("" ::: "memory"); }

// v[k] of lane q becomes the sum over the NL lanes of v[q], in v[0].
template <int NL>
__device__ __forceinline__ void transpose_sum(float (&v)[NL], int q) {
#pragma unroll
  for (int o = NL / 2; o >= 1; o >>= 1) {
    const bool up = q & o;
#pragma unroll
    for (int k = 0; k < o; ++k) {
      const float send = up ? v[k] : v[k + o];
      const float keep = up ? v[k + o] : v[k];
      v[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
}

__device__ __forceinline__ void unpack(const float4 &v, float (&o)[4]) {
  o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
}
#endif

}  // namespace seq
}  // namespace remora
