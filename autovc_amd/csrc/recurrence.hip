// Gated linear recurrence over time-major frames: f = sigmoid(g_f), z = tanh(g_c), o = sigmoid(g_o),
//   h_t = f_t h_{t-1} + (1 - f_t) z_t,   y_t = o_t h_t.
// Its time loop is linear in h, so a stretch of frames acts on the state before it as
// h -> A h + B with A = prod f and B the stretch's own state from zero, and stretches compose:
// time is split over waves (and, where there are few rows, over workgroups) and joined.
//
// The backward runs the same way from the end.  With e_t the gradient of h_t and c_t = f_t e_t what
// frame t hands to frame t - 1:  e_t = o_t dy_t + c_{t+1},  c_t = f_t e_t  (c behind the last frame
// is the gradient of the final state), a stretch acts as c -> A c + B' with the same A, and
//   dg_f = e_t (h_{t-1} - z) f (1 - f),  dg_c = e_t (1 - f)(1 - z^2),  dg_o = dy h_t o (1 - o).
// h is formed again from states that the forward keeps every kState frames.
//
// Everything but the loaded and stored elements is fp32.  1 - f is never formed by subtraction.
#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "typed.h"

namespace avc {
namespace {

constexpr int kW = 8;        // waves of a workgroup = stretches of its chunk
constexpr int kState = 32;   // frames between the states that the forward keeps for the backward
// Frames of a wave's stretch, all in registers.  The backward of two-channel lanes takes 4, which
// leaves room for a third workgroup a CU (128x256x512 bf16: 48 us, with 8 frames 56).
template <int VEC, bool BACK>
constexpr int stretch() { return BACK && VEC > 1 ? 4 : 8; }
template <int VEC, bool BACK>
constexpr int chunk_of() { return stretch<VEC, BACK>() * kW; }

struct RecArgs {
  int T, B, H, dirs;
  const void* gates;
  long ldg;
  const int* lengths;
  const float* h0;   // [D][B][H]
  void* y;
  long ldy;
  float* hT;         // [D][B][H]
  float* states;     // [ceil(T / kState)][D][B][H]
  const void* dy;
  long lddy;
  const float* dhT;
  void* dgates;
  long lddg;
  float* dh0;
  float* agg;        // [nseg][2][D][B][H]: A and B (B') of each segment
  int nseg, seg_chunks;
  int log_g, nct;    // lanes of a wave per row (log2), channel tiles per row
  unsigned pack;     // workgroups that are reordered among themselves (0: none)
  unsigned tile0;    // first tile of the launch
};

// The forget gate as f = 1 / (1 + e), 1 - f = e f with e = exp(-g).  Below -80 (f < 2e-35) e is held
// there, so that neither it nor f leaves the normal range; a NaN passes.
__device__ __forceinline__ void forget_gate(float g, float& f, float& e) {
  e = __expf(-__builtin_elementwise_maximum(g, -80.0f));
  f = __builtin_amdgcn_rcpf(1.0f + e);
}
// tanh of the candidate.  fp32 gates take gate_tanh; 16-bit ones, whose lanes form two a frame and feel every
// instruction, the same with a shorter polynomial: a minimax one of x^7 below 0.35 (off by 0.7 units of
// 2^-24 relative, 1.7 with its roundings), and above it 1 - 2 / (1 + exp 2|x|) with x's sign, whose error of
// about 1 unit absolutely is 3 of the value there.  Over all bf16 and fp16 values either form is off by
// 3.1 units at most: the state that a call hands to the next is fp32 whatever the gates' type.
// (60001x1x500 fp16 forward 95 us, with gate_tanh 100; 1024x32x256 both directions ragged bf16 45 and 48.)
template <typename E>
__device__ __forceinline__ float candidate(float x) {
  if (sizeof(E) == 4) return gate_tanh(x);
  const float x2 = x * x, ax = fabsf(x);
  const float p = fmaf(fmaf(x2, -0.0491485037f, 0.132998258f), x2, -0.333326638f);
  const float small = fmaf(x * x2, p, x);
  const float big = fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __expf(2.0f * ax)), 1.0f);
  return ax < 0.35f ? small : copysignf(big, x);
}

// Where a lane works: VEC channels of one row b in one direction.  Rows narrower than a wave share
// it.  The last vector of a row is moved back to end at H (channels that two lanes share get the
// same value twice), so no vector is cut; lanes past the row or the batch repeat its last place
// and store nothing.  Frames are the same for the whole wave: an address is a scalar one for the
// frame plus the lane's 32-bit offset in it.
template <typename E, int VEC>
struct Place {
  int wave, lane, row0, lr, j, d, len, seg;
  bool ok, rev;
  __device__ explicit Place(const RecArgs& a) {
    unsigned bx = blockIdx.x;
    seg = blockIdx.y, d = blockIdx.z;
    if (a.pack) {
      // the channel tiles of a row, 8 workgroups apart, go to the XCD that has the row's other tiles
      const unsigned gx = gridDim.x, gy = gridDim.y;
      unsigned id = bx + gx * (blockIdx.y + gy * blockIdx.z);
      const unsigned in = id % a.pack;
      if (id - in + a.pack <= gx * gy * gridDim.z) id = id - in + (in & 7) * a.nct + (in >> 3);
      bx = id % gx, id /= gx;
      seg = id % gy, d = id / gy;
    }
    bx += a.tile0;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    const int g = 1 << a.log_g;
    const int cv = (bx % a.nct) * g + (lane & (g - 1));
    row0 = (int)(bx / a.nct) * (64 >> a.log_g);
    lr = lane >> a.log_g;
    ok = cv * VEC < a.H && row0 + lr < a.B;
    j = min(cv * VEC, a.H - VEC);
    lr = min(lr, a.B - 1 - row0);
    rev = a.dirs == 2 || d == 1;
    len = a.lengths ? min(max(a.lengths[row0 + lr], 0), a.T) : a.T;
  }
  // a matrix of frame rows of stride ld, `width` elements a direction
  __device__ E* rows(const void* p, long ld, int width) const {
    return static_cast<E*>(const_cast<void*>(p)) + (long)row0 * ld + (long)d * width;
  }
  __device__ unsigned off(long ld) const { return (unsigned)lr * (unsigned)ld + (unsigned)j; }
  // the state of [D][B][H] floats
  __device__ long state0(const RecArgs& a) const { return ((long)d * a.B + row0) * a.H; }
};
template <int VEC, typename E>
__device__ __forceinline__ Vec<E, VEC> take(const E* scalar, unsigned off) {
  return vload<E, VEC>(reinterpret_cast<const E*>(reinterpret_cast<const char*>(scalar) + off * (unsigned)sizeof(E)));
}
template <int VEC, typename E>
__device__ __forceinline__ void give(E* scalar, unsigned off, const float (&x)[VEC]) {
  vstore<E, VEC>(reinterpret_cast<E*>(reinterpret_cast<char*>(scalar) + off * (unsigned)sizeof(E)), x);
}
template <int VEC>
__device__ __forceinline__ void take_to(float (&x)[VEC], const float* scalar, unsigned off) {
  const Vec<float, VEC> r = take<VEC>(scalar, off);
#pragma unroll
  for (int v = 0; v < VEC; ++v) x[v] = r.v[v];
}

// frame of step s of a direction's own order (s < T)
__device__ __forceinline__ int frame_of(const RecArgs& a, int s, bool rev) { return rev ? a.T - 1 - s : s; }
// What of the S frames from step s0 is live for the wave: nothing, everything for every lane, or a part
enum Live { kNone, kPart, kAll };
template <bool RAGGED, int S>
__device__ __forceinline__ Live live_of(const RecArgs& a, int s0, bool rev, int len) {
  if (s0 >= a.T) return kNone;
  if (!RAGGED) return s0 + S <= a.T ? kAll : kPart;
  const int t0 = rev ? max(a.T - s0 - S, 0) : s0, t1 = rev ? a.T - s0 : min(s0 + S, a.T);
  if (!__any(t0 < len)) return kNone;
  return s0 + S <= a.T && __all(t1 <= len) ? kAll : kPart;
}
template <bool RAGGED>
__device__ __forceinline__ bool is_live(const RecArgs& a, int s, bool rev, int len) {
  return s < a.T && (!RAGGED || frame_of(a, s, rev) < len);
}

// A gate that is not read: f = 1 and 1 - f = 0 (kept), z = 0, o = 0
template <typename E, int VEC>
__device__ __forceinline__ Vec<E, VEC> constant(float x) {
  Vec<E, VEC> r;
#pragma unroll
  for (int v = 0; v < VEC; ++v) r.v[v] = static_cast<E>(x);
  return r;
}

// Carries x through the segments lo .. hi-1 (BACK: from the last to the first): the waves join a
// run of segments each, side by side, and every wave then joins the runs.
template <int VEC, bool BACK>
__device__ void join_segments(const RecArgs& a, int lo, int hi, const float* agg, unsigned off, long nstate, int wave,
                              int lane, float (*part)[2 + BACK][64][VEC], float (&x)[VEC]) {
  if (lo >= hi) return;
  const int per = (hi - lo + kW - 1) / kW;
  float A[VEC], Bv[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) A[v] = 1.0f, Bv[v] = 0.0f;
  const int q0 = lo + wave * per, q1 = min(q0 + per, hi);
#pragma unroll 4
  for (int i = q0; i < q1; ++i) {
    const float* p = agg + (long)(BACK ? q0 + q1 - 1 - i : i) * 2 * nstate;
    float pa[VEC], pb[VEC];
    take_to<VEC>(pa, p, off);
    take_to<VEC>(pb, p + nstate, off);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      Bv[v] = fmaf(pa[v], Bv[v], pb[v]);
      A[v] *= pa[v];
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) part[wave][0][lane][v] = A[v], part[wave][1][lane][v] = Bv[v];
  __syncthreads();
#pragma unroll
  for (int ww = 0; ww < kW; ++ww) {
    const int w = BACK ? kW - 1 - ww : ww;
#pragma unroll
    for (int v = 0; v < VEC; ++v) x[v] = fmaf(part[w][0][lane][v], x[v], part[w][1][lane][v]);
  }
  __syncthreads();
}

// A workgroup walks its segment chunk by chunk: each wave forms its stretch's action from gates that were
// asked for a chunk earlier, the actions meet in LDS (double-buffered: one barrier a chunk), and each
// wave goes over its own stretch, still in registers, with the state that comes to it.  Gates are read
// once and y written once: 128x256x512 alone fp32 55 us (4.9 TB/s, the rate of a large copy), bf16 32; in a
// training pass, behind a backward whose writes are still on their way to memory, fp32 69.
template <typename E, int VEC, bool RAGGED>
__global__ __launch_bounds__(kW * 64, 4) void recurrence_forward_kernel(RecArgs a) {
  constexpr int kS = stretch<VEC, false>(), kChunk = kS * kW;
  const Place<E, VEC> at(a);
  const int wave = at.wave, lane = at.lane;
  __shared__ float part[2][kW][2][64][VEC];
  const E* g = at.rows(a.gates, a.ldg, 3 * a.H);
  E* y = at.rows(a.y, a.ldy, a.H);
  const unsigned goff = at.off(a.ldg), yoff = at.off(a.ldy), soff = at.off(a.H);
  const long gstep = (long)a.B * a.ldg, ystep = (long)a.B * a.ldy;
  const long st0 = at.state0(a), nstate = (long)(a.dirs == 3 ? 2 : 1) * a.B * a.H;

  float h[VEC] = {};
  if (a.h0) take_to<VEC>(h, a.h0 + st0, soff);
  const int first = at.seg * a.seg_chunks;
  const int last = min(first + a.seg_chunks, (a.T + kChunk - 1) / kChunk);
  Vec<E, VEC> rf[kS], rc[kS], ro[kS];
  auto load = [&](int chunk) {
    const int s0 = chunk * kChunk + wave * kS;
    if (chunk >= last) return;
    auto frame = [&](int k) {
      const E* p = g + frame_of(a, s0 + k, at.rev) * gstep;
      rf[k] = take<VEC>(p, goff);
      rc[k] = take<VEC>(p + a.H, goff);
      ro[k] = take<VEC>(p + 2 * a.H, goff);
    };
    const Live live = live_of<RAGGED, kS>(a, s0, at.rev, at.len);
    if (live == kAll) {
#pragma unroll
      for (int k = 0; k < kS; ++k) frame(k);
    } else if (live == kPart) {
#pragma unroll
      for (int k = 0; k < kS; ++k) {
        rf[k] = constant<E, VEC>(INFINITY), rc[k] = constant<E, VEC>(0.0f), ro[k] = constant<E, VEC>(-INFINITY);
        if (is_live<RAGGED>(a, s0 + k, at.rev, at.len)) frame(k);
      }
    }
  };
  load(first);
  join_segments<VEC, false>(a, 0, at.seg, a.agg + st0, soff, nstate, wave, lane, part[first & 1], h);
  for (int chunk = first; chunk < last; ++chunk) {
    const int s0 = chunk * kChunk + wave * kS;
    const Live live = live_of<RAGGED, kS>(a, s0, at.rev, at.len);
    float prod[kS][VEC], loc[kS][VEC], o[kS][VEC];
    float A[VEC], Bv[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.0f, Bv[v] = 0.0f;
    if (live != kNone) {
#pragma unroll
      for (int k = 0; k < kS; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          float f, e;
          forget_gate((float)rf[k].v[v], f, e);
          o[k][v] = gate_sigmoid((float)ro[k].v[v]);
          loc[k][v] = Bv[v] = f * fmaf(e, candidate<E>((float)rc[k].v[v]), Bv[v]);  // f h + (1 - f) z
          prod[k][v] = A[v] *= f;
        }
    }
    float (*mine)[2][64][VEC] = part[chunk & 1];
#pragma unroll
    for (int v = 0; v < VEC; ++v) mine[wave][0][lane][v] = A[v], mine[wave][1][lane][v] = Bv[v];
    load(chunk + 1);
    __syncthreads();
    float hin[VEC];
#pragma unroll
    for (int w = 0; w < kW; ++w) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (w == wave) hin[v] = h[v];
        h[v] = fmaf(mine[w][0][lane][v], h[v], mine[w][1][lane][v]);
      }
    }
    if (s0 >= a.T || !at.ok) continue;
    if (a.states && s0 % kState == 0) give<VEC>(a.states + (long)(s0 / kState) * nstate + st0, soff, hin);
#pragma unroll
    for (int k = 0; k < kS; ++k) {
      if (s0 + k < a.T) {
        const int t = frame_of(a, s0 + k, at.rev);
        const bool on = !RAGGED || t < at.len;
        float out[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) out[v] = on ? o[k][v] * fmaf(prod[k][v], hin[v], loc[k][v]) : 0.0f;
        give<VEC>(y + t * ystep, yoff, out);
      }
    }
  }
  if (a.hT && last == (a.T + kChunk - 1) / kChunk && wave == 0 && at.ok) give<VEC>(a.hT + st0, soff, h);
}

// The same walk from the last chunk to the first, with the action on the state too (from the state kept
// at the chunk's beginning), so that h needs no pass of its own.  Bound by reading gates and dy and
// writing dgates once: 128x256x512 alone fp32 102 us (4.6 TB/s; 88 right behind the forward, which leaves
// some of the gates in the last-level cache), bf16 49 us.
template <typename E, int VEC, bool RAGGED>
__global__ __launch_bounds__(kW * 64, 2) void recurrence_backward_kernel(RecArgs a) {
  constexpr int kS = stretch<VEC, true>(), kChunk = kS * kW;
  static_assert(kChunk % kState == 0, "a chunk begins at a kept state");
  const Place<E, VEC> at(a);
  const int wave = at.wave, lane = at.lane;
  __shared__ float part[2][kW][3][64][VEC];
  const E* g = at.rows(a.gates, a.ldg, 3 * a.H);
  const E* dy = at.rows(a.dy, a.lddy, a.H);
  E* dg = at.rows(a.dgates, a.lddg, 3 * a.H);
  const unsigned goff = at.off(a.ldg), dyoff = at.off(a.lddy), dgoff = at.off(a.lddg), soff = at.off(a.H);
  const long gstep = (long)a.B * a.ldg, dystep = (long)a.B * a.lddy, dgstep = (long)a.B * a.lddg;
  const long st0 = at.state0(a), nstate = (long)(a.dirs == 3 ? 2 : 1) * a.B * a.H;

  float c[VEC] = {};  // what the frames behind this chunk hand back
  if (a.dhT) take_to<VEC>(c, a.dhT + st0, soff);
  const int first = at.seg * a.seg_chunks;
  const int last = min(first + a.seg_chunks, (a.T + kChunk - 1) / kChunk);
  Vec<E, VEC> rf[kS], rc[kS], ro[kS], ry[kS];
  float hs[VEC];
  auto load = [&](int chunk) {
    if (chunk < first) return;
    const int s0 = chunk * kChunk + wave * kS;
    const Live live = live_of<RAGGED, kS>(a, s0, at.rev, at.len);
    if (live == kNone) return;
    take_to<VEC>(hs, a.states + (long)(chunk * (kChunk / kState)) * nstate + st0, soff);
    auto frame = [&](int k) {
      const int t = frame_of(a, s0 + k, at.rev);
      const E* p = g + t * gstep;
      rf[k] = take<VEC>(p, goff);
      rc[k] = take<VEC>(p + a.H, goff);
      ro[k] = take<VEC>(p + 2 * a.H, goff);
      ry[k] = take<VEC>(dy + t * dystep, dyoff);
    };
    if (live == kAll) {
#pragma unroll
      for (int k = 0; k < kS; ++k) frame(k);
    } else {
      // a frame behind the end keeps the state and hands every gradient through
#pragma unroll
      for (int k = 0; k < kS; ++k) {
        rf[k] = constant<E, VEC>(INFINITY), rc[k] = constant<E, VEC>(0.0f), ro[k] = constant<E, VEC>(-INFINITY);
        ry[k] = constant<E, VEC>(0.0f);
        if (is_live<RAGGED>(a, s0 + k, at.rev, at.len)) frame(k);
      }
    }
  };
  load(last - 1);
  join_segments<VEC, true>(a, at.seg + 1, a.nseg, a.agg + st0, soff, nstate, wave, lane, part[last & 1], c);
  for (int chunk = last - 1; chunk >= first; --chunk) {
    const int s0 = chunk * kChunk + wave * kS;
    const Live live = live_of<RAGGED, kS>(a, s0, at.rev, at.len);
    float f[kS][VEC], i[kS][VEC], z[kS][VEC], o[kS][VEC], d[kS][VEC];
    float A[VEC], Bv[VEC], Cv[VEC], hin[VEC], cin[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.0f, Bv[v] = 0.0f, Cv[v] = 0.0f, hin[v] = hs[v];
    if (live != kNone) {
#pragma unroll
      for (int k = 0; k < kS; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          forget_gate((float)rf[k].v[v], f[k][v], i[k][v]);
          i[k][v] *= f[k][v];
          z[k][v] = candidate<E>((float)rc[k].v[v]);
          o[k][v] = gate_sigmoid((float)ro[k].v[v]);
          d[k][v] = (float)ry[k].v[v];
          Bv[v] = fmaf(f[k][v], Bv[v], i[k][v] * z[k][v]);
          A[v] *= f[k][v];
        }
#pragma unroll
      for (int k = kS - 1; k >= 0; --k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) Cv[v] = f[k][v] * fmaf(o[k][v], d[k][v], Cv[v]);
    }
    float (*mine)[3][64][VEC] = part[chunk & 1];
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      mine[wave][0][lane][v] = A[v], mine[wave][1][lane][v] = Bv[v], mine[wave][2][lane][v] = Cv[v];
    load(chunk - 1);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kW; ++w)
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (w < wave) hin[v] = fmaf(mine[w][0][lane][v], hin[v], mine[w][1][lane][v]);
#pragma unroll
    for (int w = kW - 1; w >= 0; --w)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (w == wave) cin[v] = c[v];
        c[v] = fmaf(mine[w][0][lane][v], c[v], mine[w][2][lane][v]);
      }
    if (s0 >= a.T || !at.ok) continue;
    if (live == kNone) {
      // nothing but frames behind the ends of their sequences: no gradient
#pragma unroll
      for (int k = 0; k < kS; ++k) {
        const float none[VEC] = {};
        if (s0 + k < a.T) {
          E* p = dg + frame_of(a, s0 + k, at.rev) * dgstep;
          give<VEC>(p, dgoff, none);
          give<VEC>(p + a.H, dgoff, none);
          give<VEC>(p + 2 * a.H, dgoff, none);
        }
      }
      continue;
    }
    float h[kS + 1][VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) h[0][v] = hin[v];
#pragma unroll
    for (int k = 0; k < kS; ++k)
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[k + 1][v] = fmaf(f[k][v], h[k][v], i[k][v] * z[k][v]);
#pragma unroll
    for (int k = kS - 1; k >= 0; --k) {
      float df[VEC], dc[VEC], dov[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float e = fmaf(o[k][v], d[k][v], cin[v]);
        cin[v] = f[k][v] * e;
        df[v] = cin[v] * i[k][v] * (h[k][v] - z[k][v]);
        dc[v] = e * i[k][v] * fmaf(-z[k][v], z[k][v], 1.0f);
        dov[v] = d[k][v] * h[k + 1][v] * fmaf(-o[k][v], o[k][v], o[k][v]);
      }
      if (s0 + k < a.T) {
        const int t = frame_of(a, s0 + k, at.rev);
        E* p = dg + t * dgstep;
        if (RAGGED && t >= at.len) {  // also where the state or a gradient is not finite
#pragma unroll
          for (int v = 0; v < VEC; ++v) df[v] = dc[v] = dov[v] = 0.0f;
        }
        give<VEC>(p, dgoff, df);
        give<VEC>(p + a.H, dgoff, dc);
        give<VEC>(p + 2 * a.H, dgoff, dov);
      }
    }
  }
  if (a.dh0 && first == 0 && wave == 0 && at.ok) give<VEC>(a.dh0 + st0, soff, c);
}

// What one segment of time does to the state before it (BACK: to the gradient behind it): each
// wave walks a run of stretches of its own, then the waves' runs are joined in order.  It reads two
// thirds of the gates (60001x1x500 fp16: 40 us, then 60 us for the forward).  One pass in which the
// workgroups hand the state on as they go read them once and took longer: 137 us instead of 111 then.
template <typename E, int VEC, bool RAGGED, bool BACK>
__global__ __launch_bounds__(kW * 64, 6) void recurrence_segment_kernel(RecArgs a) {
  constexpr int kS = 16;  // frames in flight (1024x32x256, both directions, ragged, bf16: 46 + 62 us, with 4 47.5 + 64)
  const Place<E, VEC> at(a);
  const int wave = at.wave, lane = at.lane;
  __shared__ float part[kW][2][64][VEC];
  const E* g = at.rows(a.gates, a.ldg, 3 * a.H);
  const E* dy = BACK ? at.rows(a.dy, a.lddy, a.H) : nullptr;
  const unsigned goff = at.off(a.ldg), dyoff = at.off(a.lddy), soff = at.off(a.H);
  const long gstep = (long)a.B * a.ldg, dystep = (long)a.B * a.lddy;
  const long st0 = at.state0(a), nstate = (long)(a.dirs == 3 ? 2 : 1) * a.B * a.H;
  const int steps = a.seg_chunks * stretch<VEC, BACK>();  // of a wave's run
  // (the last segment in the order of work acts on nothing)
  const int seg = BACK ? at.seg + 1 : at.seg;
  const int base = (seg * kW + wave) * steps;
  float A[VEC], Bv[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) A[v] = 1.0f, Bv[v] = 0.0f;
  for (int q = 0; q < steps; q += kS) {
    const int s0 = base + (BACK ? max(steps - q - kS, 0) : q), n = min(kS, steps - q);
    const Live live = live_of<RAGGED, kS>(a, s0, at.rev, at.len);
    if (live == kNone) continue;
    Vec<E, VEC> r0[kS], r1[kS], r2[kS];
    auto frame = [&](int k) {
      const int t = frame_of(a, s0 + k, at.rev);
      const E* p = g + t * gstep;
      r0[k] = take<VEC>(p, goff);
      if (BACK) {
        r1[k] = take<VEC>(p + 2 * a.H, goff);
        r2[k] = take<VEC>(dy + t * dystep, dyoff);
      } else {
        r1[k] = take<VEC>(p + a.H, goff);
      }
    };
    if (live == kAll && n == kS) {
#pragma unroll
      for (int k = 0; k < kS; ++k) frame(k);
    } else {
#pragma unroll
      for (int k = 0; k < kS; ++k) {
        r0[k] = constant<E, VEC>(INFINITY), r1[k] = r2[k] = constant<E, VEC>(0.0f);
        if (k < n && is_live<RAGGED>(a, s0 + k, at.rev, at.len)) frame(k);
      }
    }
#pragma unroll
    for (int kk = 0; kk < kS; ++kk) {
      const int k = BACK ? kS - 1 - kk : kk;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float f, e;
        forget_gate((float)r0[k].v[v], f, e);
        Bv[v] = f * (BACK ? fmaf(gate_sigmoid((float)r1[k].v[v]), (float)r2[k].v[v], Bv[v])
                          : fmaf(e, candidate<E>((float)r1[k].v[v]), Bv[v]));
        A[v] *= f;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) part[wave][0][lane][v] = A[v], part[wave][1][lane][v] = Bv[v];
  __syncthreads();
  if (wave == 0 && at.ok) {
    float* p = a.agg + (long)seg * 2 * nstate + st0;
    float A2[VEC], B2[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A2[v] = 1.0f, B2[v] = 0.0f;
#pragma unroll
      for (int ww = 0; ww < kW; ++ww) {
        const int w = BACK ? kW - 1 - ww : ww;
        B2[v] = fmaf(part[w][0][lane][v], B2[v], part[w][1][lane][v]);
        A2[v] *= part[w][0][lane][v];
      }
    }
    give<VEC>(p, soff, A2);
    give<VEC>(p + nstate, soff, B2);
  }
}

// One frame of every row: the served form.  Bound by its launch (512 channels 2.0 us).
template <typename E, int VEC>
__global__ __launch_bounds__(256) void recurrence_step_kernel(int B, int H, const E* gates, long ldg, const float* h,
                                                              float* h_out, E* y, long ldy) {
  const int nv = (H + VEC - 1) / VEC;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const int b = (int)(id / nv);
  if (b >= B) return;
  // (no shared vectors here: with h_out = h a channel computed twice could be read after its
  // first write)
  const int j = (int)(id % nv) * VEC;
  const E* g = gates + (long)b * ldg + j;
  const int n = min(VEC, H - j);
  const long st = (long)b * H + j;
  float out[VEC], hn[VEC];
  Vec<E, VEC> rf, rc, ro;
  float hv[VEC];
  if (n == VEC) {
    rf = vload<E, VEC>(g), rc = vload<E, VEC>(g + H), ro = vload<E, VEC>(g + 2 * H);
    const Vec<float, VEC> t = vload<float, VEC>(h + st);
#pragma unroll
    for (int v = 0; v < VEC; ++v) hv[v] = t.v[v];
  } else {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const int w = min(v, n - 1);
      rf.v[v] = g[w], rc.v[v] = g[H + w], ro.v[v] = g[2 * H + w], hv[v] = h[st + w];
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float f, e;
    forget_gate((float)rf.v[v], f, e);
    hn[v] = f * fmaf(e, candidate<E>((float)rc.v[v]), hv[v]);
    out[v] = gate_sigmoid((float)ro.v[v]) * hn[v];
  }
  E* yo = y + (long)b * ldy + j;
  if (n == VEC) {
    vstore<float, VEC>(h_out + st, hn);
    vstore<E, VEC>(yo, out);
  } else {
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      if (v < n) h_out[st + v] = hn[v], yo[v] = static_cast<E>(out[v]);
  }
}

// Channels of a lane: 4 bytes.  (8-byte lanes hold twice the registers: a training pass of
// 128x256x512 takes 88 + 98 us in fp32 instead of 55 + 102, 77 + 56 us in bf16 instead of 32 + 49;
// 2-byte lanes of 16-bit gates 37 + 56.)
template <typename E>
constexpr int wide() { return sizeof(E) == 4 ? 1 : 2; }

// How a call is laid over the chip: lanes per row, row tiles, and segments of time.  With row tiles
// enough to fill the chip each workgroup walks its rows' whole time; with fewer, time is cut into as
// many segments as bring the grid to two workgroups a CU, which costs a pass over most of the gates
// for the segments' actions and a launch.  1024 frames in 128 tiles (bf16, ragged): cut in four
// 46 us, in two 53, whole 61; 60001 frames in 4 tiles: 128 segments 95 us, 64 107; twice as many segments
// 48 and 100.  Up to 512 frames are not cut: 400 frames in 180 tiles 36 us cut, 26 whole; 200 frames in 16
// tiles 13 us either way.
struct Layout {
  int log_g = 0, nct, nseg, seg_chunks;
  long tiles;
  Layout(int T, int B, int H, int D, int vec, int chunk) {
    while (log_g < 6 && (vec << log_g) < H) ++log_g;
    nct = (H + (vec << log_g) - 1) / (vec << log_g);
    const int rows = 64 >> log_g, chunks = (T + chunk - 1) / chunk;
    tiles = (long)nct * ((B + rows - 1) / rows);
    long n = tiles * D >= 256 || T <= 512 ? 1 : 512 / (tiles * D);
    if (n > chunks) n = chunks;
    seg_chunks = (int)((chunks + n - 1) / n);
    nseg = (chunks + seg_chunks - 1) / seg_chunks;
  }
  size_t workspace(int B, int H, int D) const { return nseg > 1 ? (size_t)nseg * 2 * D * B * H * sizeof(float) : 0; }
};
template <typename E, bool BACK>
Layout layout(int T, int B, int H, int D) {
  return H >= wide<E>() ? Layout(T, B, H, D, wide<E>(), chunk_of<wide<E>(), BACK>()) : Layout(T, B, H, D, 1, chunk_of<1, BACK>());
}

template <typename E, int VEC, bool BACK>
int run_recurrence(RecArgs a, size_t ws_bytes, hipStream_t s) {
  const int D = a.dirs == 3 ? 2 : 1;
  const Layout l = layout<E, BACK>(a.T, a.B, a.H, D);
  a.log_g = l.log_g, a.nct = l.nct, a.nseg = l.nseg, a.seg_chunks = l.seg_chunks;
  const size_t need = l.workspace(a.B, a.H, D);
  AVC_CHECK_ARG(ws_bytes >= need && (need == 0 || a.agg), "workspace smaller than avc_gated_recurrence_workspace");
  AVC_CHECK_ARG(l.tiles < 1L << 32, "B * H too large");
  // the rows that share a wave are reached by 32-bit offsets from the first of them
  const long widest = std::max(a.ldg, std::max(a.ldy, std::max(a.lddy, a.lddg)));
  AVC_CHECK_ARG(widest < (1L << 29) >> (6 - l.log_g), "row stride too large");
  // Tiles that begin inside a 128-byte line share it with their neighbours: they then run on one XCD,
  // whose L2 reads it once (60001 frames of 500 fp16 channels: 95 + 146 us, in launch order 101 + 165;
  // with tiles on whole lines the reordering only costs, 1 us of 37 + 59).
  const long line = 128 / (long)sizeof(E);
  const bool split = a.H % line || a.ldg % line || reinterpret_cast<uintptr_t>(a.gates) % 128;
  a.pack = split && l.nct > 1 ? 8u * l.nct : 0;
  // More tiles than a grid takes (2^32 threads) go in launches of nearly equal parts; time is not cut then.
  const long most = (1L << 32) / (kW * 64) - 1, parts = (l.tiles + most - 1) / most, per = (l.tiles + parts - 1) / parts;
  for (long tile = 0; tile < l.tiles; tile += per) {
    a.tile0 = (unsigned)tile;
    const unsigned tiles = (unsigned)std::min(per, l.tiles - tile);
    const dim3 grid(tiles, a.nseg, D);
    if (a.nseg > 1) {
      const dim3 before(tiles, a.nseg - 1, D);
      if (a.lengths) recurrence_segment_kernel<E, VEC, true, BACK><<<before, kW * 64, 0, s>>>(a);
      else recurrence_segment_kernel<E, VEC, false, BACK><<<before, kW * 64, 0, s>>>(a);
      AVC_LAUNCH_CHECK();
    }
    if constexpr (BACK) {
      if (a.lengths) recurrence_backward_kernel<E, VEC, true><<<grid, kW * 64, 0, s>>>(a);
      else recurrence_backward_kernel<E, VEC, false><<<grid, kW * 64, 0, s>>>(a);
    } else {
      if (a.lengths) recurrence_forward_kernel<E, VEC, true><<<grid, kW * 64, 0, s>>>(a);
      else recurrence_forward_kernel<E, VEC, false><<<grid, kW * 64, 0, s>>>(a);
    }
    AVC_LAUNCH_CHECK();
  }
  return AVC_OK;
}

int check_shape(int dtype, int T, int B, int H, int dirs, long ldg) {
  AVC_CHECK_ARG(dtype_ok(dtype), "dtype is one of AVC_DTYPE_F32, _BF16, _F16");
  AVC_CHECK_ARG(T >= 1 && B >= 0 && H >= 1, "T >= 1, B >= 0, H >= 1");
  AVC_CHECK_ARG(T <= 1 << 30 && B <= 1 << 30 && H <= 1 << 28, "T, B or H too large");
  AVC_CHECK_ARG(dirs >= 1 && dirs <= 3, "dirs is 1 (forward), 2 (reverse) or 3 (both)");
  AVC_CHECK_ARG(ldg >= (long)(dirs == 3 ? 6 : 3) * H, "a gate row is narrower than its gates");
  return AVC_OK;
}

}  // namespace
}  // namespace avc

using namespace avc;

extern "C" size_t avc_gated_recurrence_states(int T, int B, int H, int dirs) {
  if (T < 0 || B < 0 || H < 1 || dirs < 1 || dirs > 3) return 0;
  return (size_t)(T / kState + (T % kState != 0)) * (dirs == 3 ? 2 : 1) * B * H;
}

extern "C" size_t avc_gated_recurrence_workspace(int dtype, int T, int B, int H, int dirs) {
  if (!dtype_ok(dtype) || T < 1 || B < 1 || H < 1 || dirs < 1 || dirs > 3) return 0;
  const int D = dirs == 3 ? 2 : 1;
  size_t n = 0;
  with_dtype(dtype, [&](auto e) {
    using E = decltype(e);  // enough for either direction's call
    n = std::max(layout<E, false>(T, B, H, D).workspace(B, H, D), layout<E, true>(T, B, H, D).workspace(B, H, D));
    return AVC_OK;
  });
  return n;
}

extern "C" int avc_gated_recurrence_forward(int dtype, int T, int B, int H, int dirs, const void* gates, long ldg,
                                            const float* h0, const int* lengths, void* y, long ldy, float* hT,
                                            float* states, void* workspace, size_t workspace_bytes, void* stream) {
  AVC_TRY(check_shape(dtype, T, B, H, dirs, ldg));
  const int D = dirs == 3 ? 2 : 1;
  AVC_CHECK_ARG(ldy >= (long)D * H, "an output row is narrower than D * H");
  if (B == 0) return AVC_OK;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  AVC_CHECK_ARG(gates && y, "gates and y are needed");
  RecArgs a{};
  a.T = T, a.B = B, a.H = H, a.dirs = dirs, a.gates = gates, a.ldg = ldg, a.lengths = lengths, a.h0 = h0;
  a.y = y, a.ldy = ldy, a.hT = hT, a.states = states, a.agg = static_cast<float*>(workspace);
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return H >= wide<E>() ? run_recurrence<E, wide<E>(), false>(a, workspace_bytes, s)
                          : run_recurrence<E, 1, false>(a, workspace_bytes, s);
  });
}

extern "C" int avc_gated_recurrence_backward(int dtype, int T, int B, int H, int dirs, const void* gates, long ldg,
                                             const int* lengths, const float* states, const void* dy, long lddy,
                                             const float* dhT, void* dgates, long lddg, float* dh0, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  AVC_TRY(check_shape(dtype, T, B, H, dirs, ldg));
  const int D = dirs == 3 ? 2 : 1;
  AVC_CHECK_ARG(lddy >= (long)D * H && lddg >= (long)D * 3 * H, "a gradient row is narrower than its contents");
  if (B == 0) return AVC_OK;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  AVC_CHECK_ARG(gates && dy && dgates && states, "gates, states, dy and dgates are needed");
  RecArgs a{};
  a.T = T, a.B = B, a.H = H, a.dirs = dirs, a.gates = gates, a.ldg = ldg, a.lengths = lengths;
  a.states = const_cast<float*>(states), a.dy = dy, a.lddy = lddy, a.dhT = dhT, a.dgates = dgates, a.lddg = lddg;
  a.dh0 = dh0, a.agg = static_cast<float*>(workspace);
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return H >= wide<E>() ? run_recurrence<E, wide<E>(), true>(a, workspace_bytes, s)
                          : run_recurrence<E, 1, true>(a, workspace_bytes, s);
  });
}

extern "C" int avc_gated_recurrence_step(int dtype, int B, int H, const void* gates, long ldg, const float* h,
                                         float* h_out, void* y, long ldy, void* stream) {
  AVC_TRY(check_shape(dtype, 1, B, H, 1, ldg));
  AVC_CHECK_ARG(ldy >= H, "an output row is narrower than H");
  if (B == 0) return AVC_OK;
  AVC_CHECK_ARG(gates && h && h_out && y, "gates, h, h_out and y are needed");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    constexpr int VEC = 4;
    const long n = (long)B * ((H + VEC - 1) / VEC);
    AVC_CHECK_ARG(n < (1L << 32) - 256, "B * H too large");
    recurrence_step_kernel<E, VEC><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(
        B, H, static_cast<const E*>(gates), ldg, h, h_out, static_cast<E*>(y), ldy);
    AVC_LAUNCH_CHECK();
    return AVC_OK;
  });
}
