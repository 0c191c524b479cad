// Dropout from a counter-based stream: y = residual + x keep / (1 - p).  keep is a function of
// (seed, step, layer, element), formed again where it is needed (the gradient of x is the same
// pass over the gradient of y), so no mask is read, written or kept.  One 64-bit word of the
// stream decides two neighbouring elements.
#include "typed.h"

namespace avc {
namespace {

constexpr unsigned long long kGolden = 0x9E3779B97F4A7C15ull;

struct DropArgs {
  long rows, cols;
  const void* x;
  long ldx;
  const void* res;
  long ldr;
  const long long* rng;
  unsigned layer;
  unsigned long long threshold;  // p 2^32: a word below it drops its element
  float scale;
  void* y;
  long ldy;
};

template <typename E>
constexpr int width() { return 16 / (int)sizeof(E); }
constexpr int kUnroll = 4;  // vectors of a thread in flight

// VEC elements from flat element e (row-major, strides left out) at the three places; n of them exist
template <typename E, int VEC, bool RES>
__device__ __forceinline__ void drop_vec(const DropArgs& a, unsigned long long key, long e, const Vec<E, VEC>& x,
                                         const Vec<E, VEC>& r, float (&out)[VEC]) {
  // a vector may begin on the second half of a word: one word more than VEC / 2 then
  const unsigned long long w0 = key + ((unsigned long long)(e >> 1) + 1) * kGolden;
  const bool odd = e & 1;
  unsigned u[VEC + 2];
#pragma unroll
  for (int k = 0; k <= VEC / 2; ++k) {
    if (k < VEC / 2 || odd) {
      const unsigned long long z = mix64(w0 + (unsigned long long)k * kGolden);
      u[2 * k] = (unsigned)z, u[2 * k + 1] = (unsigned)(z >> 32);
    } else {
      u[2 * k] = u[2 * k + 1] = 0;
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const unsigned word = odd ? u[v + 1] : u[v];
    const float k = word >= a.threshold ? (float)x.v[v] * a.scale : 0.0f;
    out[v] = RES ? (float)r.v[v] + k : k;
  }
}

// Bound by its reads and the write: 65536x1024 bf16 with a residual 83 us (4.9 TB/s, the rate of a large
// copy), its gradient 58 us (4.6 TB/s).  A thread takes kUnroll vectors; a row's last vector is moved
// back to end at the row's end (the elements it shares with its neighbour get the same value twice), so
// none is cut unless the row is shorter than one.  FLAT: the rows follow one another and are taken as one.
template <typename E, bool FLAT, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
  constexpr int VEC = width<E>();
  const unsigned long long key =
      mix64(mix64(mix64((unsigned long long)a.rng[0] + kGolden) + (unsigned long long)a.rng[1]) + a.layer);
  const long nv = (a.cols + VEC - 1) / VEC;  // vectors of a row; below 2^31 unless FLAT
  const long q0 = (long)blockIdx.x * (256 * kUnroll);
  const long row0 = FLAT ? 0 : q0 / nv, v0 = q0 - row0 * nv;
  const bool cut = a.cols < VEC;
  long row[kUnroll], c[kUnroll];
  Vec<E, VEC> x[kUnroll], r[kUnroll];
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
    if (FLAT) {
      const long w = v0 + k * 256 + threadIdx.x;
      row[k] = w < nv ? 0 : 1;
      c[k] = w * VEC;
    } else {
      const unsigned w = (unsigned)v0 + k * 256 + threadIdx.x;
      row[k] = row0 + w / (unsigned)nv;
      c[k] = (long)(w % (unsigned)nv) * VEC;
    }
    if (row[k] >= a.rows) continue;
    const E* xr = static_cast<const E*>(a.x) + row[k] * a.ldx;
    const E* rr = RES ? static_cast<const E*>(a.res) + row[k] * a.ldr : nullptr;
    if (!cut) {
      c[k] = c[k] + VEC <= a.cols ? c[k] : a.cols - VEC;
      x[k] = vload<E, VEC>(xr + c[k]);
      if (RES) r[k] = vload<E, VEC>(rr + c[k]);
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const int w = v < a.cols ? v : 0;
        x[k].v[v] = xr[w];
        if (RES) r[k].v[v] = rr[w];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kUnroll; ++k) {
    if (row[k] >= a.rows) continue;
    float out[VEC];
    drop_vec<E, VEC, RES>(a, key, row[k] * a.cols + c[k], x[k], r[k], out);
    E* yr = static_cast<E*>(a.y) + row[k] * a.ldy;
    if (!cut) {
      vstore<E, VEC>(yr + c[k], out);
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (v < a.cols) yr[v] = static_cast<E>(out[v]);
    }
  }
}

}  // namespace
}  // namespace avc

using namespace avc;

extern "C" int avc_dropout(int dtype, long rows, long cols, const void* x, long ldx, const void* residual, long ldr,
                           double p, const long long* rng, unsigned layer, void* y, long ldy, void* stream) {
  AVC_CHECK_ARG(dtype_ok(dtype), "dtype is one of AVC_DTYPE_F32, _BF16, _F16");
  AVC_CHECK_ARG(rows >= 0 && cols >= 0, "rows >= 0, cols >= 0");
  AVC_CHECK_ARG(p >= 0.0 && p < 1.0, "0 <= p < 1");
  if (rows == 0 || cols == 0) return AVC_OK;
  AVC_CHECK_ARG(rows <= (1L << 40) && cols <= (1L << 40) && rows <= (1L << 46) / cols, "rows * cols too large");
  AVC_CHECK_ARG(x && y && rng, "x, y and rng are needed");
  AVC_CHECK_ARG(ldx >= cols && ldy >= cols && (!residual || ldr >= cols), "a row stride is smaller than cols");
  DropArgs a{rows, cols, x, ldx, residual, ldr, rng, layer, (unsigned long long)(p * 4294967296.0),
             (float)(1.0 / (1.0 - p)), y, ldy};
  if (rows == 1 || (ldx == cols && ldy == cols && (!residual || ldr == cols))) a.cols = rows * cols, a.rows = 1;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    const long nv = (a.cols + width<E>() - 1) / width<E>();
    const long blocks = (a.rows * nv + 256 * kUnroll - 1) / (256 * kUnroll);
    AVC_CHECK_ARG(blocks < 1L << 24 && (a.rows == 1 || nv < 1L << 31), "rows * cols too large");
    const unsigned grid = (unsigned)blocks;
    if (a.rows == 1) {
      if (a.res) dropout_kernel<E, true, true><<<grid, 256, 0, s>>>(a);
      else dropout_kernel<E, true, false><<<grid, 256, 0, s>>>(a);
    } else {
      if (a.res) dropout_kernel<E, false, true><<<grid, 256, 0, s>>>(a);
      else dropout_kernel<E, false, false><<<grid, 256, 0, s>>>(a);
    }
    AVC_LAUNCH_CHECK();
    return AVC_OK;
  });
}
