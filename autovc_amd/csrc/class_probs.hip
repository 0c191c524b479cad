// Log-probabilities of given classes under rows of logits, with each row's entropy and its most
// probable classes.  One pass over the logits keeps, for every thread,
//   m = max z,   s = sum exp(z - m),   u = sum exp(z - m) (z - m),
// moved to a new maximum m' by s' = s e^(m - m'), u' = (u + (m - m') s) e^(m - m').  Then
//   log p_i = (z_i - m) - log s,   entropy = log s - u / s   (both terms >= 0: nothing cancels).
// All statistics are fp32.
//
// The alternatives: every thread also keeps the largest class of its own slice of the row.  The k
// largest classes of a row lie in the slices of the k threads whose own largest are the k largest
// (a class elsewhere has k classes above it), so only those slices are read again.
// Classes are ordered by one 64-bit key, the value's bits made monotone above the complement of
// the class number: larger values first, equal ones by the lower class, no two keys alike.
#include "typed.h"

namespace avc {
namespace {

typedef unsigned long long u64;
constexpr int kMaxTop = 32;
constexpr float kFar = -200.0f;  // e^-200 is 0 in fp32: keeps 0 * -inf out of the sums

template <typename E>
constexpr int width() { return 16 / (int)sizeof(E); }

struct ProbArgs {
  long N, V;
  const void* z;
  long ldz;
  const long long* tokens;
  long long ignore;
  int top, nseg;
  long seg;  // classes of a segment
  float *logp, *entropy, *stats, *top_logp;
  long long* top_ids;
  float* part;   // [N][nseg][3]: m, s, u of a segment
  u64* part_top; // [N][nseg][top]: its classes in order, 0 behind the last
};

__device__ __forceinline__ u64 class_key(float z, long c) {
  if (!(z > -INFINITY)) z = -INFINITY;  // a NaN ranks as -inf
  const unsigned b = __float_as_uint(z + 0.0f);  // -0 -> +0
  return (u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xffffffffu - (unsigned)c);
}
__device__ __forceinline__ float key_value(u64 k) {
  const unsigned b = (unsigned)(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ long key_class(u64 k) { return 0xffffffffu - (unsigned)k; }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ u64 wave_max(u64 x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 y = __shfl_xor(x, o);
    x = y > x ? y : x;
  }
  return x;
}

struct Sums {
  float m = -INFINITY, s = 0.0f, u = 0.0f;
  // to the maximum `to` >= m (-inf: nothing seen yet)
  __device__ void move(float to) {
    const float d = fmaxf(m - (to == -INFINITY ? 0.0f : to), kFar);
    const float e = __expf(d);
    u = fmaf(d, s, u) * e;
    s *= e;
    m = to;
  }
  template <int N>
  __device__ void add(const float (&z)[N]) {
    float top = m;
#pragma unroll
    for (int k = 0; k < N; ++k) top = fmaxf(top, z[k]);
    move(top);
    const float mm = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float d = z[k] - mm;
      const float e = __expf(d);
      s += e;
      u = fmaf(e, fmaxf(d, kFar), u);
    }
  }
  __device__ void join_wave() {
    move(wave_max(m));
    s = wave_sum(s);
    u = wave_sum(u);
  }
};

// barrier among the GT threads that share a row (one wave's LDS operations stay in order)
template <int GT>
__device__ __forceinline__ void row_sync() {
  if (GT == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

template <int GT>
struct TopShared {
  static constexpr int kCap = GT == 64 ? 192 : 1024;  // candidates that are ranked at once
  u64 best[GT];
  int sel[kMaxTop];
  u64 tau;
  int count;
  u64 cand[kCap];
};

// The row segment's `k` largest keys in order, emit(rank, key).  best: the thread's largest key (0:
// its slice is empty); key_of(t, j): the j-th key of thread t's slice, j < per (0 past its end).
template <int GT, typename KeyOf, typename Emit>
__device__ void select_top(TopShared<GT>& sh, int tid, int k, u64 best, int per, KeyOf key_of, Emit emit) {
  sh.best[tid] = best;
  if (tid == 0) sh.tau = 1, sh.count = 0;
  row_sync<GT>();
  int rank = 0, held = 0;
  for (int i = 0; i < GT; ++i) {
    const u64 o = sh.best[i];
    rank += o > best;
    held += o != 0;
  }
  if (best != 0 && rank < k) {
    sh.sel[rank] = tid;
    if (rank == k - 1) sh.tau = best;
  }
  row_sync<GT>();
  const int nsel = min(k, held);
  const u64 tau = sh.tau;
  for (int i = tid; i < nsel * per; i += GT) {
    const u64 key = key_of(sh.sel[i / per], i % per);
    if (key >= tau) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < TopShared<GT>::kCap) sh.cand[at] = key;
    }
  }
  row_sync<GT>();
  const int n = sh.count;
  if (n <= TopShared<GT>::kCap) {
    // the candidates stand in any order; their ranks do not depend on it
    for (int i = tid; i < n; i += GT) {
      const u64 key = sh.cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += sh.cand[j] > key;
      if (r < k) emit(r, key);
    }
  } else {
    // many large classes in few slices: one class a round
    u64 under = ~0ull;
    for (int r = 0; r < k; ++r) {
      u64 mine = 0;
      for (int i = tid; i < nsel * per; i += GT) {
        const u64 key = key_of(sh.sel[i / per], i % per);
        if (key < under && key > mine) mine = key;
      }
      mine = wave_max(mine);
      if (GT > 64) {
        row_sync<GT>();
        if ((tid & 63) == 0) sh.best[tid >> 6] = mine;
        row_sync<GT>();
#pragma unroll
        for (int w = 0; w < GT / 64; ++w) mine = sh.best[w] > mine ? sh.best[w] : mine;
      }
      under = mine;
      if (tid == 0) emit(r, mine);
    }
  }
}

// one thread: the row's statistics and its token's log-probability
template <typename E>
__device__ void finish_row(const ProbArgs& a, long row, const Sums& t) {
  const bool empty = t.m == -INFINITY;  // (a NaN row has a NaN sum)
  const bool none = empty && t.s == 0.0f;
  const float logs = none ? 0.0f : logf(t.s);
  const float H = none ? 0.0f : logs - t.u / t.s;
  a.entropy[row] = H;
  if (a.stats) a.stats[row * 3] = t.m, a.stats[row * 3 + 1] = t.s, a.stats[row * 3 + 2] = H;
  const long long tok = a.tokens[row];
  float lp;
  if (tok == a.ignore) lp = 0.0f;
  else if (tok < 0 || tok >= a.V) lp = NAN;
  else if (none) lp = -INFINITY;
  else lp = ((float)static_cast<const E*>(a.z)[row * a.ldz + tok] - t.m) - logs;
  a.logp[row] = lp;
}
__device__ __forceinline__ void emit_top(const ProbArgs& a, long row, int r, u64 key, const Sums& t) {
  const float z = key_value(key);
  const bool none = t.m == -INFINITY && t.s == 0.0f;
  a.top_logp[row * a.top + r] = none ? -INFINITY : (z - t.m) - logf(t.s);
  a.top_ids[row * a.top + r] = key_class(key);
}

// GT threads a row segment, 256 / GT rows a workgroup (GT = 256: blockIdx.y is the segment).
template <typename E, int GT, bool TOP>
__global__ __launch_bounds__(256) void class_probs_forward_kernel(ProbArgs a) {
  constexpr int VEC = width<E>(), U = 4;
  const int grp = threadIdx.x / GT, tid = threadIdx.x % GT;
  const long row = (long)blockIdx.x * (256 / GT) + grp;
  if (row >= a.N) return;  // a whole wave (GT = 64) or, with one row a workgroup, never
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  const long c0 = (long)blockIdx.y * a.seg, c1 = c0 + a.seg < a.V ? c0 + a.seg : a.V;
  Sums t;
  float best = -INFINITY;
  long best_c = c0 + (long)tid * VEC;
  for (long c = c0 + (long)tid * VEC; c < c1; c += (long)GT * VEC * U) {
    float x[U * VEC];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const long ck = c + (long)k * GT * VEC;
      if (ck + VEC <= c1) {
        const Vec<E, VEC> r = vload<E, VEC>(z + ck);
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[k * VEC + v] = (float)r.v[v];
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[k * VEC + v] = ck + v < c1 ? (float)z[ck + v] : -INFINITY;
      }
    }
    t.add(x);
    if (TOP) {
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          if (x[k * VEC + v] > best) best = x[k * VEC + v], best_c = c + (long)k * GT * VEC + v;
    }
  }
  t.join_wave();
  if (GT > 64) {
    __shared__ float part[4][3];
    const int w = tid >> 6;
    if ((tid & 63) == 0) part[w][0] = t.m, part[w][1] = t.s, part[w][2] = t.u;
    __syncthreads();
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < GT / 64; ++i) m = fmaxf(m, part[i][0]);
    Sums all;
    all.m = m;
#pragma unroll
    for (int i = 0; i < GT / 64; ++i) {
      Sums p;
      p.m = part[i][0], p.s = part[i][1], p.u = part[i][2];
      p.move(m);
      all.s += p.s, all.u += p.u;
    }
    t = all;
  }
  const bool whole = a.nseg == 1;
  if (tid == 0) {
    if (whole) {
      finish_row<E>(a, row, t);
    } else {
      float* p = a.part + (row * a.nseg + blockIdx.y) * 3;
      p[0] = t.m, p[1] = t.s, p[2] = t.u;
    }
  }
  if (TOP) {
    __shared__ TopShared<GT> sh[256 / GT];
    const long n = c1 - c0;
    const int per = (int)((n + (long)GT * VEC - 1) / ((long)GT * VEC)) * VEC;
    const u64 mine = c0 + (long)tid * VEC < c1 ? class_key(best, best_c) : 0;
    u64* list = whole ? nullptr : a.part_top + (row * a.nseg + blockIdx.y) * a.top;
    if (!whole) {
      // a segment may hold fewer classes than are wanted
      for (long i = tid; i < a.top; i += GT)
        if (i >= n) list[i] = 0;
    }
    select_top<GT>(
        sh[grp], tid, a.top, mine, per,
        [&](int th, int j) -> u64 {
          const long c = c0 + ((long)(j / VEC) * GT + th) * VEC + j % VEC;
          return c < c1 ? class_key((float)z[c], c) : 0;
        },
        [&](int r, u64 key) {
          if (whole) emit_top(a, row, r, key, t);
          else list[r] = key;
        });
  }
}

// One wave a row: joins the segments' statistics and merges their lists (one lane a segment).
template <typename E>
__global__ __launch_bounds__(64) void class_probs_join_kernel(ProbArgs a) {
  const long row = blockIdx.x;
  const int lane = threadIdx.x;
  Sums t;
  if (lane < a.nseg) {
    const float* p = a.part + (row * a.nseg + lane) * 3;
    t.m = p[0], t.s = p[1], t.u = p[2];
  }
  t.join_wave();
  if (lane == 0) finish_row<E>(a, row, t);
  const u64* list = a.part_top + (row * a.nseg + lane) * a.top;
  int at = 0;
  u64 head = lane < a.nseg && a.top > 0 ? list[0] : 0;
  for (int r = 0; r < a.top; ++r) {
    const u64 key = wave_max(head);
    if (head == key) {
      emit_top(a, row, r, key, t);
      ++at;
      head = at < a.top ? list[at] : 0;
    }
  }
}

// dz = -p (dlogp + dentropy (log p + H)), + dlogp at the token: one read, one write.
template <typename E>
__global__ __launch_bounds__(256) void class_probs_backward_kernel(ProbArgs a, const float* dlogp,
                                                                   const float* dentropy, void* dz, long lddz,
                                                                   unsigned tiles) {
  constexpr int VEC = width<E>(), U = 2;
  const unsigned item = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const long row = item / tiles;
  if (row >= a.N) return;
  const long c0 = (long)(item % tiles) * (64 * VEC * U) + (threadIdx.x & 63) * VEC;
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  E* d = static_cast<E*>(dz) + row * lddz;
  const float m = a.stats[row * 3], s = a.stats[row * 3 + 1], H = a.stats[row * 3 + 2];
  const bool none = m == -INFINITY && s == 0.0f;
  const long long tok = a.tokens[row];
  const bool bad = tok != a.ignore && (tok < 0 || tok >= a.V);
  const float gl = !dlogp || tok == a.ignore ? 0.0f : bad ? NAN : dlogp[row];
  const float ge = dentropy ? dentropy[row] : 0.0f;
  const float inv = 1.0f / s, off = H - logf(s);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const long c = c0 + (long)k * 64 * VEC;
    if (c >= a.V) break;
    float x[VEC];
    const bool full = c + VEC <= a.V;
    if (full) {
      const Vec<E, VEC> r = vload<E, VEC>(z + c);
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = (float)r.v[v];
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = c + v < a.V ? (float)z[c + v] : 0.0f;
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float e = x[v] - m;
      const float p = __expf(e) * inv;
      float g = -p * fmaf(ge, fmaxf(e, kFar) + off, gl);
      if (c + v == tok) g += gl;
      x[v] = !none ? g : gl != gl ? gl : 0.0f;
    }
    if (full) {
      vstore<E, VEC>(d + c, x);
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (c + v < a.V) d[c + v] = static_cast<E>(x[v]);
    }
  }
}

constexpr long kWaveRow = 2048;  // up to this many classes one wave takes a row

// Segments of a row: rows enough to fill the chip take one workgroup each; fewer rows are cut, a
// segment no shorter than four vectors for each of its threads, at most one lane's worth in number.
int row_segments(long N, long V, int vec, long* seg) {
  *seg = V;
  if (V <= kWaveRow || N >= 512) return 1;
  const long least = 256L * vec * 4;
  long n = 512 / N;
  if (n > (V + least - 1) / least) n = (V + least - 1) / least;
  if (n > 64) n = 64;
  long len = (V + n - 1) / n;
  len = (len + vec - 1) / vec * vec;
  *seg = len;
  return (int)((V + len - 1) / len);
}

size_t probs_workspace(long N, long V, int top, int vec) {
  long seg;
  const int n = row_segments(N, V, vec, &seg);
  return n > 1 ? (size_t)N * n * (top * sizeof(u64) + 4 * sizeof(float)) : 0;
}

int check_rows(int dtype, long N, long V, long ldz) {
  AVC_CHECK_ARG(dtype_ok(dtype), "dtype is one of AVC_DTYPE_F32, _BF16, _F16");
  AVC_CHECK_ARG(N >= 0 && V >= 1, "N >= 0, V >= 1");
  AVC_CHECK_ARG(V <= 1L << 30 && N < 1L << 24, "N or V too large");
  AVC_CHECK_ARG(ldz >= V, "a row stride is smaller than V");
  return AVC_OK;
}

template <typename E, bool TOP>
int run_forward(ProbArgs a, hipStream_t s) {
  if (a.V <= kWaveRow) {
    class_probs_forward_kernel<E, 64, TOP><<<(unsigned)((a.N + 3) / 4), 256, 0, s>>>(a);
    AVC_LAUNCH_CHECK();
    return AVC_OK;
  }
  class_probs_forward_kernel<E, 256, TOP><<<dim3((unsigned)a.N, a.nseg), 256, 0, s>>>(a);
  AVC_LAUNCH_CHECK();
  if (a.nseg > 1) {
    class_probs_join_kernel<E><<<(unsigned)a.N, 64, 0, s>>>(a);
    AVC_LAUNCH_CHECK();
  }
  return AVC_OK;
}

}  // namespace
}  // namespace avc

using namespace avc;

extern "C" size_t avc_token_log_probs_workspace(int dtype, long N, long V, int top) {
  if (!dtype_ok(dtype) || N < 1 || V < 1 || top < 0 || top > kMaxTop) return 0;
  return probs_workspace(N, V, top, dtype == AVC_DTYPE_F32 ? width<float>() : width<__bf16>());
}

extern "C" int avc_token_log_probs_forward(int dtype, long N, long V, const void* logits, long ldz,
                                           const long long* tokens, long long ignore_index, int top, float* logp,
                                           float* entropy, float* stats, float* top_logp, long long* top_ids,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  AVC_TRY(check_rows(dtype, N, V, ldz));
  AVC_CHECK_ARG(top >= 0 && top <= kMaxTop && top <= V, "top is 0 .. min(32, V)");
  if (N == 0) return AVC_OK;
  AVC_CHECK_ARG(logits && tokens && logp && entropy, "logits, tokens, logp and entropy are needed");
  AVC_CHECK_ARG(top == 0 || (top_logp && top_ids), "top > 0 needs top_logp and top_ids");
  const int vec = dtype == AVC_DTYPE_F32 ? width<float>() : width<__bf16>();
  const size_t need = probs_workspace(N, V, top, vec);
  AVC_CHECK_ARG(workspace_bytes >= need && (need == 0 || workspace),
                "workspace smaller than avc_token_log_probs_workspace");
  ProbArgs a{};
  a.N = N, a.V = V, a.z = logits, a.ldz = ldz, a.tokens = tokens, a.ignore = ignore_index, a.top = top;
  a.nseg = row_segments(N, V, vec, &a.seg);
  a.logp = logp, a.entropy = entropy, a.stats = stats, a.top_logp = top_logp, a.top_ids = top_ids;
  a.part_top = static_cast<u64*>(workspace);
  a.part = reinterpret_cast<float*>(a.part_top + (size_t)N * a.nseg * top);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return top ? run_forward<E, true>(a, s) : run_forward<E, false>(a, s);
  });
}

extern "C" int avc_token_log_probs_backward(int dtype, long N, long V, const void* logits, long ldz,
                                            const long long* tokens, long long ignore_index, const float* stats,
                                            const float* dlogp, const float* dentropy, void* dlogits, long lddz,
                                            void* stream) {
  AVC_TRY(check_rows(dtype, N, V, ldz));
  AVC_CHECK_ARG(lddz >= V, "a row stride is smaller than V");
  if (N == 0) return AVC_OK;
  AVC_CHECK_ARG(logits && tokens && stats && dlogits, "logits, tokens, stats and dlogits are needed");
  ProbArgs a{};
  a.N = N, a.V = V, a.z = logits, a.ldz = ldz, a.tokens = tokens, a.ignore = ignore_index;
  a.stats = const_cast<float*>(stats);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return with_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    const long tile = 64L * width<E>() * 2, tiles = (V + tile - 1) / tile;
    AVC_CHECK_ARG(N <= (1L << 25) / tiles, "N * V too large");
    class_probs_backward_kernel<E><<<(unsigned)((N * tiles + 3) / 4), 256, 0, s>>>(a, dlogp, dentropy, dlogits, lddz,
                                                                                 (unsigned)tiles);
    AVC_LAUNCH_CHECK();
    return AVC_OK;
  });
}
