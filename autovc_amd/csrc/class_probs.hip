// Log-probabilities of given classes under rows of logits, with each row's entropy and its most
// probable classes.  One pass over the logits keeps, for every thread, the maximum m so far and the
// sums of e^(z - m) and e^(z - m) (z - m), moved to a new maximum m' by
//   s' = s e^(m - m'),   u' = (u + (m - m') s) e^(m - m').
// With the largest class kept apart (s = 1 + rest),
//   log p_i = (z_i - m) - log1p(rest),   entropy = log1p(rest) - u / s   (both terms >= 0),
// and the gradient needs log p_i + entropy = (z_i - m) - u / s: nothing cancels.
// All statistics are fp32.
//
// The alternatives: every thread also keeps the largest class of its own slice of the row.  The k
// largest classes of a row lie in the slices of the k threads whose own largest are the k largest
// (a class elsewhere has k classes above it), so only those slices are read again.
// Classes are ordered by one 64-bit key, the value's bits made monotone above the complement of
// the class number: larger values first, equal ones by the lower class, no two keys alike.
#include <algorithm>
#include <climits>
#include <utility>

#include "typed.h"

namespace avc {
namespace {

typedef unsigned long long u64;
constexpr int kMaxTop = 32;
constexpr int kMaxSeg = 64;  // segments of a row: lanes of the wave that joins them
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
  float* part;   // [N][nseg][4]: Sums of a segment
  u64* part_top; // [N][nseg][top]: its classes in order, 0 behind the last
};

// (never 0, which stands for no class)
__device__ __forceinline__ unsigned value_bits(float z) {
  if (!(z > -INFINITY)) z = -INFINITY;  // a NaN ranks as -inf
  const unsigned b = __float_as_uint(z + 0.0f);  // -0 -> +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 class_key(float z, long c) {
  return (u64)value_bits(z) << 32 | (0xffffffffu - (unsigned)c);
}
__device__ __forceinline__ float key_value(u64 k) {
  const unsigned b = (unsigned)(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ long key_class(u64 k) { return 0xffffffffu - (unsigned)k; }

// Reductions over a wave by data-parallel-primitive moves (a few cycles a step, where a shuffle
// through the LDS crossbar takes some hundred): after four shifts the last lane of each row of 16
// holds its row, two broadcasts join the rows in lane 63.  The order is the same in every run.
// `none`, which the op leaves any value with, stands in for lanes that a move does not reach.
template <typename Op>
__device__ __forceinline__ int dpp_reduce(int x, int none, Op op) {
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x111, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x112, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x114, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x118, 0xf, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x142, 0xa, 0xf, false));
  x = op(x, __builtin_amdgcn_update_dpp(none, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ float wave_sum(float x) {
  return __int_as_float(dpp_reduce(__float_as_int(x), 0, [](int p, int q) {
    return __float_as_int(__int_as_float(p) + __int_as_float(q));
  }));
}
// (as integers of the same order: a float maximum would first quiet what a move has brought)
__device__ __forceinline__ float wave_max(float x) {
  auto ordered = [](int b) { return b ^ ((b >> 31) & 0x7fffffff); };
  return __int_as_float(ordered(dpp_reduce(ordered(__float_as_int(x)), INT_MIN, [](int p, int q) { return max(p, q); })));
}
__device__ __forceinline__ u64 wave_max(u64 x) {
  auto most = [](unsigned p) {
    return (unsigned)dpp_reduce((int)p, 0, [](int a, int b) { return (int)max((unsigned)a, (unsigned)b); });
  };
  const unsigned hi = most((unsigned)(x >> 32));
  return (u64)hi << 32 | most((unsigned)(x >> 32) == hi ? (unsigned)x : 0u);
}

// What a part of a row adds up to, about the largest logit m seen: s = sum e^(z - m) over the classes
// below m, c = the classes at m, u = sum e^(z - m) (z - m).  The largest class is kept out of s
// because the rest is what a confident row's entropy and log-probability are made of: in a sum
// that begins with its 1 they would lose what lies below 2^-24.  A wave's lanes share m, so that
// classes at or above it are a branch that a wave seldom takes.
struct Sums {
  float m = -INFINITY, s = 0.0f, c = 0.0f, u = 0.0f;
  // to a maximum `to` > m (or a part that has seen nothing)
  __device__ __forceinline__ void move(float to) {
    const float d = fmaxf(m - to, kFar);
    const float e = __expf(d), all = s + c;
    u = fmaf(d, all, u) * e;
    s = all * e;
    c = 0.0f;
    m = to;
  }
  // the wave's next N classes a lane; `own`, the largest of the lane's
  template <int N>
  __device__ __forceinline__ void add(const float (&z)[N], float& own) {
    float top = z[0];
#pragma unroll
    for (int k = 1; k < N; ++k) top = fmaxf(top, z[k]);
    own = fmaxf(own, top);
    if (!__any(top >= m)) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float d = __builtin_elementwise_maximum(z[k] - m, kFar);  // (a NaN passes)
        const float e = __expf(d);
        s += e;
        u = fmaf(e, d, u);
      }
      return;
    }
    const float most = wave_max(top);
    if (most > m) move(most);
    const float mm = m == -INFINITY ? 0.0f : m;
    float below = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float d = __builtin_elementwise_maximum(z[k] - mm, kFar);
      const float e = __expf(d);
      const float less = __builtin_amdgcn_fmed3f(d * -0x1p126f, 0.0f, 1.0f);  // 0 at m, else 1
      s = fmaf(e, less, s);
      below += less;
      u = fmaf(e, d, u);
    }
    c += (float)N - below;
  }
  __device__ __forceinline__ void join_wave() {
    s = wave_sum(s);
    u = wave_sum(u);
    // Mostly one lane holds the one class at m.  (c is no whole number where a class lies less than 2^-126
    // below m: `less` is a part of 1 then, and s and c hold such a class's term together.)
    c = __any(c != 0.0f && c != 1.0f) ? wave_sum(c) : (float)__popcll(__ballot(c == 1.0f));
  }
};

// A row's result: its largest logit, the others' sum against it, and the mean of m - z under p
struct RowStats {
  float m, rest, mean;
  bool none;  // nothing left in the row (a NaN row has a NaN sum)
  __device__ explicit RowStats(const Sums& t) : m(t.m) {
    none = t.m == -INFINITY && t.s == 0.0f;
    rest = none ? 0.0f : t.s + (t.c - 1.0f);
    mean = none ? 0.0f : -t.u / (1.0f + rest);
  }
  __device__ explicit RowStats(const float* p) : m(p[0]), rest(p[1]), mean(p[2]) { none = m == -INFINITY && rest == 0.0f; }
  __device__ float log_sum() const { return log1pf(rest); }
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

// The wave's k-th largest value, bit by bit (0 where fewer than k lanes are above 0).
template <typename T>
__device__ __forceinline__ T wave_kth(T x, int k) {
  T least = 0;
  for (T bit = (T)1 << (sizeof(T) * 8 - 1); bit; bit >>= 1)
    if (__popcll(__ballot(x >= (least | bit))) >= k) least |= bit;
  return least;
}
// Appends the lanes' keys for which `in` holds to a list in LDS that has room for cap: one atomic
// a wave.  `count` goes on counting past cap.
__device__ __forceinline__ void append(u64* list, int* count, int cap, bool in, u64 key) {
  const u64 m = __ballot(in);
  if (!in) return;
  const int lane = threadIdx.x & 63, first = __ffsll(m) - 1;
  int at = 0;
  if (lane == first) at = atomicAdd(count, __popcll(m));
  at = __shfl(at, first) + __popcll(m & ((1ull << lane) - 1));
  if (at < cap) list[at] = key;
}

template <int GT>
struct TopShared {
  // Candidates that are ranked at once: all of a dense row with fewer than kMaxTop slices in a wave, 31 of 8
  // classes at most (1x200 fp16 classes with 32 alternatives 17 us; with a list of 128, a class a round, 31)
  static constexpr int kCap = 256;
  u64 cand[kCap];
  unsigned tau;
  int count, nsel;
  int ties[GT / 64];
  short sel[GT];
};
// n keys in any order: those whose rank is below k go out with it
template <int GT, typename Emit>
__device__ __forceinline__ void rank_out(const u64* cand, int n, int tid, int k, Emit emit) {
  for (int i = tid; i < n; i += GT) {
    const u64 key = cand[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += cand[j] > key;
    if (r < k) emit(r, key);
  }
}

// The `k` largest keys of classes c0 .. c1-1 in order, emit(rank, key).  mine: the largest value_bits
// of the thread's slice (0: empty); a slice is the thread's vectors, GT vectors apart.  Only slices
// whose largest is at least a value that k classes are known to reach can hold one of the k.
template <typename E, int GT, typename Emit>
__device__ void select_top(TopShared<GT>& sh, int tid, int k, unsigned mine, const E* z, long c0, long c1, Emit emit) {
  constexpr int VEC = width<E>(), kCap = TopShared<GT>::kCap;
  const int lane = tid & 63, wave = tid >> 6;
  if (tid == 0) sh.tau = 1, sh.count = 0, sh.nsel = 0;
  row_sync<GT>();
  // k of a wave's slices reach its k-th best, so the largest of those is reached by k in all
  const unsigned kth = wave_kth(mine, k);
  if (lane == 0) atomicMax(&sh.tau, kth);
  row_sync<GT>();
  const unsigned tau = sh.tau;
  if (mine >= tau) sh.sel[atomicAdd(&sh.nsel, 1)] = (short)tid;
  row_sync<GT>();
  const int nsel = sh.nsel;
  const long rounds = (c1 - c0 + (long)GT * VEC - 1) / ((long)GT * VEC);
  auto vector = [&](long c, float (&x)[VEC]) {
    if (c + VEC <= c1) {
      const Vec<E, VEC> r = vload<E, VEC>(z + c);
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = (float)r.v[v];
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[v] = c + v < c1 ? (float)z[c + v] : 0.0f;
    }
  };
  // 2^lg lanes a slice, a vector a lane
  int lg = 0;
  while (lg < 6 && (1 << lg) < rounds) ++lg;
  auto slices = [&](auto take) {
    for (int i = tid >> lg; i < nsel; i += GT >> lg) {
      const int th = sh.sel[i];
      for (long q = tid & ((1 << lg) - 1); q < rounds; q += 1 << lg) {
        const long c = c0 + (q * GT + th) * VEC;
        float x[VEC];
        vector(c, x);
#pragma unroll
        for (int v = 0; v < VEC; ++v) take(c + v < c1, x[v], c + v);
      }
    }
  };
  // (tau is -inf's where fewer than k classes are left, all the others being equal then, and below it, at 1,
  // where no wave has k slices: every class is above it)
  if (tau > value_bits(-INFINITY)) {
    slices([&](bool in, float x, long c) {
      append(sh.cand, &sh.count, kCap, in && value_bits(x) >= tau, class_key(x, c));
    });
    row_sync<GT>();
    if (sh.count <= kCap) {
      rank_out<GT>(sh.cand, sh.count, tid, k, emit);
      return;
    }
  }
  // More candidates than fit: classes equal to tau, as where fewer than k are not ruled out.  Those
  // above it go first, then the lowest of the equal ones, looked for from the row's beginning.
  row_sync<GT>();
  if (tid == 0) sh.count = 0;
  row_sync<GT>();
  slices([&](bool in, float x, long c) {
    append(sh.cand, &sh.count, kCap, in && value_bits(x) > tau, class_key(x, c));
  });
  row_sync<GT>();
  const int above = sh.count;
  if (above <= kCap) {
    int have = above;
    for (long base = c0; base < c1 && have < k; base += (long)GT * VEC) {
      const long c = base + (long)tid * VEC;
      float x[VEC];
      vector(c, x);
      int before = 0, total = 0;
      bool tie[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        tie[v] = c + v < c1 && value_bits(x[v]) == tau;
        const u64 m = __ballot(tie[v]);
        before += __popcll(m & ((1ull << lane) - 1));
        total += __popcll(m);
      }
      if (GT > 64) {
        row_sync<GT>();
        if (lane == 0) sh.ties[wave] = total;
        row_sync<GT>();
        total = 0;
        for (int w = 0; w < GT / 64; ++w) {
          if (w < wave) before += sh.ties[w];
          total += sh.ties[w];
        }
      }
      int at = have + before;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (tie[v]) {
          if (at < k) sh.cand[at] = class_key(x[v], c + v);
          ++at;
        }
      }
      have += total;
    }
    row_sync<GT>();
    rank_out<GT>(sh.cand, above > k ? above : have < k ? have : k, tid, k, emit);
    return;
  }
  // many different large classes in few slices: one class a round
  u64 under = ~0ull;
  for (int r = 0; r < k; ++r) {
    u64 most = 0;
    slices([&](bool in, float x, long c) {
      const u64 key = class_key(x, c);
      if (in && key < under && key > most) most = key;
    });
    most = wave_max(most);
    if (GT > 64) {
      row_sync<GT>();
      if (lane == 0) sh.cand[wave] = most;  // (the candidates are not used any more)
      row_sync<GT>();
      for (int w = 0; w < GT / 64; ++w) most = sh.cand[w] > most ? sh.cand[w] : most;
    }
    under = most;
    if (tid == 0 && most != 0) emit(r, most);
  }
}

// a row's token and its logit, asked for before the row is read
struct Token {
  long long tok;
  float z;
  template <typename E>
  __device__ Token(const ProbArgs& a, long row, const E* logits) {
    tok = a.tokens[row];
    z = (float)logits[tok >= 0 && tok < a.V ? tok : 0];
  }
};

// one thread: the row's statistics and its token's log-probability
__device__ __forceinline__ void finish_row(const ProbArgs& a, long row, const RowStats& t, const Token& k) {
  const float logs = t.log_sum();
  a.entropy[row] = logs + t.mean;
  if (a.stats) a.stats[row * 3] = t.m, a.stats[row * 3 + 1] = t.rest, a.stats[row * 3 + 2] = t.mean;
  float lp;
  if (k.tok == a.ignore) lp = 0.0f;
  else if (k.tok < 0 || k.tok >= a.V) lp = NAN;
  else if (t.none) lp = -INFINITY;
  else lp = (k.z - t.m) - logs;
  a.logp[row] = lp;
}
__device__ __forceinline__ void emit_top(const ProbArgs& a, long row, int r, u64 key, const RowStats& t) {
  a.top_logp[row * a.top + r] = t.none ? -INFINITY : (key_value(key) - t.m) - t.log_sum();
  a.top_ids[row * a.top + r] = key_class(key);
}

// GT threads a row segment: a wave, four of them a workgroup, or a workgroup of 256 (blockIdx.y is
// the segment).  A thread reads U vectors at a time and asks for the next U before it adds the first.
// Bound by the one read of the logits: 4096 rows of 50001 bf16 classes alone 83 us, 4.9 TB/s (73 traced);
// in a training pass, behind a backward whose writes are still on their way to memory, 106.  Few rows are
// bound by the chain of load, reduction and store: one of 512 fp32 classes with 5 alternatives 5 us.
template <int GT>
constexpr int kRows = GT == 64 ? 4 : 1;  // rows of a workgroup

template <typename E, int GT, bool TOP>
__global__ __launch_bounds__(GT * kRows<GT>) void class_probs_forward_kernel(ProbArgs a) {
  constexpr int VEC = width<E>(), U = 2;
  constexpr long kRound = (long)GT * VEC * U;
  const int grp = GT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / GT) : 0, tid = threadIdx.x % GT;
  const long row = (long)blockIdx.x * kRows<GT> + grp;
  if (row >= a.N) return;  // a whole wave (GT = 64) or, with one row a workgroup, never
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  const long c0 = (long)blockIdx.y * a.seg, c1 = c0 + a.seg < a.V ? c0 + a.seg : a.V;
  const Token token(a, row, z);
  Sums t;
  float own = -INFINITY;  // the largest of the thread's classes
  Vec<E, VEC> r[U];
  long c = c0;
  auto load = [&](long from) {
#pragma unroll
    for (int k = 0; k < U; ++k) r[k] = vload<E, VEC>(z + from + (k * GT + tid) * VEC);
  };
  if (c + kRound <= c1) load(c);
  for (; c + kRound <= c1; c += kRound) {
    float x[U][VEC];
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[k][v] = (float)r[k].v[v];
    if (c + 2 * kRound <= c1) load(c + kRound);
    t.add(reinterpret_cast<const float(&)[U * VEC]>(x), own);
  }
  if (c < c1) {  // less than a round is left, its last vector perhaps cut
    float x[U][VEC];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const long ck = c + (k * GT + tid) * VEC;
      if (ck + VEC <= c1) {
        const Vec<E, VEC> q = vload<E, VEC>(z + ck);
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[k][v] = (float)q.v[v];
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[k][v] = ck + v < c1 ? (float)z[ck + v] : -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (c + (long)k * GT * VEC >= c1) break;
      t.add(x[k], own);
    }
  }
  t.join_wave();
  if (GT > 64) {
    __shared__ float part[GT / 64][4];
    const int w = tid >> 6;
    if ((tid & 63) == 0) part[w][0] = t.m, part[w][1] = t.s, part[w][2] = t.c, part[w][3] = t.u;
    __syncthreads();
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < GT / 64; ++i) m = fmaxf(m, part[i][0]);
    Sums all;
    all.m = m;
#pragma unroll
    for (int i = 0; i < GT / 64; ++i) {
      Sums p;
      p.m = part[i][0], p.s = part[i][1], p.c = part[i][2], p.u = part[i][3];
      if (m > p.m) p.move(m);
      all.s += p.s, all.c += p.c, all.u += p.u;
    }
    t = all;
  }
  const bool whole = a.nseg == 1;
  if (tid == 0) {
    if (whole) {
      finish_row(a, row, RowStats(t), token);
    } else {
      float* p = a.part + (row * a.nseg + blockIdx.y) * 4;
      p[0] = t.m, p[1] = t.s, p[2] = t.c, p[3] = t.u;
    }
  }
  if (TOP) {
    __shared__ TopShared<GT> sh[kRows<GT>];
    const unsigned mine = c0 + (long)tid * VEC < c1 ? value_bits(own) : 0;
    u64* list = whole ? nullptr : a.part_top + (row * a.nseg + blockIdx.y) * a.top;
    if (!whole && tid < a.top && tid >= c1 - c0) list[tid] = 0;  // a segment may hold fewer classes than are wanted
    const RowStats st(t);
    select_top<E, GT>(sh[grp], tid, a.top, mine, z, c0, c1, [&](int r, u64 key) {
      if (whole) emit_top(a, row, r, key, st);
      else list[r] = key;
    });
  }
}

// Many rows of at most kShort classes: a wave takes four of them, 16 lanes each, whole in registers,
// which spares three quarters of what a row costs beside its classes (reductions, logarithms) -- with
// a wave a row that is what bounds it.  35200 rows of 512 fp32 classes 14.6 us (4.9 TB/s, the rate of a
// large copy), with a wave a row 19.9; with 5 alternatives 26 and 38; 60000 rows of 100 fp32 classes with
// 5 alternatives 18 and 57.  (Where it does not: short_rows.)
constexpr int kShort = 512;
constexpr int kShortCand = 64;  // candidates of a row that are ranked at once

// the value J lanes round the lane's 16
template <int J>
__device__ __forceinline__ float turned(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + J, 0xf, 0xf, true));
}
// a sum or maximum over 16 lanes, the same bits in each of them
template <typename Op>
__device__ __forceinline__ float reduce16(float x, Op op) {
  x = op(x, turned<8>(x));
  x = op(x, turned<4>(x));
  x = op(x, turned<2>(x));
  return op(x, turned<1>(x));
}
__device__ __forceinline__ float max16(float x) {
  return reduce16(x, [](float p, float q) { return fmaxf(p, q); });
}
// how many of the other 15 lanes' values are at least v
template <int... J>
__device__ __forceinline__ int at_least(float x, float v, std::integer_sequence<int, J...>) {
  return (0 + ... + (int)(turned<J + 1>(x) >= v));
}
// A value that k of a row's classes are known to reach, the highest that the lanes' R largest tell
// (-inf where they do not).
template <int R, int M>
__device__ __forceinline__ float reached(const float (&x)[M], int k) {
  float best[R];
#pragma unroll
  for (int r = 0; r < R; ++r) best[r] = -INFINITY;
#pragma unroll
  for (int i = 0; i < M; ++i) {
    float v = R == 1 ? x[i] : fmaxf(x[i], -INFINITY);  // (a NaN ranks as -inf)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float less = fminf(best[r], v);
      best[r] = fmaxf(best[r], v);
      v = less;
    }
  }
  float tau = -INFINITY;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    int n = r + 1;
#pragma unroll
    for (int q = 0; q < R; ++q)
      n += at_least(best[q], best[r], std::make_integer_sequence<int, 15>()) + (q > r && best[q] >= best[r]);
    if (n >= k) tau = fmaxf(tau, best[r]);
  }
  return max16(tau);
}

// select_top for a row that 16 lanes hold: x[i] is class (i / VEC) 16 VEC + l VEC + i % VEC of V.
// `live`: the row exists.
template <typename E, int M, typename Emit>
__device__ void select_short(u64* cand, int k, const float (&x)[M], const E* z, int V, bool live, Emit emit) {
  constexpr int VEC = width<E>();
  const int lane = threadIdx.x & 63, l = lane & 15, shift = lane & 48;
  auto class_of = [&](int i) { return i / VEC * 16 * VEC + l * VEC + i % VEC; };
  // the lanes of the row for which `in` holds: those before this one, and all
  auto count = [&](bool in, int& before) {
    const unsigned m = (unsigned)(__ballot(in) >> shift) & 0xffffu;
    before = __popc(m & ((1u << l) - 1));
    return __popc(m);
  };
  // of as many of the lanes' largest as let about k, and seldom more than the list holds, reach it
  const float tau = k <= 8 ? reached<1>(x, k) : k <= 16 ? reached<2>(x, k) : reached<4>(x, k);
  int n = 0;
  auto gather = [&](auto wanted) {
    n = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const bool in = wanted(x[i]);
      if (!__any(in)) continue;
      int before;
      const int all = count(in, before);
      if (in && n + before < kShortCand) cand[n + before] = class_key(x[i], class_of(i));
      n += all;
    }
    row_sync<64>();
  };
  auto rank = [&](int n) {
    for (int i = l; i < n; i += 16) {
      const u64 key = cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += cand[j] > key;
      if (r < k && live) emit(r, key);
    }
    row_sync<64>();
  };
  const bool some = tau > -INFINITY;
  if (__any(some)) gather([&](float v) { return some && v >= tau; });
  const bool few = some && n <= kShortCand;
  if (__any(few)) rank(few ? n : 0);
  if (!__any(!few)) return;
  // as in select_top: those above tau, then the first of those at tau
  gather([&](float v) { return !few && v > tau; });
  const bool ties = !few && n <= kShortCand;
  int have = ties ? n : k;
  for (int base = 0; __any(have < k && base < V); base += 16) {
    const int c = base + l;
    const float v = c < V ? (float)z[c] : 0.0f;
    int before;
    const bool in = have < k && c < V && value_bits(v) == value_bits(tau);
    const int all = count(in, before);
    if (in && have + before < k) cand[have + before] = class_key(v, c);
    have += all;
  }
  row_sync<64>();
  rank(ties ? (n > k ? n : k) : 0);
  if (!__any(!few && !ties)) return;
  u64 under = !few && !ties ? ~0ull : 0;
  for (int r = 0; r < k; ++r) {
    u64 most = 0;
#pragma unroll 1
    for (int c = l; c < V; c += 16) {
      const u64 key = class_key((float)z[c], c);
      if (key < under && key > most) most = key;
    }
    for (int by = 8; by; by >>= 1) {
      const u64 other = __shfl_xor(most, by);
      most = other > most ? other : most;
    }
    under = most;
    if (l == 0 && live && most != 0) emit(r, most);
  }
}

template <typename E, int NV, bool TOP>
__global__ __launch_bounds__(256) void class_probs_short_kernel(ProbArgs a) {
  constexpr int VEC = width<E>(), kAcross = 16 * VEC;
  const int l = threadIdx.x & 15;
  const long at = (long)blockIdx.x * 16 + (threadIdx.x >> 4), row = at < a.N ? at : a.N - 1;
  const E* z = static_cast<const E*>(a.z) + row * a.ldz;
  const int V = (int)a.V;
  const Token token(a, row, z);
  float x[NV * VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = k * kAcross + l * VEC;
    if (c + VEC <= V) {
      const Vec<E, VEC> r = vload<E, VEC>(z + c);
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[k * VEC + v] = (float)r.v[v];
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) x[k * VEC + v] = c + v < V ? (float)z[c + v] : -INFINITY;
    }
  }
  Sums t;
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) t.m = fmaxf(t.m, x[i]);
  t.m = max16(t.m);
  const float mm = t.m == -INFINITY ? 0.0f : t.m;
  float below = 0.0f;
#pragma unroll
  for (int i = 0; i < NV * VEC; ++i) {
    const float d = __builtin_elementwise_maximum(x[i] - mm, kFar);  // (a NaN passes)
    const float e = __expf(d);
    const float less = __builtin_amdgcn_fmed3f(d * -0x1p126f, 0.0f, 1.0f);  // 0 at m, else 1
    t.s = fmaf(e, less, t.s);
    below += less;
    t.u = fmaf(e, d, t.u);
  }
  auto plus = [](float p, float q) { return p + q; };
  t.s = reduce16(t.s, plus);
  t.u = reduce16(t.u, plus);
  t.c = NV * kAcross - reduce16(below, plus);
  const RowStats st(t);
  if (l == 0 && at < a.N) finish_row(a, row, st, token);
  if (TOP) {
    __shared__ u64 cand[16][kShortCand];
    select_short<E>(cand[threadIdx.x >> 4], a.top, x, z, V, at < a.N,
                    [&](int r, u64 key) { emit_top(a, row, r, key, st); });
  }
}

// One workgroup a row: the first wave joins the segments' statistics (a lane a segment); of the
// segments' lists the keys that can be among the first `top` are ranked.  5 rows of 151001 fp16 classes
// with 20 alternatives: 9 to 10 us for the segments and 5.6 for this, both chains of a few dependent steps.
template <typename E>
__global__ __launch_bounds__(256) void class_probs_join_kernel(ProbArgs a) {
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  __shared__ float whole[3];
  __shared__ u64 tau;
  __shared__ int count;
  __shared__ u64 cand[kMaxSeg * kMaxTop];
  const u64* list = a.part_top + row * a.nseg * a.top;
  const int keys = a.nseg * a.top;
  u64 key[kMaxSeg * kMaxTop / 256];
#pragma unroll
  for (int i = 0; i < kMaxSeg * kMaxTop / 256; ++i) key[i] = i * 256 + tid < keys ? list[i * 256 + tid] : 0;
  if (tid < 64) {
    const Token token(a, row, static_cast<const E*>(a.z) + row * a.ldz);
    const bool has = tid < a.nseg && a.top > 0;
    const u64 head = has ? list[(long)tid * a.top] : 0, tail = has ? list[(long)tid * a.top + a.top - 1] : 0;
    Sums t;
    if (tid < a.nseg) {
      const float* p = a.part + (row * a.nseg + tid) * 4;
      t.m = p[0], t.s = p[1], t.c = p[2], t.u = p[3];
    }
    const float most = wave_max(t.m);
    if (most > t.m) t.move(most);
    t.join_wave();
    // a.top keys reach the a.top-th of the segments' first keys, and the last key of any one segment
    const u64 kth = a.top > 0 ? wave_kth(head, a.top) : 0, own = wave_max(tail);
    if (tid == 0) {
      const RowStats st(t);
      finish_row(a, row, st, token);
      whole[0] = st.m, whole[1] = st.rest, whole[2] = st.mean;
      tau = kth > own ? kth : own ? own : 1, count = 0;
    }
  }
  if (a.top == 0) return;
  __syncthreads();
  const RowStats t(whole);
#pragma unroll
  for (int i = 0; i < kMaxSeg * kMaxTop / 256; ++i)
    append(cand, &count, kMaxSeg * kMaxTop, key[i] >= tau, key[i]);
  __syncthreads();
  rank_out<256>(cand, count, tid, a.top, [&](int r, u64 k) { emit_top(a, row, r, k, t); });
}

// dz = dlogp (onehot - p) - dentropy p ((z - m) + mean): one read, one write, and bound by them (4096
// rows of 50001 bf16 classes 175 us, 4.7 TB/s); a wave takes two vectors a lane of a row, so the rows'
// lengths do not matter to the balance.  1 - p of the largest class is rest / (1 + rest).
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
  const RowStats t(a.stats + row * 3);
  const long long tok = a.tokens[row];
  const bool bad = tok != a.ignore && (tok < 0 || tok >= a.V);
  const float gl = !dlogp || tok == a.ignore ? 0.0f : bad ? NAN : dlogp[row];
  const float ge = dentropy ? dentropy[row] : 0.0f;
  const float inv = 1.0f / (1.0f + t.rest);
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
      const float e = x[v] - t.m;
      const float p = __expf(e) * inv;
      const float through = ge * (fmaxf(e, kFar) + t.mean);
      float g = -p * (through + gl);
      if (c + v == tok) g = fmaf(gl, e == 0.0f ? t.rest * inv : 1.0f - p, -p * through);
      x[v] = !t.none ? g : gl != gl ? gl : 0.0f;
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

// Whether 16 lanes take a row (fewer rows than 4096 take 5 to 7 us either way).  With more than 16 alternatives
// of more than kShort / 2 classes their list costs most, and a wave a row, which in fp32 has as many slices as
// it can, is faster while rows are few or their classes many.  16 lanes and a wave, us, with 20 and 32:
//   fp32  4096x300  10.1  8.9  11.6  9.6    8192x384  14.2 13.7  15.7 14.5    12000x384 18.0 18.0  19.4 19.3
//         4096x512  11.1  9.1  12.5  9.6   12000x512  18.7 17.4  20.6 18.2    35200x512 41.4 40.1  45.8 42.5
//        35200x300  37.7 40.8  41.8 42.9   35200x448  39.7 41.8  43.8 44.2
//   bf16  4096x300  10.8 10.9  12.3 13.6    4096x512  11.0 10.2  12.4 10.8     8192x512 14.1 16.3  15.9 17.0
// (4096x512 fp32 with 16: 9.6 and 8.8; 4096x256 with 32: 9.6 and 8.9.)
bool short_rows(long N, long V, int top, int vec) {
  if (V > kShort) return false;
  if (top <= 16 || V <= kShort / 2) return N >= 4096;
  return vec == 4 ? N >= 12000 && V <= 448 : N >= (V <= 384 ? 4096 : 8192);
}

// A wave takes a row where rows are short, or many enough to fill the chip so (4096 rows of 50001
// bf16 classes alone: 83 us, with a workgroup a row 90); else a workgroup does.
bool wave_rows(long N, long V) { return V <= 2048 || N >= 4096; }

// Segments of a row: where there are few long rows (below 16 rounds of a workgroup the second launch
// costs more than it gives: 64 rows of 8192 fp32 classes 8.3 us cut, 5.3 whole) each is cut until the
// chip is full, into pieces of two rounds at least (5 rows of 151001 fp16 classes with 20 alternatives:
// pieces of two rounds 14.0 us, of four 21.9, of eight 20.5; without alternatives 8 us each way).
int row_segments(long N, long V, int vec, long* seg) {
  *seg = V;
  const long round = 256L * vec;
  if (wave_rows(N, V) || N >= 512 || V < 16 * round) return 1;
  long n = 512 / N;
  if (n > (V + 2 * round - 1) / (2 * round)) n = (V + 2 * round - 1) / (2 * round);
  if (n > kMaxSeg) n = kMaxSeg;
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
  AVC_CHECK_ARG(V <= 1L << 30 && N <= 1L << 40, "N or V too large");
  AVC_CHECK_ARG(ldz >= V, "a row stride is smaller than V");
  return AVC_OK;
}

// More rows than a grid takes go in launches of nearly equal parts, each with rows enough for the whole's
// layout.  (a is the part: its first row and number of rows set)
template <typename E, typename Launch>
int in_parts(const ProbArgs& all, long most, Launch launch) {
  const long parts = (all.N + most - 1) / most, per = (all.N + parts - 1) / parts;
  for (long r = 0; r < all.N; r += per) {
    ProbArgs a = all;
    a.N = std::min(per, all.N - r);
    a.z = static_cast<const E*>(all.z) + r * all.ldz;
    a.tokens = all.tokens + r;
    if (all.stats) a.stats = all.stats + r * 3;
    AVC_TRY(launch(a, r));
  }
  return AVC_OK;
}

template <typename E, bool TOP>
int run_forward(ProbArgs a, hipStream_t s) {
  if (short_rows(a.N, a.V, a.top, width<E>())) {
    constexpr int most = kShort / 16 / width<E>();  // vectors a lane
    const unsigned grid = (unsigned)((a.N + 15) / 16);
    if (a.V <= kShort / 4) class_probs_short_kernel<E, most / 4, TOP><<<grid, 256, 0, s>>>(a);
    else if (a.V <= kShort / 2) class_probs_short_kernel<E, most / 2, TOP><<<grid, 256, 0, s>>>(a);
    else class_probs_short_kernel<E, most, TOP><<<grid, 256, 0, s>>>(a);
    AVC_LAUNCH_CHECK();
    return AVC_OK;
  }
  if (wave_rows(a.N, a.V)) {
    class_probs_forward_kernel<E, 64, TOP><<<(unsigned)((a.N + 3) / 4), 256, 0, s>>>(a);
    AVC_LAUNCH_CHECK();
    return AVC_OK;
  }
  class_probs_forward_kernel<E, 256, TOP><<<dim3((unsigned)a.N, a.nseg), 256, 0, s>>>(a);
  AVC_LAUNCH_CHECK();
  if (a.nseg > 1) {
    class_probs_join_kernel<E><<<(unsigned)a.N, 256, 0, s>>>(a);
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
    return in_parts<E>(a, 1L << 23, [&](ProbArgs part, long r) {
      part.logp += r, part.entropy += r;
      if (top) part.top_logp += r * top, part.top_ids += r * top;
      return top ? run_forward<E, true>(part, s) : run_forward<E, false>(part, s);
    });
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
    return in_parts<E>(a, (1L << 25) / tiles, [&](const ProbArgs& part, long r) {
      class_probs_backward_kernel<E><<<(unsigned)((part.N * tiles + 3) / 4), 256, 0, s>>>(
          part, dlogp ? dlogp + r : nullptr, dentropy ? dentropy + r : nullptr, static_cast<E*>(dlogits) + r * lddz, lddz,
          (unsigned)tiles);
      AVC_LAUNCH_CHECK();
      return AVC_OK;
    });
  });
}
