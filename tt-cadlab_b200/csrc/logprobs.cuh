// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits, in one pass.
//
// For a row x of `vocab` logits, with M = max x and R = sum over all elements but one that equals M of exp(x - M):
//   log Z = M + log1p(R),   log p_t = (x_t - M) - log1p(R),
//   H = -sum p log p = log1p(R) - (sum exp(x - M) (x - M)) / (1 + R).
// Leaving the maximum out of R keeps the small numbers of a peaked distribution (log p of a sure token is -log1p(R), not
// the log of a sum that was rounded to 1). Everything is held in fp32.
//
// Bound by reading the logits once. A row is read by a cluster of 1 to 8 CTAs (few rows: more CTAs a row, joined over
// distributed shared memory; no workspace, no atomics, one launch), each thread of which owns every 128th 16-byte chunk
// of the CTA's slice: it copies them into its own ring in shared memory (cp.async, so loads run ahead of the arithmetic
// and into the next row) and keeps its own (maximum, R, T) until the slice is done.
//
// Per element that is an exponential (16 a clock and SM: 1051 MB of bf16 keep them busy for 3/4 of the time that reading
// takes) and about six more instructions, so the loop has no branch that data takes often: the maximum is kept out of
// R by a comparator per element, which passes the larger one on and hands the smaller one to the sum (on pairs of bf16
// at once), and the sums refer to a value that moves only when the maximum outgrows it by e^60. (With the exact running
// maximum as reference, every chunk in which one of a warp's 32 maxima grew took a slow path: 4096 x 128256 took 600 us.)
//
// Top k: elements are ordered by value, NaN highest, equal ones by the lower index; as one 64-bit key per element all
// keys differ. With t the k-th largest of the threads' maxima, every element of the top k is at least t and belongs to a
// thread whose maximum is at least t: those look again at the stage that brought their maximum, or, where a second one of
// their stages reaches t, at all of their chunks. (Looking at all chunks of all k threads reads 64 bytes of DRAM for
// each, the rows in flight being more than L2 holds: 4096 x 128256 bf16 with 20 alternatives took 350 us, 180 without.)
// What is found to be at least t is sorted in lists of 32 keys, one a lane, and merged.
#pragma once
#include <cooperative_groups.h>

#include "palu_common.cuh"

namespace palu {
namespace lp {

constexpr int kThreads = 128, kWarps = kThreads / 32;
// Chunks of a thread in a stage, stages of its ring, CTAs an SM. 4096 x 128256 bf16, us: 3 x 3 with 7 CTAs 186, with 8 CTAs
// 216; 4 x 3 with 7 CTAs 210; 2 x 4 with 7 CTAs 203; 256 threads, 2 x 3 with 4 CTAs 220.
constexpr int kPerStage = 3, kStages = 3, kCtas = 7;
constexpr int kStageBytes = kThreads * kPerStage * 16;
constexpr int kMaxTop = 32;
constexpr int kCands = 9 * kThreads;  // candidates for the top that a CTA holds: what one unit a thread can bring at least

struct Params {
  const void* logits;
  int64_t ld;            // elements from row to row
  int64_t rows;
  int vocab, top;
  const void* tokens;    // [rows] int64 or int32
  int tokens64;
  float* logprob;        // [rows]
  float* entropy;        // [rows]
  float* top_logprob;    // [rows][top]
  int64_t* top_id;       // [rows][top]
};

// Order of floats as unsigned numbers: -inf lowest, NaN highest, -0 and +0 equal. Every value's number is above 0.
PALU_DEVINL uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) return 0xFFFFFFFFu;
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
PALU_DEVINL float value_of(uint32_t o) {
  if (o == 0xFFFFFFFFu) return NAN;
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
PALU_DEVINL uint64_t key_of(uint32_t order, uint32_t index) { return (uint64_t)order << 32 | (0xFFFFFFFFu - index); }
PALU_DEVINL uint32_t index_of(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

// 32 keys, one a lane, into descending order.
template <typename K>
PALU_DEVINL K sort_desc(K v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j; j >>= 1) {
      const K o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool high = ((lane & k) == 0) == ((lane & j) == 0);  // this lane keeps the larger one
      v = high ? (v > o ? v : o) : (v > o ? o : v);
    }
  return v;
}
// The 32 largest of two descending lists, descending.
template <typename K>
PALU_DEVINL K merge_desc(K a, K b, int lane) {
  const K r = __shfl_sync(0xffffffffu, b, 31 - lane);
  K v = a > r ? a : r;
#pragma unroll
  for (int j = 16; j; j >>= 1) {
    const K o = __shfl_xor_sync(0xffffffffu, v, j);
    v = (lane & j) == 0 ? (v > o ? v : o) : (v > o ? o : v);
  }
  return v;
}

template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
};
PALU_DEVINL void widen(const uint4& w, float (&x)[8]) {  // 8 bf16
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(v[i] << 16);
    x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
  }
}
PALU_DEVINL void widen(const uint4& w, float (&x)[4]) {  // 4 fp32
  x[0] = __uint_as_float(w.x);
  x[1] = __uint_as_float(w.y);
  x[2] = __uint_as_float(w.z);
  x[3] = __uint_as_float(w.w);
}
// Two bf16 at a time; NaN wins a maximum and loses a minimum.
PALU_DEVINL uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
PALU_DEVINL uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
PALU_DEVINL uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
PALU_DEVINL float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
PALU_DEVINL uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
PALU_DEVINL void un2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v)); }
PALU_DEVINL uint64_t f2add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
PALU_DEVINL uint64_t f2mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
PALU_DEVINL uint64_t f2fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The elements seen: the largest, and R and T = sum e^(x - m) (x - m) log2(e) over the others.
struct Stat {
  float m, r, t;
  PALU_DEVINL void join(const Stat& b) {  // no element: m = -inf, r = t = 0
    const bool up = b.m > m || isnan(b.m);
    const Stat lo = up ? *this : b;
    if (up) *this = b;
    if (lo.m == -INFINITY) return;  // adds nothing
    const float d = (lo.m - m) * kLog2e, a = fast_exp2(d), all = lo.r + 1.f;  // lo's maximum is one of the others here
    r += all * a;
    if (a != 0.f) t += a * (lo.t + all * d);
  }
};

// The lanes' parts as one, the same in every lane.
PALU_DEVINL Stat warp_join(const Stat& s, int lane) {
  const uint32_t o = order_of(s.m), hi = __reduce_max_sync(0xffffffffu, o);
  const int first = __ffs(__ballot_sync(0xffffffffu, o == hi)) - 1;
  Stat w{value_of(hi), s.r, s.t};
  if (lane != first) {  // its maximum is one of the others now
    const float d = (s.m - w.m) * kLog2e, a = s.m == -INFINITY ? 0.f : fast_exp2(d), all = s.r + 1.f;
    w.r = a == 0.f ? 0.f : a * all;
    w.t = a == 0.f ? 0.f : a * (s.t + all * d);
  }
#pragma unroll
  for (int x = 16; x; x >>= 1) {
    w.r += __shfl_xor_sync(0xffffffffu, w.r, x);
    w.t += __shfl_xor_sync(0xffffffffu, w.t, x);
  }
  return w;
}

// A thread's sums of 2^d and 2^d d over its elements, d = x log2(e) - c in one rounding. c belongs to a reference, the
// thread's first maximum; it moves when the maximum outgrows it by kOutgrown, so that the sums stay in range. The same d
// of the row's maximum is subtracted at the end, which takes c's own rounding out again. Elements are held above kLowest
// (-inf: 2^d d is 0, not 0 * inf). Where the reference is so large that c's rounding would move d by more than 1/16, d
// is taken from the difference x - ref instead, chunk by chunk on the slow path.
constexpr float kOutgrown = 60.f, kLowest = -1e30f, kLargeRef = 524288.f, kFloor = -1000.f;
struct Sums {
  float ref, c;
  uint64_t r, t;  // two partial sums each
  PALU_DEVINL void clear() {
    ref = -INFINITY;
    c = 0.f;
    r = t = 0;
  }
  PALU_DEVINL bool large() const { return !(fabsf(ref) < kLargeRef) && ref != -INFINITY; }
  PALU_DEVINL float scaled(float x) const { return large() ? fmaxf((x - ref) * kLog2e, kFloor) : fmaf(x, kLog2e, -c); }
  PALU_DEVINL void raise(float to) {
    const float d = scaled(to), a = ref == -INFINITY ? 0.f : fast_exp2(-d);
    float r0, r1, t0, t1;
    un2(r, r0, r1);
    un2(t, t0, t1);
    ref = to;
    c = to * kLog2e;
    const float back = scaled(to);  // of the new reference against itself: c's rounding
    t = a == 0.f ? 0 : f2(a * (t0 - r0 * d), a * (t1 - r1 * d));
    r = a == 0.f ? 0 : f2(r0 * a, r1 * a);
    // against `to` exactly; now against c
    const float k = fast_exp2(back);
    un2(r, r0, r1);
    un2(t, t0, t1);
    t = f2(k * (t0 + r0 * back), k * (t1 + r1 * back));
    r = f2(r0 * k, r1 * k);
  }
  PALU_DEVINL void add(float x0, float x1) {
    float d0, d1;
    un2(f2fma(f2(x0, x1), f2(kLog2e, kLog2e), f2(-c, -c)), d0, d1);
    const uint64_t e = f2(fast_exp2(d0), fast_exp2(d1));
    r = f2add(r, e);
    t = f2fma(e, f2(d0, d1), t);
  }
  PALU_DEVINL void add_slow(float x0, float x1) {
    const float d0 = fmaxf((x0 - ref) * kLog2e, kFloor), d1 = fmaxf((x1 - ref) * kLog2e, kFloor);
    const uint64_t e = f2(fast_exp2(d0), fast_exp2(d1));
    r = f2add(r, e);
    t = f2fma(e, f2(d0, d1), t);
  }
  // the sums of everything but the maximum m, against m
  PALU_DEVINL Stat stat(float m) const {
    float r0, r1, t0, t1;
    un2(r, r0, r1);
    un2(t, t0, t1);
    Stat s{m, 0.f, 0.f};
    if (m == -INFINITY) return s;
    const float d = scaled(m), a = fast_exp2(-d);
    s.r = (r0 + r1) * a;
    s.t = ((t0 + t1) - d * (r0 + r1)) * a;
    return s;
  }
};

// A thread's elements: their maximum, which stays out of the sums (each comparison passes the larger value on and gives
// the smaller one to the sums).
template <typename T>
struct Run;
template <>
struct Run<float> {
  Sums s;
  float m, limit;  // an element above the limit takes the slow path; -inf: every one does
  PALU_DEVINL void clear() {
    s.clear();
    m = limit = -INFINITY;
  }
  // M chunks; returns their maximum
  template <int M>
  PALU_DEVINL float add(const uint4 (&w)[M]) {
    float c = 0.f, lo[M][4];
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const float x0 = __uint_as_float(w[i].x), x1 = __uint_as_float(w[i].y), x2 = __uint_as_float(w[i].z), x3 = __uint_as_float(w[i].w);
      const float a = max_nan(x0, x1), b = max_nan(x2, x3), ab = max_nan(a, b), before = i ? c : m;
      lo[i][0] = fminf(x0, x1);
      lo[i][1] = fminf(x2, x3);
      lo[i][2] = fminf(a, b);
      if (i) lo[i][3] = fminf(before, ab);
      c = i ? max_nan(c, ab) : ab;
    }
    lo[0][3] = fminf(m, c);
    m = max_nan(m, c);
    if (m > limit || limit == -INFINITY) {
      if (m > s.ref + kOutgrown) s.raise(m);
      limit = s.large() ? -INFINITY : s.ref + kOutgrown;
      if (s.large()) {
#pragma unroll
        for (int i = 0; i < M; ++i) {
          s.add_slow(lo[i][0], lo[i][1]);
          s.add_slow(lo[i][2], lo[i][3]);
        }
        return c;
      }
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
      s.add(fmaxf(lo[i][0], kLowest), fmaxf(lo[i][1], kLowest));
      s.add(fmaxf(lo[i][2], kLowest), fmaxf(lo[i][3], kLowest));
    }
    return c;
  }
  PALU_DEVINL float max() const { return m; }
  PALU_DEVINL Stat stat() const { return s.stat(m); }
};
template <>
struct Run<__nv_bfloat16> {
  Sums s;
  uint32_t m, limit;  // the maxima of the even and of the odd elements; the limit for both
  PALU_DEVINL void clear() {
    s.clear();
    m = limit = kNone;
  }
  static PALU_DEVINL float low(uint32_t w) { return __uint_as_float(w << 16); }
  static PALU_DEVINL float high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
  template <int M>
  PALU_DEVINL float add(const uint4 (&w)[M]) {
    uint32_t c = 0, lo[M][4];
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const uint32_t a = max2_nan(w[i].x, w[i].y), b = max2_nan(w[i].z, w[i].w), ab = max2_nan(a, b);
      lo[i][0] = min2(w[i].x, w[i].y);
      lo[i][1] = min2(w[i].z, w[i].w);
      lo[i][2] = min2(a, b);
      if (i) lo[i][3] = min2(c, ab);
      c = i ? max2_nan(c, ab) : ab;
    }
    lo[0][3] = min2(m, c);
    m = max2_nan(m, c);
    const float top = max_nan(low(c), high(c));
    if (max2(m, limit) != limit || limit == kNone) {
      const float hi = max();
      if (hi > s.ref + kOutgrown) s.raise(hi);
      // rounded down (a step of bf16 is up to 2048 here, and the sums have no room for an element that far above the
      // reference); never below the reference, which is a bf16 value itself, so equal elements stay off this path
      const uint32_t f = __float_as_uint(s.ref + kOutgrown);
      const uint32_t l = s.large() ? kNone & 0xFFFFu : (f >> 16) + ((f >> 31) & ((f & 0xFFFFu) != 0));
      limit = l << 16 | l;
      if (s.large()) {
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
          for (int y = 0; y < 4; ++y) s.add_slow(low(lo[i][y]), high(lo[i][y]));
        return top;
      }
    }
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t l = max2(lo[i][y], kLowest2);
        s.add(low(l), high(l));
      }
    return top;
  }
  PALU_DEVINL float max() const { return max_nan(low(m), high(m)); }
  PALU_DEVINL Stat stat() const {
    const float a = low(m), b = high(m);
    Stat x = s.stat(max());
    x.join(Stat{a < b ? a : b, 0.f, 0.f});  // the other lane's maximum is an ordinary element
    return x;
  }
  static constexpr uint32_t kNone = 0xFF80FF80u;      // -inf, twice
  static constexpr uint32_t kLowest2 = 0xF14AF14Au;  // -1e30 rounded to bf16, twice
};

// Where a thread's largest element is: the stage that brought it, and the largest element of the other stages. Of no use to a
// thread that saw a NaN (a later stage takes its place).
struct Where {
  float best, rest;
  int stage;
  PALU_DEVINL void clear() {
    best = rest = -INFINITY;
    stage = 0;
  }
  PALU_DEVINL void add(float top, int at) {
    rest = fmaxf(rest, fminf(top, best));
    if (!(top <= best)) {
      best = top;
      stage = at;
    }
  }
};

// The part of a row that a CTA reads: 16-byte chunks [c0, c1) of the aligned body, whose chunk 0 starts at element
// `head`; the elements before and behind the body (a row that does not start or end on 16 bytes) go to the first CTA.
struct Slice {
  const char* body;
  int head, c0, c1, tail;  // tail: first element behind the body
};
template <typename T>
PALU_DEVINL Slice slice_of(const Params& p, int64_t row, int rank, int ranks) {
  constexpr int N = Chunk<T>::N;
  const T* x = static_cast<const T*>(p.logits) + row * p.ld;
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  Slice s;
  s.head = min(p.vocab, off ? N - off : 0);
  const int chunks = (p.vocab - s.head) / N;
  s.body = reinterpret_cast<const char*>(x + s.head);
  s.tail = s.head + chunks * N;
  s.c0 = (int)((int64_t)chunks * rank / ranks);
  s.c1 = (int)((int64_t)chunks * (rank + 1) / ranks);
  return s;
}

template <typename T>
PALU_DEVINL float load1(const Params& p, int64_t row, int i) {
  const T v = static_cast<const T*>(p.logits)[row * p.ld + i];
  if constexpr (sizeof(T) == 4) return v;
  else return __bfloat162float(v);
}

// The element outside the body that goes to a CTA's thread (counted from the last), or -1.
PALU_DEVINL int edge_element(const Slice& s, int rank, int i, int vocab) {
  if (rank != 0) return -1;
  if (i < s.head) return i;
  const int t = s.tail + i - s.head;
  return t < vocab ? t : -1;
}
// The warps' descending lists (each also in its `mine`) into one, in warp 0.
template <typename K>
PALU_DEVINL K merge_lists(K (*s_keys)[32], K mine, int warp, int lane) {
#pragma unroll
  for (int h = kWarps / 2; h; h >>= 1) {
    if (warp < h) {
      mine = merge_desc(mine, s_keys[warp + h][lane], lane);
      if (h > 1) s_keys[warp][lane] = mine;
    }
    __syncthreads();
  }
  return mine;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kCtas) palu_token_logprobs_kernel(const Params p) {
  constexpr int N = Chunk<T>::N;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  const int64_t first = blockIdx.x / ranks, step = gridDim.x / ranks;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ uint64_t s_keys[kWarps][32];
  __shared__ Stat s_stat[kWarps];
  __shared__ Stat s_cta[2];         // this CTA's part of a row, read by the cluster's first CTA
  __shared__ uint64_t s_top[2][32];  // and its best
  __shared__ uint32_t s_max[kWarps][32], s_least;
  __shared__ uint64_t s_cand[kCands];
  __shared__ int s_who[kThreads], s_owners, s_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t mine = smem_u32(ring) + tid * 16;

  // The copies run kStages - 1 stages ahead of the arithmetic, over the CTA's rows one after another; a row takes a stage
  // or more.
  constexpr int kChunks = kPerStage * kThreads;
  int64_t row_l = first;
  int left_l = 0;  // chunks of row_l's slice that are not copied yet
  const char* src_l = nullptr;
  auto next_slice = [&]() {
    if (row_l >= p.rows) return;  // left_l stays at 0 or below: nothing is copied
    const Slice s = slice_of<T>(p, row_l, rank, ranks);
    left_l = s.c1 - s.c0;
    src_l = s.body + ((int64_t)s.c0 + tid) * 16;
  };
  next_slice();
  auto copy_stage = [&](int slot) {
    const uint32_t dst = mine + slot * kStageBytes;
    if (left_l >= kChunks) {
#pragma unroll
      for (int i = 0; i < kPerStage; ++i) cp_async16(dst + i * kThreads * 16, src_l + i * kThreads * 16, 16);
    } else {
#pragma unroll
      for (int i = 0; i < kPerStage; ++i)
        if (i * kThreads + tid < left_l) cp_async16(dst + i * kThreads * 16, src_l + i * kThreads * 16, 16);
    }
    cp_async_commit();
    src_l += kChunks * 16;
    left_l -= kChunks;
    if (left_l <= 0) {
      left_l = 0;
      row_l += step;
      next_slice();
    }
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) copy_stage(s);
  int slot = 0, par = 0;

  for (int64_t row = first; row < p.rows; row += step) {
    const Slice sl = slice_of<T>(p, row, rank, ranks);
    const int n = sl.c1 - sl.c0;
    Run<T> run;
    run.clear();
    Where where;
    where.clear();
    int left = n, at = 0;
    do {
      cp_async_wait<kStages - 2>();
      const unsigned char* buf = ring + slot * kStageBytes + tid * 16;
      if (left >= kChunks) {
        uint4 w[kPerStage];
#pragma unroll
        for (int i = 0; i < kPerStage; ++i) w[i] = *reinterpret_cast<const uint4*>(buf + i * kThreads * 16);
        const float top = run.add(w);
        if (p.top > 0) where.add(top, at);
      } else {
#pragma unroll 1
        for (int i = 0; i < kPerStage; ++i)
          if (i * kThreads + tid < left) {
            const uint4 w[1] = {*reinterpret_cast<const uint4*>(buf + i * kThreads * 16)};
            const float top = run.add(w);
            if (p.top > 0) where.add(top, at);
          }
      }
      left -= kChunks;
      ++at;
      copy_stage(slot == 0 ? kStages - 1 : slot - 1);
      slot = slot == kStages - 1 ? 0 : slot + 1;
    } while (left > 0);
    // the elements before and behind the body: one each to the last threads of the first CTA
    const int edge = edge_element(sl, rank, kThreads - 1 - tid, p.vocab);
    Stat st = run.stat();
    if (edge >= 0) st.join(Stat{load1<T>(p, row, edge), 0.f, 0.f});

    // ---- the CTA's part ----
    const Stat w = warp_join(st, lane);
    if (lane == 0) s_stat[warp] = w;
    uint32_t own = 0;  // the thread's largest element
    if (p.top > 0) {
      if (n > tid) own = order_of(run.max());
      if (edge >= 0) own = max(own, order_of(load1<T>(p, row, edge)));
      if (p.top > 1) s_max[warp][lane] = sort_desc(own, lane);
    }
    if (tid == 0) s_count = s_owners = 0;
    __syncthreads();
    uint64_t list = 0;
    if (p.top > 0) {
      uint32_t least;  // the top-th largest of the threads' maxima; 0: fewer threads than that hold anything
      if (p.top == 1) {
        least = order_of(s_stat[0].m);
#pragma unroll
        for (int x = 1; x < kWarps; ++x) least = max(least, order_of(s_stat[x].m));
      } else {
        const uint32_t best = merge_lists(s_max, s_max[warp][lane], warp, lane);
        if (warp == 0 && lane == p.top - 1) s_least = best;
        __syncthreads();
        least = s_least;
      }
      // The elements of at least `least` go to the candidates. A thread whose maximum is that large looks through the stage
      // that brought it; where its other stages may hold such elements too, all threads look through its chunks. If the
      // candidates are more than fit (many equal elements), that is done over in rounds that fit, with a merge behind each.
      const int per = (n + kThreads - 1) / kThreads;  // chunks of a thread, at most
      const float floor_value = value_of(least);
      uint64_t last = 0;  // the list's top-th key: smaller ones are of no use
      auto push = [&](float v, int i) {
        const uint32_t o = order_of(v);
        const uint64_t k = key_of(o, (uint32_t)i);
        if (o >= least && k > last) {
          const int at = atomicAdd(&s_count, 1);
          if (at < kCands) s_cand[at] = k;
        }
      };
      auto look = [&](int owner, int j) {  // unit j of an owner's
        const int c = owner + j * kThreads;
        if (c < n) {
          float v[N];
          widen(*reinterpret_cast<const uint4*>(sl.body + (int64_t)(sl.c0 + c) * 16), v);
          float hi = v[0];
#pragma unroll
          for (int i = 1; i < N; ++i) hi = max_nan(hi, v[i]);
          if (!(hi < floor_value)) {  // also where one of them is NaN
#pragma unroll
            for (int i = 0; i < N; ++i)
              if (!(v[i] < floor_value)) push(v[i], sl.head + (sl.c0 + c) * N + i);
          }
        }
      };
      auto merge = [&](int have) {
        for (int x = warp * 32; x < have; x += kThreads) {
          const uint64_t k = x + lane < have ? s_cand[x + lane] : 0;
          list = merge_desc(list, sort_desc(k, lane), lane);
        }
        s_keys[warp][lane] = list;
        __syncthreads();
        list = merge_lists(s_keys, list, warp, lane);
      };
      if (own != 0 && own >= least) {
        if (n > tid) {  // it has a chunk
          if (order_of(where.rest) >= least || own == 0xFFFFFFFFu) {  // or a NaN among them
            s_who[atomicAdd(&s_owners, 1)] = tid;
          } else {
#pragma unroll
            for (int i = 0; i < kPerStage; ++i) look(tid, where.stage * kPerStage + i);
          }
        }
        if (edge >= 0) push(load1<T>(p, row, edge), edge);
      }
      __syncthreads();
      const int count = s_owners;
      if (count > 0) {
        for (int who = tid / per, j = tid % per; who < count;) {
          look(s_who[who], j);
          for (j += kThreads; j >= per; j -= per) ++who;
        }
        __syncthreads();
      }
      if (s_count <= kCands) {
        merge(s_count);
      } else {
        // every thread's chunks; then the edge elements, one more unit each
        const int64_t units = (int64_t)kThreads * (per + 1);
        for (int64_t u0 = 0; u0 < units; u0 += kThreads) {
          __syncthreads();
          if (tid == 0) s_count = 0;
          __syncthreads();
          const int j = (int)(u0 / kThreads);
          if (j < per) look(tid, j);
          else if (edge >= 0) push(load1<T>(p, row, edge), edge);
          __syncthreads();
          merge(s_count);
          if (warp == 0) s_top[par][lane] = list;
          __syncthreads();
          last = s_top[par][p.top - 1];
          if (warp != 0) list = 0;
        }
      }
    }
    if (warp == 0) {
      st = lane < kWarps ? s_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
      st = warp_join(st, lane);
      if (ranks > 1) {
        if (lane == 0) s_cta[par] = st;
        s_top[par][lane] = list;
      }
    }
    if (ranks > 1) {
      cluster.sync();
      if (rank == 0) {
        if (p.top > 0) {  // warp x takes the lists of the CTAs x, x + kWarps, ...
          list = 0;
          for (int x = warp; x < ranks; x += kWarps) list = merge_desc(list, cluster.map_shared_rank(s_top[par], x)[lane], lane);
          s_keys[warp][lane] = list;
          __syncthreads();
          list = merge_lists(s_keys, list, warp, lane);
        }
        if (warp == 0) {
          st = lane < ranks ? *cluster.map_shared_rank(&s_cta[par], lane) : Stat{-INFINITY, 0.f, 0.f};
          st = warp_join(st, lane);
        }
      }
    }
    if (rank == 0 && warp == 0) {
      const bool sound = st.m > -INFINITY && st.m < INFINITY;  // false too for NaN
      const float lz = log1pf(st.r);
      if (lane == 0) {
        const int64_t tok = p.tokens64 ? static_cast<const int64_t*>(p.tokens)[row] : static_cast<const int32_t*>(p.tokens)[row];
        float v = 0.f;  // no token
        if (tok >= p.vocab) v = NAN;
        else if (tok >= 0) v = sound ? (load1<T>(p, row, (int)tok) - st.m) - lz : NAN;
        p.logprob[row] = v;
        p.entropy[row] = sound ? lz - 0.6931471805599453f * st.t / (1.f + st.r) : NAN;
      }
      if (lane < p.top) {
        p.top_logprob[row * p.top + lane] = sound ? (value_of((uint32_t)(list >> 32)) - st.m) - lz : NAN;
        p.top_id[row * p.top + lane] = index_of(list);
      }
    }
    par ^= 1;  // the next row's parts go to the other place; the one after that comes behind the next cluster.sync
    __syncthreads();
  }
  if (ranks > 1) cluster.sync();  // the first CTA has read the others' parts
}

}  // namespace lp
}  // namespace palu
