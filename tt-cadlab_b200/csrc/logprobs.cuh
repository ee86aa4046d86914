// Log probabilities of given tokens, the entropy and the top alternatives of rows of logits, in one pass.
//
// For a row x of `vocab` logits, with M = max x and R = sum over all elements but one that equals M of exp(x - M):
//   log Z = M + log1p(R),   log p_t = (x_t - M) - log1p(R),
//   H = -sum p log p = log1p(R) - (sum exp(x - M) (x - M)) / (1 + R).
// Leaving the maximum out of R keeps the small numbers of a peaked distribution (log p of a sure token is -log1p(R), not
// the log of a sum that was rounded to 1). Everything is held in fp32.
//
// Bound by reading the logits once. A row is read by a cluster of 1 to 8 CTAs (few rows: more CTAs a row, joined over
// distributed shared memory; no workspace, no atomics, one launch), each thread of which owns every 256th 16-byte chunk
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
// keys differ. With t the k-th largest of the threads' maxima, every element of the top k is at least t and belongs to
// one of the k threads whose maximum is at least t: only the elements of those are looked at again (about k / 256 of the
// slice, from L2), one warp a thread, and kept in sorted lists of 32 keys, one a lane, that are merged.
#pragma once
#include <cooperative_groups.h>

#include "palu_common.cuh"

namespace palu {
namespace lp {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPerStage = 4, kStages = 4;  // chunks of a thread in a stage, stages of its ring
constexpr int kStageBytes = kThreads * kPerStage * 16;
constexpr int kMaxTop = 32;

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
PALU_DEVINL uint64_t sort_desc(uint64_t v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j; j >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, v, j);
      const bool high = ((lane & k) == 0) == ((lane & j) == 0);  // this lane keeps the larger one
      v = (v > o) == high ? v : o;
    }
  return v;
}
// The 32 largest of two descending lists, descending.
PALU_DEVINL uint64_t merge_desc(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
  uint64_t v = a > r ? a : r;
#pragma unroll
  for (int j = 16; j; j >>= 1) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, v, j);
    v = (v > o) == ((lane & j) == 0) ? v : o;
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

// d = (x - ref) log2(e) is kept above this, so that an element of -inf adds e^d d = 0 and not 0 * inf.
constexpr float kFloor = -1000.f;
constexpr float kOutgrown = 60.f;  // sums of e^60 stay in range

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

// A thread's running sums over its elements, against a reference that is one of its early elements.
template <typename T>
struct Run;

struct Sums {
  float ref;
  uint64_t r, t;  // two partial sums each
  PALU_DEVINL void clear() {
    ref = -INFINITY;
    r = t = 0;
  }
  PALU_DEVINL void raise(float to) {
    const float d = (ref - to) * kLog2e, a = fast_exp2(d);  // ref -inf: a = 0
    float r0, r1, t0, t1;
    un2(r, r0, r1);
    un2(t, t0, t1);
    t = a == 0.f ? 0 : f2(a * (t0 + r0 * d), a * (t1 + r1 * d));
    r = a == 0.f ? 0 : f2(r0 * a, r1 * a);
    ref = to;
  }
  PALU_DEVINL void add(float x0, float x1) {
    float d0, d1;
    un2(f2mul(f2add(f2(x0, x1), f2(-ref, -ref)), f2(kLog2e, kLog2e)), d0, d1);
    d0 = fmaxf(d0, kFloor);  // also for NaN, whose row is NaN by its maximum
    d1 = fmaxf(d1, kFloor);
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
    const float d = (m - ref) * kLog2e, a = fast_exp2(-d);
    s.r = (r0 + r1) * a;
    s.t = ((t0 + t1) - d * (r0 + r1)) * a;
    return s;
  }
};

template <>
struct Run<float> {
  Sums s;
  float m;
  int at;  // the chunk that brought m
  PALU_DEVINL void clear() {
    s.clear();
    m = -INFINITY;
    at = -1;
  }
  PALU_DEVINL void add(const uint4& w, int chunk) {
    const float x0 = __uint_as_float(w.x), x1 = __uint_as_float(w.y), x2 = __uint_as_float(w.z), x3 = __uint_as_float(w.w);
    const float a = max_nan(x0, x1), b = max_nan(x2, x3), c = max_nan(a, b);
    const float before = m;
    m = max_nan(m, c);
    if (c > s.ref + kOutgrown) s.raise(c);
    if (__float_as_uint(m) != __float_as_uint(before) || at < 0) at = chunk;
    s.add(fminf(x0, x1), fminf(x2, x3));
    s.add(fminf(a, b), fminf(before, c));
  }
  PALU_DEVINL float max() const { return m; }
  PALU_DEVINL int chunk(float) const { return at; }
  PALU_DEVINL Stat stat() const { return s.stat(m); }
};
template <>
struct Run<__nv_bfloat16> {
  Sums s;
  uint32_t m;      // the maxima of the even and of the odd elements
  int at0, at1;    // the chunks that brought them
  PALU_DEVINL void clear() {
    s.clear();
    m = 0xFF80FF80u;
    at0 = at1 = -1;
  }
  static PALU_DEVINL float low(uint32_t w) { return __uint_as_float(w << 16); }
  static PALU_DEVINL float high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
  PALU_DEVINL void add(const uint4& w, int chunk) {
    const uint32_t a = max2_nan(w.x, w.y), b = max2_nan(w.z, w.w), c = max2_nan(a, b), before = m;
    m = max2_nan(m, c);
    const float top = max_nan(low(c), high(c));
    if (top > s.ref + kOutgrown) s.raise(top);
    if (m != before || at0 < 0) {
      if ((m ^ before) & 0xFFFFu || at0 < 0) at0 = chunk;
      if ((m ^ before) >> 16 || at1 < 0) at1 = chunk;
    }
    const uint32_t lo[4] = {min2(w.x, w.y), min2(w.z, w.w), min2(a, b), min2(before, c)};
#pragma unroll
    for (int i = 0; i < 4; ++i) s.add(low(lo[i]), high(lo[i]));
  }
  PALU_DEVINL float max() const { return max_nan(low(m), high(m)); }
  // the chunk of the first element that equals the maximum v
  PALU_DEVINL int chunk(float v) const {
    const bool e0 = order_of(low(m)) == order_of(v), e1 = order_of(high(m)) == order_of(v);
    return e0 && e1 ? min(at0, at1) : (e0 ? at0 : at1);
  }
  PALU_DEVINL Stat stat() const {
    const float a = low(m), b = high(m), hi = max(), lo = fminf(a, b);
    Sums all = s;
    all.add(lo, -INFINITY);
    return all.stat(hi);
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
// The 8 warps' descending lists (each also in its `mine`) into one, in warp 0.
PALU_DEVINL uint64_t merge_lists(uint64_t (*s_keys)[32], uint64_t mine, int warp, int lane) {
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
__global__ void __launch_bounds__(kThreads, 3) palu_token_logprobs_kernel(const Params p) {
  constexpr int N = Chunk<T>::N;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  const int64_t first = blockIdx.x / ranks, step = gridDim.x / ranks;
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ uint64_t s_keys[kWarps][32];
  __shared__ Stat s_stat[kWarps];
  __shared__ Stat s_cta;           // this CTA's part of the row, read by the cluster's first CTA
  __shared__ uint64_t s_top[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t mine = smem_u32(ring) + tid * 16;

  // the copies run kStages - 1 stages ahead of the arithmetic, over the CTA's rows one after another
  int64_t row_l = first;
  int at_l = 0;  // next chunk of row_l's slice to copy, relative to c0
  Slice sl_l;
  if (row_l < p.rows) sl_l = slice_of<T>(p, row_l, rank, ranks);
  int stage_l = 0;
  auto copy_stage = [&]() {
    if (row_l < p.rows) {
      const int n = sl_l.c1 - sl_l.c0;
#pragma unroll
      for (int i = 0; i < kPerStage; ++i) {
        const int c = at_l + i * kThreads + tid;
        if (c < n) cp_async16(mine + stage_l * kStageBytes + i * kThreads * 16, sl_l.body + (int64_t)(sl_l.c0 + c) * 16, 16);
      }
      at_l += kPerStage * kThreads;
      if (at_l >= n) {
        at_l = 0;
        row_l += step;
        if (row_l < p.rows) sl_l = slice_of<T>(p, row_l, rank, ranks);
      }
    }
    cp_async_commit();
    stage_l = stage_l + 1 == kStages ? 0 : stage_l + 1;
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) copy_stage();

  int stage = 0;
  for (int64_t row = first; row < p.rows; row += step) {
    const Slice sl = slice_of<T>(p, row, rank, ranks);
    const int n = sl.c1 - sl.c0;
    Run<T> run;
    run.clear();
    int at = 0;
    do {  // an empty slice still takes its stage of the ring
      cp_async_wait<kStages - 2>();
      const unsigned char* buf = ring + stage * kStageBytes + tid * 16;
#pragma unroll
      for (int i = 0; i < kPerStage; ++i) {
        const int c = at + i * kThreads + tid;
        if (c < n) run.add(*reinterpret_cast<const uint4*>(buf + i * kThreads * 16), c);
      }
      copy_stage();
      stage = stage + 1 == kStages ? 0 : stage + 1;
      at += kPerStage * kThreads;
    } while (at < n);
    // the elements before and behind the body: one each to the last threads of the first CTA
    const int edge = edge_element(sl, rank, kThreads - 1 - tid, p.vocab);
    Stat st = run.stat();
    if (edge >= 0) st.join(Stat{load1<T>(p, row, edge), 0.f, 0.f});

    // ---- the CTA's part ----
    // the thread's largest element as a key
    uint64_t own = 0;
    if (p.top > 0) {
      const float v = run.max();
      if (n > tid) {
        uint32_t o = order_of(v);
        int c = run.chunk(v), c1 = c;
        if (o == 0x80000000u) {  // zeros: -0 gave way to a later +0, but the first of them counts
          c = tid;
          c1 = n - 1;
        }
        for (; c <= c1 && own == 0; c += kThreads) {
          float x[N];
          widen(*reinterpret_cast<const uint4*>(sl.body + (int64_t)(sl.c0 + c) * 16), x);
#pragma unroll
          for (int i = N - 1; i >= 0; --i)
            if (order_of(x[i]) == o) own = key_of(o, (uint32_t)(sl.head + (sl.c0 + c) * N + i));
        }
      }
      if (edge >= 0) {
        const uint64_t k = key_of(order_of(load1<T>(p, row, edge)), (uint32_t)edge);
        own = k > own ? k : own;
      }
    }
    Stat w = st;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      Stat b;
      b.m = __shfl_xor_sync(0xffffffffu, w.m, o);
      b.r = __shfl_xor_sync(0xffffffffu, w.r, o);
      b.t = __shfl_xor_sync(0xffffffffu, w.t, o);
      w.join(b);
    }
    if (lane == 0) s_stat[warp] = w;
    uint64_t list = 0;
    if (p.top > 0) {
      list = sort_desc(own, lane);
      s_keys[warp][lane] = list;
    }
    __syncthreads();
    if (p.top > 0) list = merge_lists(s_keys, list, warp, lane);  // warp 0: the 32 largest thread maxima
    if (p.top > 1) {
      if (warp == 0) s_top[lane] = list;
      __syncthreads();
      // every warp: the elements of the owners warp, warp + 8, ...
      const uint64_t best = s_top[lane];
      const uint64_t least = __shfl_sync(0xffffffffu, best, p.top - 1);  // 0: fewer threads than that hold anything
      list = 0;
      for (int x = warp; x < p.top; x += kWarps) {
        const uint64_t who = __shfl_sync(0xffffffffu, best, x);
        if (who == 0) break;
        const int id = (int)index_of(who);
        int owner;
        if (id < sl.head) owner = kThreads - 1 - id;
        else if (id >= sl.tail) owner = kThreads - 1 - (sl.head + id - sl.tail);
        else owner = ((id - sl.head) / N - sl.c0) % kThreads;
        auto take = [&](float v, int i, bool have) {
          uint64_t k = have ? key_of(order_of(v), (uint32_t)i) : 0;
          if (k < least) k = 0;
          if (__any_sync(0xffffffffu, k != 0)) list = merge_desc(list, sort_desc(k, lane), lane);
        };
        for (int c = owner; c < n; c += 32 * kThreads) {
          const int mc = c + lane * kThreads;
          const bool have = mc < n;
          float v[N];
          uint4 raw = make_uint4(0, 0, 0, 0);
          if (have) raw = *reinterpret_cast<const uint4*>(sl.body + (int64_t)(sl.c0 + mc) * 16);
          widen(raw, v);
#pragma unroll 1
          for (int i = 0; i < N; ++i) {
            float vi = v[0];
#pragma unroll
            for (int y = 1; y < N; ++y) vi = y == i ? v[y] : vi;
            take(vi, sl.head + (sl.c0 + mc) * N + i, have);
          }
        }
        const int e = edge_element(sl, rank, kThreads - 1 - owner, p.vocab);
        if (e >= 0) take(load1<T>(p, row, e), e, lane == 0);
      }
      s_keys[warp][lane] = list;
      __syncthreads();
      list = merge_lists(s_keys, list, warp, lane);
    }
    if (warp == 0) {
      Stat a = s_stat[0];
#pragma unroll 1
      for (int x = 1; x < kWarps; ++x) a.join(s_stat[x]);
      if (ranks > 1) {
        if (lane == 0) s_cta = a;
        s_top[lane] = list;
      } else {
        st = a;
      }
    }
    if (ranks > 1) {
      cluster.sync();
      if (rank == 0) {
        if (p.top > 0) {  // warp x takes CTA x's list
          list = warp < ranks ? cluster.map_shared_rank(s_top, warp)[lane] : 0;
          s_keys[warp][lane] = list;
          __syncthreads();
          list = merge_lists(s_keys, list, warp, lane);
        }
        if (warp == 0) {
          st = s_cta;
          for (int x = 1; x < ranks; ++x) st.join(*cluster.map_shared_rank(&s_cta, x));
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
    if (ranks > 1) cluster.sync();  // the others' parts have been read
    else __syncthreads();
  }
}

}  // namespace lp
}  // namespace palu
