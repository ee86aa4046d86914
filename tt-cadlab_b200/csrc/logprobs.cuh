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
PALU_DEVINL float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// A product of e^d and d (d <= 0, in units of log 2) in which e^-inf wins.
constexpr float kFloor = -1000.f;

// Running (maximum, R, T = sum e^(x - m) (x - m) log2(e)) of the elements seen.
struct Stat {
  uint32_t order;  // of the maximum; 0: nothing seen
  uint32_t index;  // its lowest index
  float m, r, t;
  PALU_DEVINL void clear() {
    order = 0;
    index = 0;
    m = -INFINITY;
    r = t = 0.f;
  }
  // move the reference up to m2 (not below m); the old maximum becomes an ordinary element
  PALU_DEVINL void raise(float m2) {
    if (order != 0 && m != -INFINITY) {
      const float d = (m - m2) * kLog2e, a = fast_exp2(d), all = r + 1.f;
      t = a == 0.f ? 0.f : a * (t + all * d);
      r = all * a;
    } else {
      r = t = 0.f;
    }
    m = m2;
  }
  template <int N>
  PALU_DEVINL void add(const float (&x)[N], uint32_t first) {
    float hi = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) hi = max_nan(hi, x[i]);
    const uint32_t o = order_of(hi);
    if (o > order) {  // rare after the first chunks
      raise(hi);
      order = o;
      bool out = false;  // the new maximum itself stays out of R
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!out && order_of(x[i]) == o) {
          out = true;
          index = first + i;
        } else if (x[i] != -INFINITY) {
          const float d = (x[i] - m) * kLog2e, e = fast_exp2(d);
          r += e;
          t += e * fmaxf(d, kFloor);
        }
      }
    } else if (m != -INFINITY) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = (x[i] - m) * kLog2e, e = fast_exp2(d);
        r += e;
        t += e * fmaxf(d, kFloor);
      }
    }
  }
  // join another's elements
  PALU_DEVINL void join(const Stat& b) {
    if (b.order == 0) return;
    const uint64_t ka = order ? key_of(order, index) : 0, kb = key_of(b.order, b.index);
    Stat lo = b;
    if (kb > ka) {
      lo = *this;
      *this = b;
    }
    if (lo.order == 0 || lo.m == -INFINITY) return;
    const float d = (lo.m - m) * kLog2e, a = fast_exp2(d), all = lo.r + 1.f;  // lo's maximum is an ordinary element here
    r += all * a;
    if (a != 0.f) t += a * (lo.t + all * d);
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
    Stat st;
    st.clear();
    if (rank == 0 && tid == 0)
      for (int i = 0; i < sl.head; ++i) {
        const float x[1] = {load1<T>(p, row, i)};
        st.add(x, i);
      }
    int at = 0;
    do {  // an empty slice still takes its stage of the ring
      cp_async_wait<kStages - 2>();
      const unsigned char* buf = ring + stage * kStageBytes + tid * 16;
#pragma unroll
      for (int i = 0; i < kPerStage; ++i) {
        const int c = at + i * kThreads + tid;
        if (c < n) {
          float x[N];
          widen(*reinterpret_cast<const uint4*>(buf + i * kThreads * 16), x);
          st.add(x, sl.head + (sl.c0 + c) * N);
        }
      }
      copy_stage();
      stage = stage + 1 == kStages ? 0 : stage + 1;
      at += kPerStage * kThreads;
    } while (at < n);
    if (rank == 0 && tid == 1)
      for (int i = sl.tail; i < p.vocab; ++i) {
        const float x[1] = {load1<T>(p, row, i)};
        st.add(x, i);
      }

    // ---- the CTA's part ----
    const uint64_t own = st.order ? key_of(st.order, st.index) : 0;
    Stat w = st;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      Stat b;
      b.order = __shfl_xor_sync(0xffffffffu, w.order, o);
      b.index = __shfl_xor_sync(0xffffffffu, w.index, o);
      b.m = __shfl_xor_sync(0xffffffffu, w.m, o);
      b.r = __shfl_xor_sync(0xffffffffu, w.r, o);
      b.t = __shfl_xor_sync(0xffffffffu, w.t, o);
      w.join(b);
    }
    if (lane == 0) s_stat[warp] = w;
    uint64_t list = 0;
    if (p.top > 1) {
      list = sort_desc(own, lane);
      s_keys[warp][lane] = list;
    }
    __syncthreads();
    if (p.top > 1) {
      // every warp: the 32 largest thread maxima, then the elements of the owners warp, warp + 8, ...
      uint64_t best = s_keys[0][lane];
#pragma unroll 1
      for (int x = 1; x < kWarps; ++x) best = merge_desc(best, s_keys[x][lane], lane);
      const uint64_t least = __shfl_sync(0xffffffffu, best, p.top - 1);  // 0: fewer threads than that hold anything
      list = 0;
      for (int x = warp; x < p.top; x += kWarps) {
        const uint64_t who = __shfl_sync(0xffffffffu, best, x);
        if (who == 0) break;
        const int id = (int)index_of(who);
        const bool edge = id < sl.head || id >= sl.tail;
        const int owner = edge ? (id < sl.head ? 0 : 1) : ((id - sl.head) / N - sl.c0) % kThreads;
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
#pragma unroll
          for (int i = 0; i < N; ++i) take(v[i], sl.head + (sl.c0 + mc) * N + i, have);
        }
        if (rank == 0 && owner == 0 && sl.head > 0)
          take(lane < sl.head ? load1<T>(p, row, lane) : 0.f, lane, lane < sl.head);
        if (rank == 0 && owner == 1 && sl.tail < p.vocab) {
          const bool have = sl.tail + lane < p.vocab;
          take(have ? load1<T>(p, row, sl.tail + lane) : 0.f, sl.tail + lane, have);
        }
      }
      __syncthreads();
      s_keys[warp][lane] = list;
      __syncthreads();
    }
    if (warp == 0) {
      Stat a = s_stat[0];
#pragma unroll 1
      for (int x = 1; x < kWarps; ++x) a.join(s_stat[x]);
      if (p.top > 1) {
        list = s_keys[0][lane];
#pragma unroll 1
        for (int x = 1; x < kWarps; ++x) list = merge_desc(list, s_keys[x][lane], lane);
      } else {
        list = lane == 0 && a.order ? key_of(a.order, a.index) : 0;
      }
      if (ranks > 1) {
        if (lane == 0) s_cta = a;
        s_top[lane] = list;
      } else {
        st = a;
      }
    }
    if (ranks > 1) {
      cluster.sync();
      if (rank == 0 && warp == 0) {
        st = s_cta;
        list = s_top[lane];
        for (int x = 1; x < ranks; ++x) {
          st.join(*cluster.map_shared_rank(&s_cta, x));
          if (p.top > 0) list = merge_desc(list, cluster.map_shared_rank(s_top, x)[lane], lane);
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
