// Causal attention of packed prompts on the 5th-generation tensor cores (tcgen05 + TMEM + TMA).
//
// Sequence s has q_len query positions and k_len keys, its last query aligned with its last key: the query at
// offset i sees the keys 0 .. i + k_len - q_len. With x_ij = scale q_i . k_j,
//   o_i = sum_j exp(x_ij - m_i) v_j / l_i,   l_i = sum_j exp(x_ij - m_i),
// in one pass over the keys with a running reference m_i and sum l_i (fp32); the exponentials are rounded to bf16
// (half a step, 2^-8 relative) as the A operand of the second product, the two products accumulate in fp32.
//
// A work item is (sequence, query tile, KV head): two chains of 128 rows, where a chain's row is one (position, query
// head of the KV head's group) pair, positions outermost, so that the heads that share K and V share their tiles and
// a chain of rep heads per KV head covers 128 / rep positions (little masked work on the diagonal, and a prompt of
// one token still fills rep rows). Items, or pieces of items along the keys, are laid out per CTA by the host's plan;
// CTAs are persistent. A piece that is not a whole item writes a partial record (O, m, l) that the merge joins.
// Per key tile t of 128 keys and chain c:
//   MMA      S_c[128 x 128] (f32, TMEM) = Q_c (smem) x K_t^T (smem), 8 steps of K = 16
//   softmax  one thread per row: exp2 against the reference, P_c (bf16) -> TMEM. The reference is the maximum of the row's
//            first 32 keys and moves (rescaling O_c and l) only when the tile's sum shows that a score may have outgrown
//            it by 2^9 or more: any reference within that keeps P and l in range, and the final division cancels it. So
//            no exponential waits for a maximum.
//   MMA      O_c[128 x d_v] (f32, TMEM) += P_c (TMEM) x V_t (smem, MN-major: as TMA wrote it)
// The chains run half a period apart: while the tensor cores work on one chain's PV and next S, the other chain's softmax
// warps exponentiate. Values at most 64 wide leave TMEM columns for P of its own, and the next S does not wait for PV; wider
// ones write P over S.
//
// What bounds it: at d_v 128 a tile and chain takes the tensor cores 1290 cycles (16 MMAs; S alone 700, its operands' 64 KB
// being what shared memory delivers in 512) and the softmax warps 1870 (128 exponentials of the special-function unit a row
// are 1024), one behind the other: 3230 a tile for both chains, against 2580 if the tensor cores never waited. Measured, 32
// query and 8 KV heads: 32768 tokens, d_v 128 7.7 ms (1140 TFLOP/s, under the power cap); 8192 tokens 470 us (1170); d_v 64
// 429 us (960). A piece takes about 7000 cycles besides its tiles (its first loads and reference, the last PV, the epilogue):
// 32 prompts of 512 tokens at d_v 128 135 us, 8 prompts of 64 to 2048 tokens at d_v 64 111.
// Tried and not kept: a polynomial for every second to eighth exponential (no faster at any share: the chain's latency is
// what counts); leaving out the keys of a diagonal tile that a chain does not see (PV alone, by predicates: those 8 prompts
// 117 -> 123 us; the exponentials too, as a second body for at most 64 keys: 120); S in two halves of 64 keys so that the
// upper one need not wait for PV (32768 tokens 9.2 ms: an MMA takes its 64 cycles at N = 64 too).
//
// Masked places hold anything. Scores behind a row's last visible key are replaced, never added to. V rows behind the
// item's last visible key are zeroed in shared memory before the product, and non-finite values in the V rows that
// only some rows of the item see are zeroed too and added back, in the epilogue, to exactly the rows that see them
// (0 * NaN in the tensor core would reach the others). A tile's V is checked only where the mask cuts it.
//
// Warps: 0..3 softmax of chain 0, 4..7 of chain 1, 8 TMA producer, 9 MMA issuer, 10 and 11 check V. Every wait is
// bounded; on expiry the CTA records a status code, all roles stop, copies and MMAs in flight are drained, TMEM is
// freed and the rows not yet written get NaN.
#pragma once
#include <type_traits>

#include "decode_tc.cuh"

namespace palu {
namespace pf {

using namespace palu::tc;

constexpr int kPfThreads = 384;
constexpr int kRows = 128;      // rows of a chain
constexpr int kKeys = 128;      // keys of a tile
constexpr int kQBytes = 2 * kBox, kKBytes = 2 * kBox, kOutBytes = 32 * 128;
constexpr float kOutgrown = 65536.f;  // a tile's sum of exponentials above which a row's reference is looked at

// One work piece: key tiles [t0, t1) of one (query tile, KV head).
struct PfPiece {
  int32_t q0;    // first packed query position
  int32_t npos;  // query positions of the item (1 .. 2 * ppt)
  int32_t vis0;  // keys that the first position sees (may be <= 0)
  int32_t k0;    // packed index of the sequence's first key
  int32_t kvh;
  int32_t t0, t1;
  int32_t slot;  // -1: the whole item; else the index of its partial record
};
// One cut item: its records are slots slot0 .. slot0 + n - 1.
struct PfMerge {
  int32_t q0, npos, vis0, kvh, slot0, n;
};

struct PfParams {
  const PfPiece* pieces;
  const int32_t* cta_start;  // [gridDim.x + 1]
  __nv_bfloat16* out;        // [T][n_q][d_v]
  float* ws_o;               // [slots][2][d_v][128]: a chain's rows innermost
  float* ws_ml;              // [slots][256][2]
  int* status;
  const __nv_bfloat16* v;    // [Tk][n_kv][d_v] with the strides below (elements)
  int64_t v_tok, v_head;
  int n_q, rep, ppt, dv;
  float sl2;                 // scale * log2(e)
  unsigned long long wait_ns;
  int starve;                // test of the timeout path: the producer loads no V
};

template <bool ALIAS>
struct PfLayout {
  static constexpr int NS_K = 2, NS_V = ALIAS ? 2 : 3;
  // Registers a thread of the role warps and of the softmax warps: 4 x 32 and 8 x 32 threads of the 384 x 168 launched. (us for
  // 8192 tokens with 152 / 176, 136 / 184, 120 / 192: d_v 128 470, 485, 506; d_v 64 442, 429, 443.)
  static constexpr int ROLE_REGS = ALIAS ? 152 : 136, SOFT_REGS = ALIAS ? 176 : 184;
  static_assert(4 * 32 * ROLE_REGS + 8 * 32 * SOFT_REGS <= kPfThreads * 168, "the warpgroups' shares of the launch's registers");
  static constexpr int V_BYTES = ALIAS ? 2 * kBox : kBox;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * kQBytes;
  static constexpr int OFF_V = OFF_K + NS_K * kKBytes;
  static constexpr int OFF_OUT = OFF_V + NS_V * V_BYTES;  // 32 rows x 64 results (bf16) a softmax warp
  static constexpr int OFF_MISC = OFF_OUT + 8 * kOutBytes;
  static constexpr int TOTAL = OFF_MISC + 512 + kRows * 8 + 1024;
  // TMEM columns
  static constexpr uint32_t S = 0;                       // + 128 c
  static constexpr uint32_t P = ALIAS ? 0 : 256;         // + P_STEP c
  static constexpr uint32_t P_STEP = ALIAS ? 128 : 64;
  static constexpr uint32_t O = ALIAS ? 256 : 384;       // + O_STEP c
  static constexpr uint32_t O_STEP = ALIAS ? 128 : 64;
  static_assert(TOTAL <= kSmemBudget, "shared memory budget");
};

// The tiles that chain c of a piece works on: t0 .. t0 + n - 1.
struct PfChains {
  int n[2];
  int vis_first[2];  // keys that the chain's first position sees
  int vis_max;       // keys that the item's last position sees
  int nt;            // tiles of the piece
  bool active[2];
};
PALU_DEVINL PfChains chains_of(const PfPiece& w, int ppt) {
  PfChains s;
  s.vis_max = w.vis0 + w.npos - 1;
  s.nt = 0;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    s.active[c] = w.npos > c * ppt;
    s.vis_first[c] = w.vis0 + c * ppt;
    const int last = w.vis0 + min(w.npos, (c + 1) * ppt) - 1;  // keys that the chain's last position sees
    const int tiles = s.active[c] && last > 0 ? (last + kKeys - 1) / kKeys : 0;
    s.n[c] = max(0, min(w.t1, tiles) - w.t0);
    s.nt = max(s.nt, s.n[c]);
  }
  return s;
}
// Whether some row of the item does not see every key of tile t.
PALU_DEVINL bool tile_cut(const PfPiece& w, int t) { return (t + 1) * kKeys > w.vis0; }

PALU_DEVINL float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
PALU_DEVINL uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
PALU_DEVINL void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v)); }
PALU_DEVINL uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
PALU_DEVINL uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
PALU_DEVINL void touch16(uint32_t* r) {  // a use of r that stays behind the volatile wait before it
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                    "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
PALU_DEVINL void tmem_ld32p(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
PALU_DEVINL void tmem_st32p(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Nonzero when one of the two bf16 in w is an infinity or a NaN (exponent all ones).
PALU_DEVINL uint32_t nonfinite_bf16x2(uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; }

// w with its infinities and NaNs as zeros.
PALU_DEVINL uint32_t finite_bf16x2(uint32_t w) {
  const uint32_t f = nonfinite_bf16x2(w);
  return w & ~((f >> 15 & 1u) * 0xFFFFu | (f >> 31) * 0xFFFF0000u);
}
// Shared memory by its own address space: loads through generic pointers stay behind the global stores before them.
PALU_DEVINL uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
PALU_DEVINL int2 lds64(uint32_t at) {
  int2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
PALU_DEVINL bool elect_one() {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok));
  return ok != 0;
}

template <bool ALIAS>
__global__ void __launch_bounds__(kPfThreads, 1)
    palu_prefill_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const PfParams p) {
  using Lay = PfLayout<ALIAS>;
  constexpr int NS_K = Lay::NS_K, NS_V = Lay::NS_V;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int w0 = p.cta_start[blockIdx.x], w1 = p.cta_start[blockIdx.x + 1];

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Lay::OFF_MISC);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  // QF / QE: Q of chain c landed / free. KF / KE, VF / VE: ring slots. VC: the V tile of a cut tile has landed and is to
  // be checked (by count of cut tiles, four in turn: more than the V ring holds); the arrivals of the two warps
  // that check, instead of the copy's own, then complete VF, so that looking at some tiles only they never lose count of a
  // phase. SF: S_c written. SR: S_c read (P of its own only). PF: P_c written. OD: PV_c done. OE: O_c read by the epilogue.
  constexpr int B_QF = 0, B_QE = 2, B_KF = 4, B_KE = B_KF + NS_K, B_VF = B_KE + NS_K, B_VE = B_VF + NS_V,
                B_VC = B_VE + NS_V, B_SF = B_VC + 4, B_SR = B_SF + 2, B_PF = B_SR + 2, B_OD = B_PF + 2, B_OE = B_OD + 2,
                B_DRAIN = B_OE + 2, B_COUNT = B_DRAIN + 1;
  static_assert(B_COUNT * 8 + 64 <= 512, "misc area");
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + B_COUNT);
  int2* s_row = reinterpret_cast<int2*>(smem + Lay::OFF_MISC + 512);  // [128] a row's position and its place in the output behind the chain's
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  // 1 + index of the last piece with non-finite V so far. It only grows, so an epilogue that comes late still sees its piece's
  // mark; a mark of a later piece makes it look at V rows that hold nothing to add.
  volatile int* s_bad = reinterpret_cast<volatile int*>(s_tmem + 2);

  auto wait = [&](uint32_t b, uint32_t ph) -> bool { return mbar_wait(b, ph, s_abort, p.status, p.wait_ns); };
  auto wait_all = [&](uint32_t b, uint32_t ph) -> bool {
    if (__all_sync(0xffffffffu, mbar_try(b, ph))) return true;
    return __all_sync(0xffffffffu, mbar_wait_slow(b, ph, s_abort, p.status, p.wait_ns)) != 0;
  };

  // the same, inlined: the softmax warps run on more registers than the launch gave them, where no call compiles
  auto wait_all_inline = [&](uint32_t b, uint32_t ph) -> bool {
    bool done = mbar_try(b, ph);
    if (!done) {
      const unsigned long long t0 = globaltimer();
      while (!(done = mbar_try(b, ph))) {
        if (*s_abort) break;
        if (globaltimer() - t0 > p.wait_ns) {
          *s_abort = 1;
          atomicExch(p.status, kStatusTimeout);
          break;
        }
      }
    }
    return __all_sync(0xffffffffu, done) != 0;
  };

  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // the merge, which waits for this grid's end
  if (threadIdx.x == 0) {
    for (int c = 0; c < 2; ++c) {
      mbar_init(bar(B_QF + c), 1);
      mbar_init(bar(B_QE + c), 1);
      mbar_init(bar(B_SF + c), 1);
      mbar_init(bar(B_SR + c), 4);
      mbar_init(bar(B_PF + c), 4);
      mbar_init(bar(B_OD + c), 1);
      mbar_init(bar(B_OE + c), 4);
    }
    for (int s = 0; s < NS_K; ++s) {
      mbar_init(bar(B_KF + s), 1);
      mbar_init(bar(B_KE + s), 2);
    }
    for (int s = 0; s < NS_V; ++s) {
      mbar_init(bar(B_VF + s), 2);
      mbar_init(bar(B_VE + s), 2);
    }
    for (int s = 0; s < 4; ++s) mbar_init(bar(B_VC + s), 1);
    mbar_init(bar(B_DRAIN), 1);
    *s_abort = 0;
    *s_bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (threadIdx.x < kRows) {
    const int pos = threadIdx.x / p.rep;
    s_row[threadIdx.x] = make_int2(pos, (pos * p.n_q + (int)threadIdx.x - pos * p.rep) * p.dv);
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(s_tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *s_tmem;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(Lay::ROLE_REGS));
    if (warp == 8 && lane == 0) {
      // ============================== TMA producer ==============================
      tma_prefetch_map(&tm_q);
      tma_prefetch_map(&tm_k);
      tma_prefetch_map(&tm_v);
      const uint32_t q_bytes = (uint32_t)p.rep * p.ppt * 256;
      const int vbox = (p.dv + 63) >> 6;
      int nq[2] = {0, 0}, nk = 0, nv = 0, cut = 0;
      uint32_t history = 0;  // which of the last V tiles were cut
      bool ok = true;
      auto load_k = [&](const PfPiece& w, int t) -> bool {
        const int s = nk % NS_K, u = nk / NS_K;
        if (u >= 1 && !wait(bar(B_KE + s), (u - 1) & 1)) return false;
        mbar_expect_tx(bar(B_KF + s), kKBytes);
        for (int b = 0; b < 2; ++b)
          tma_load_3d(sbase + Lay::OFF_K + s * kKBytes + b * kBox, &tm_k, bar(B_KF + s), b * 64, w.kvh, w.k0 + t * kKeys);
        ++nk;
        return true;
      };
      for (int i = w0; ok && i < w1; ++i) {
        const PfPiece w = p.pieces[i];
        const PfChains ch = chains_of(w, p.ppt);
        for (int c = 0; ok && c < 2; ++c) {
          if (ch.n[c] == 0) continue;
          if (nq[c] >= 1 && !(ok = wait(bar(B_QE + c), (nq[c] - 1) & 1))) break;
          mbar_expect_tx(bar(B_QF + c), q_bytes);
          for (int b = 0; b < 2; ++b)
            tma_load_3d(sbase + Lay::OFF_Q + c * kQBytes + b * kBox, &tm_q, bar(B_QF + c), b * 64, w.kvh * p.rep,
                        w.q0 + c * p.ppt);
          ++nq[c];
          if (c == 0 && ch.nt > 0) ok = load_k(w, w.t0);
        }
        if (ok && ch.n[0] == 0 && ch.nt > 0) ok = load_k(w, w.t0);
        for (int j = 0; ok && j < ch.nt; ++j) {
          if (j + 1 < ch.nt && !(ok = load_k(w, w.t0 + j + 1))) break;
          const int s = nv % NS_V, u = nv / NS_V;
          if (u >= 1 && !(ok = wait(bar(B_VE + s), (u - 1) & 1))) break;
          if (p.starve) continue;
          const bool is_cut = tile_cut(w, w.t0 + j);
          const uint32_t full = is_cut ? bar(B_VC + (cut & 3)) : bar(B_VF + s);
          mbar_expect_tx(full, vbox * kBox);
          for (int b = 0; b < vbox; ++b)
            tma_load_3d(sbase + Lay::OFF_V + s * Lay::V_BYTES + b * kBox, &tm_v, full, b * 64, w.kvh,
                        w.k0 + (w.t0 + j) * kKeys);
          if (!is_cut) mbar_arrive(full);
          cut += is_cut;
          history = history << 1 | (uint32_t)is_cut;
          ++nv;
        }
      }
      if (*s_abort) {  // let every copy already issued land before the CTA can exit
        for (int c = 0; c < 2; ++c)
          if (nq[c] > 0) mbar_drain(bar(B_QF + c), (nq[c] - 1) & 1);
        for (int n = max(0, nk - NS_K); n < nk; ++n) mbar_drain(bar(B_KF + n % NS_K), (n / NS_K) & 1);
        for (int n = nv - 1; n >= max(0, nv - NS_V); --n, history >>= 1) {
          if (history & 1) {
            --cut;
            mbar_drain(bar(B_VC + (cut & 3)), (cut >> 2) & 1);
          } else {
            mbar_drain(bar(B_VF + n % NS_V), (n / NS_V) & 1);
          }
        }
      }
    } else if (warp == 9) {
      // ============================== MMA issuer ==============================
      // The whole warp runs this and one elected lane issues, so that what the instructions take stays warp-uniform. For
      // each tile, chain 0 then chain 1: PV_c of the tile, then the chain's next S (the next piece's first one included),
      // so that the chains' turns at the tensor cores alternate.
      const uint32_t ID_QK = idesc_f16(kKeys, 1, false, false), ID_PV = idesc_f16(p.dv, 1, false, true);
      const uint64_t q_desc = sdesc(sbase + Lay::OFF_Q, 16, 1024), k_desc = sdesc(sbase + Lay::OFF_K, 16, 1024),
                     v_desc = sdesc(sbase + Lay::OFF_V, kBox, 1024);
      int ns0 = 0, ns1 = 0, np0 = 0, np1 = 0, nq0 = 0, nq1 = 0, no0 = 0, no1 = 0;  // S, PV, Q loads and pieces per chain so far
      int kb = 0;                    // ring index of the piece's first tile
      int ahead0 = -1, ahead1 = -1;  // the piece whose first S the chain has issued already
      bool ok = true;
      auto commit = [&](uint32_t b) {
        if (elect_one()) mma_commit(b);
        __syncwarp();
      };
      auto issue_s = [&](int c, int& ns, int& nq, int n, bool first, bool last) -> bool {  // n: ring index of the K tile
        if (first && !wait_all(bar(B_QF + c), nq++ & 1)) return false;
        if (!ALIAS && ns >= 1 && !wait_all(bar(B_SR + c), (ns - 1) & 1)) return false;
        const int st = n % NS_K;
        if (!wait_all(bar(B_KF + st), (n / NS_K) & 1)) return false;
        fence_after();
        const uint64_t qd = q_desc + c * (kQBytes >> 4), kd = k_desc + st * (kKBytes >> 4);
        const uint32_t d = tmem + Lay::S + 128 * c;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t off = ((kk >> 2) * kBox + (kk & 3) * 32) >> 4;
            mma_ss(d, qd + off, kd + off, ID_QK, kk > 0);
          }
          mma_commit(bar(B_SF + c));
          mma_commit(bar(B_KE + st));
          if (last) mma_commit(bar(B_QE + c));
        }
        __syncwarp();
        ++ns;
        return true;
      };
      for (int i = w0; ok && i < w1; ++i) {
        const PfPiece w = p.pieces[i];
        const PfChains ch = chains_of(w, p.ppt);
        int nx0 = 0, nx1 = 0;
        if (i + 1 < w1) {
          const PfChains nx = chains_of(p.pieces[i + 1], p.ppt);
          nx0 = nx.n[0];
          nx1 = nx.n[1];
        }
        auto begin = [&](int c, int n, int ahead, int& ns, int& nq) {
          if (n > 0) {
            if (ahead != i) ok = issue_s(c, ns, nq, kb, true, n == 1);
          } else if (ch.nt > 0) {
            commit(bar(B_KE + kb % NS_K));
          }
        };
        begin(0, ch.n[0], ahead0, ns0, nq0);
        if (ok) begin(1, ch.n[1], ahead1, ns1, nq1);
        for (int j = 0; ok && j < ch.nt; ++j) {
          const int n = kb + j, sv = n % NS_V;
          const uint64_t vd = v_desc + sv * (Lay::V_BYTES >> 4);
          auto step = [&](int c, int mine, int next, int& ns, int& np, int& nq, int& no, int& ahead) -> bool {
            if (j >= mine) {  // this chain sees nothing of the tile
              commit(bar(B_VE + sv));
              if (j + 1 < ch.nt) commit(bar(B_KE + (n + 1) % NS_K));
              return true;
            }
            // the chain's next S: behind PV where P lies over S, else as soon as this S has been read
            auto next_s = [&]() -> bool {
              if (j + 1 < mine) return issue_s(c, ns, nq, n + 1, false, j + 2 == mine);
              if (j + 1 < ch.nt) commit(bar(B_KE + (n + 1) % NS_K));
              if (next > 0) {
                ahead = i + 1;
                return issue_s(c, ns, nq, kb + ch.nt, true, next == 1);
              }
              return true;
            };
            if (!ALIAS && !next_s()) return false;
            if (!wait_all(bar(B_VF + sv), (n / NS_V) & 1) || !wait_all(bar(B_PF + c), np & 1)) return false;
            if (j == 0 && no >= 1 && !wait_all(bar(B_OE + c), (no - 1) & 1)) return false;
            fence_after();
            const uint32_t d = tmem + Lay::O + Lay::O_STEP * c, a = tmem + Lay::P + Lay::P_STEP * c;
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < 8; ++kk) mma_ts(d, a + 8 * kk, vd + kk * (2048 >> 4), ID_PV, (j | kk) != 0);
              if (!ALIAS || j + 1 == mine) mma_commit(bar(B_OD + c));
              mma_commit(bar(B_VE + sv));
            }
            __syncwarp();
            ++np;
            no += j + 1 == mine;
            return !ALIAS || next_s();
          };
          ok = step(0, ch.n[0], nx0, ns0, np0, nq0, no0, ahead0) && step(1, ch.n[1], nx1, ns1, np1, nq1, no1, ahead1);
        }
        kb += ch.nt;
      }
      commit(bar(B_DRAIN));
      mbar_drain(bar(B_DRAIN), 0);
    } else if (warp >= 10) {
      // ============================== V of cut tiles ==============================
      const int half = warp - 10, chunks = p.dv >> 3;
      int kb = 0, cut = 0;
      bool ok = true;
      for (int i = w0; ok && i < w1; ++i) {
        const PfPiece w = p.pieces[i];
        const PfChains ch = chains_of(w, p.ppt);
        for (int j = 0; ok && j < ch.nt; ++j) {
          const int t = w.t0 + j;
          if (!tile_cut(w, t)) continue;
          const int sv = (kb + j) % NS_V;
          if (!(ok = wait_all(bar(B_VC + (cut & 3)), (cut >> 2) & 1))) break;
          unsigned char* sV = smem + Lay::OFF_V + sv * Lay::V_BYTES;
          const int r0 = max(0, w.vis0 - t * kKeys);         // rows below: every row of the item sees them
          const int r1 = min(kKeys, ch.vis_max - t * kKeys);  // rows from here on: none does
          uint32_t bad = 0;
          for (int r = r0 + half * 32 + lane; r < kKeys; r += 64) {  // a row a lane
            unsigned char* at = sV + r * 128;
            if (r >= r1) {
#pragma unroll 4
              for (int k = 0; k < chunks; ++k) *reinterpret_cast<uint4*>(at + (k >> 3) * kBox + (((k & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
              continue;
            }
#pragma unroll 4
            for (int k = 0; k < chunks; ++k) {
              uint4* x = reinterpret_cast<uint4*>(at + (k >> 3) * kBox + (((k & 7) ^ (r & 7)) << 4));
              uint4 v = *x;
              if (nonfinite_bf16x2(v.x) | nonfinite_bf16x2(v.y) | nonfinite_bf16x2(v.z) | nonfinite_bf16x2(v.w)) {
                bad = 1;
                v.x = finite_bf16x2(v.x);
                v.y = finite_bf16x2(v.y);
                v.z = finite_bf16x2(v.z);
                v.w = finite_bf16x2(v.w);
                *x = v;
              }
            }
          }
          if (bad) atomicMax(const_cast<int*>(s_bad), i + 1);
          fence_proxy_async();  // these reads and writes before the tensor core's reads and the slot's next copy
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(B_VF + sv));
          ++cut;
        }
        kb += ch.nt;
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(Lay::SOFT_REGS));
    // ============================== softmax ==============================
    const int c = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t tlane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tS = tlane + Lay::S + 128 * c, tP = tlane + Lay::P + Lay::P_STEP * c, tO = tlane + Lay::O + Lay::O_STEP * c;
    const int pos = row / p.rep, head = row - pos * p.rep;
    int n_s = 0, n_o = 0;  // tiles and pieces with tiles of this chain so far
    bool ok = true;
    int i = w0;
    PfPiece ahead;  // the next piece, read while this one is worked on
    if (w0 < w1) ahead = p.pieces[w0];
    for (; i < w1; ++i) {
      const PfPiece w = ahead;
      if (i + 1 < w1) ahead = p.pieces[i + 1];
      const PfChains ch = chains_of(w, p.ppt);
      if (!ch.active[c]) continue;
      const int lpos = c * p.ppt + pos;                       // position within the item
      const bool have = pos < p.ppt && lpos < w.npos;
      const int vis = have ? w.vis0 + lpos : 0;               // keys that this row sees
      float m_true = -INFINITY, m_ref = -INFINITY;
      float l = 0.f;
      const int nt = ch.n[c];
      for (int j = 0; j < nt; ++j, ++n_s) {
        if (!(ok = wait_all_inline(bar(B_SF + c), n_s & 1))) break;
        fence_after();
        const int kb = (w.t0 + j) * kKeys;
        const int nvis = kb + kKeys > ch.vis_first[c] ? vis - kb : kKeys;  // keys of the tile that this row sees
        const bool cut = kb + kKeys > ch.vis_first[c];
        uint32_t pk[64];
        float lt;  // the tile's sum
        // P of the tile against m_ref, and its sum
        auto stream = [&](auto is_cut) {
          constexpr bool CUT = decltype(is_cut)::value;
          const float mb = m_ref == -INFINITY ? 0.f : -__fmul_rn(m_ref, p.sl2);
          const uint64_t sl2 = pack2(p.sl2, p.sl2), mb2 = pack2(mb, mb);
          uint64_t l2[2] = {0, 0};
          uint32_t s[2][32];
          tmem_ld32p(tS, s[0]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t* x = s[q & 1];
            tmem_wait_ld();
            touch16(x);
            touch16(x + 16);
            if (q < 3) tmem_ld32p(tS + 32 * (q + 1), s[(q + 1) & 1]);
            if constexpr (CUT) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (32 * q + i >= nvis) x[i] = 0xFF800000u;  // -inf
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint64_t y = fma2(pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), sl2, mb2);
              float a, b;
              unpack2(y, a, b);
              a = fast_exp2(a);
              b = fast_exp2(b);
              l2[i & 1] = add2(l2[i & 1], pack2(a, b));
              pk[16 * q + i] = pack_bf16(a, b);
            }
          }
          float la, lb;
          unpack2(add2(l2[0], l2[1]), la, lb);
          lt = la + lb;
        };
        auto tile_max = [&](int chunks) -> float {
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
          for (int q = 0; q < chunks; ++q) {
            uint32_t x[32];
            tmem_ld32p(tS + 32 * q, x);
            tmem_wait_ld();
            touch16(x);
            touch16(x + 16);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * q + i >= nvis) x[i] = 0xFF800000u;
#pragma unroll
            for (int i = 0; i < 32; i += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y) mx[y] = max3_nan(mx[y], __uint_as_float(x[i + y]), __uint_as_float(x[i + 4 + y]));
          }
          return max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]);
        };
        if (j == 0) {  // a first reference: the maximum of the first keys
          m_true = tile_max(1);
          m_ref = isnan(m_true) ? 0.f : m_true;
        }
        for (;;) {
          if (cut) stream(std::true_type{});
          else stream(std::false_type{});
          // The maximum is looked at where the sum says that it may have outgrown the reference (a sum of at most 2^16 holds no
          // term above it; a NaN or infinity among the scores makes the sum NaN or huge), and while a row has no reference.
          const bool look = have && (!(lt <= kOutgrown) || (m_ref == -INFINITY && nvis > 0));
          if (!__any_sync(0xffffffffu, look)) break;
          const float tm = tile_max(4);
          float ref = m_ref;
          if (look) {
            m_true = max3_nan(m_true, tm, tm);
            if (tm > m_ref && tm < INFINITY) ref = tm;
          }
          if (!__any_sync(0xffffffffu, ref != m_ref)) break;
          // New references: O and l follow, and the tile is done over. By the references' products as the exponentials took them,
          // each rounded: at scores of 2^20 the difference taken first is off by up to 2^-3 from theirs.
          const float alpha = ref == m_ref ? 1.f : (m_ref == -INFINITY ? 0.f : fast_exp2(__fmul_rn(m_ref, p.sl2) - __fmul_rn(ref, p.sl2)));
          if (j > 0) {
            if (!ALIAS && !(ok = wait_all_inline(bar(B_OD + c), (n_s - 1) & 1))) break;  // PV of the tile before is in O
            fence_after();
            for (int x = 0; x < p.dv; x += 16) {
              uint32_t o[16];
              tmem_ld16(tO + x, o);
              tmem_wait_ld();
              touch16(o);
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
              tmem_st16(tO + x, o);
            }
            tmem_wait_st();
          }
          l *= alpha;
          m_ref = ref;
        }
        if (!ok) break;
        // PV of the tile before has read P; with P over S, S of this tile came behind it
        if (!ALIAS && j > 0 && !(ok = wait_all_inline(bar(B_OD + c), (n_s - 1) & 1))) break;
        if (!ALIAS) {
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(B_SR + c));
        }
        tmem_st32p(tP, pk);
        tmem_st32p(tP + 32, pk + 32);
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_PF + c));
        l += lt;
      }
      if (!ok) break;
      // ---- epilogue ----
      if (nt > 0) {
        if (!(ok = wait_all_inline(bar(B_OD + c), (ALIAS ? n_o : n_s - 1) & 1))) break;
        ++n_o;
        fence_after();
      }
      // a NaN or +infinity among the row's scores makes the row NaN, as do scores that are all -infinity
      const bool lost = isnan(m_true) || m_true == INFINITY || (m_ref == -INFINITY && vis > 0 && w.slot < 0);
      const bool bad = nt > 0 && *s_bad > i;
      const float inv = lost ? NAN : 1.f / l;
      for (int x = 0; x < p.dv; x += 64) {
        const uint32_t stage = sbase + Lay::OFF_OUT + warp * kOutBytes;
        const int width = min(64, p.dv - x);
#pragma unroll 1
        for (int y = 0; y < width; y += 32) {  // the last 16 columns may be behind d_v: read and dropped
          uint32_t o[32];
          if (nt > 0) {
            tmem_ld32p(tO + x + y, o);
            tmem_wait_ld();
            touch16(o);
            touch16(o + 16);
            if (x + y + 32 >= p.dv) {  // O has been read: the next piece's first PV may overwrite it
              fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(B_OE + c));
            }
          } else {
#pragma unroll
            for (int z = 0; z < 32; ++z) o[z] = 0;
          }
          if (bad && have) {  // non-finite values of the partly visible V rows, to the rows that see them
            const int k_lo = max(max(w.vis0, w.t0 * kKeys), 0), k_hi = min(vis, w.t1 * kKeys), n = min(32, width - y);
            for (int k = k_lo; k < k_hi; ++k) {
              const __nv_bfloat16* vr = p.v + (int64_t)(w.k0 + k) * p.v_tok + w.kvh * p.v_head + x + y;
              for (int z = 0; z < n; ++z) {
                const float f = __bfloat162float(vr[z]);
                if (!(fabsf(f) < INFINITY)) {
#pragma unroll
                  for (int q = 0; q < 32; ++q)
                    if (q == z) o[q] = __float_as_uint(__uint_as_float(o[q]) + f);
                }
              }
            }
          }
          if (w.slot >= 0) {
            float* po = p.ws_o + (((size_t)w.slot * 2 + c) * p.dv + x + y) * kRows + row;
#pragma unroll
            for (int z = 0; z < 32; ++z)
              if (y + z < width) po[z * kRows] = __uint_as_float(o[z]);
          } else {
            // through shared memory, so that 8 lanes write 128 bytes of a row: chunk k of row r at chunk k ^ r & 7 (straight from
            // the registers, every store touched 32 lines: 3000 to 4000 cycles a piece at d_v 128; now 1300, the warps' stores
            // coming behind their loads, not in turn with them)
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              uint32_t h[4];
#pragma unroll
              for (int q = 0; q < 4; ++q)
                h[q] = vis <= 0 ? 0u : pack_bf16(__uint_as_float(o[8 * z + 2 * q]) * inv, __uint_as_float(o[8 * z + 2 * q + 1]) * inv);
              *reinterpret_cast<uint4*>(smem + Lay::OFF_OUT + warp * kOutBytes + lane * 128 + ((((y >> 3) + z) ^ (lane & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
            }
          }
        }
        if (w.slot < 0) {
          __syncwarp();
          const int k = lane & 7, npos = min(p.ppt, w.npos - c * p.ppt);
          __nv_bfloat16* out = p.out + (((size_t)w.q0 + c * p.ppt) * p.n_q + w.kvh * p.rep) * p.dv + x + 8 * k;
          const uint32_t rows = sbase + Lay::OFF_MISC + 512 + ((warp & 3) * 32 + (lane >> 3)) * 8;
#pragma unroll 1
          for (int z0 = 0; z0 < 8; z0 += 4) {
            uint4 v[4];
            int2 at[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const int r = 4 * (z0 + z) + (lane >> 3);
              v[z] = lds128(stage + r * 128 + ((k ^ (r & 7)) << 4));
              at[z] = lds64(rows + (z0 + z) * 32);
            }
#pragma unroll
            for (int z = 0; z < 4; ++z)
              if (at[z].x < npos && 8 * k < width) *reinterpret_cast<uint4*>(out + at[z].y) = v[z];
          }
          __syncwarp();
        }
      }
      if (w.slot >= 0 && have) {
        float* ml = p.ws_ml + ((size_t)w.slot * 2 * kRows + c * kRows + row) * 2;
        ml[0] = lost ? NAN : (m_ref == -INFINITY ? -INFINITY : __fmul_rn(m_ref, p.sl2));
        ml[1] = l;
      }
    }
    if (!ok) {  // the rows that this chain still owed become NaN
      for (; i < w1; ++i) {
        const PfPiece w = p.pieces[i];
        const int lpos = c * p.ppt + pos;
        if (pos >= p.ppt || lpos >= w.npos) continue;
        if (w.slot >= 0) {
          p.ws_ml[((size_t)w.slot * 2 * kRows + c * kRows + row) * 2] = NAN;
          continue;
        }
        __nv_bfloat16* go = p.out + (((size_t)w.q0 + lpos) * p.n_q + w.kvh * p.rep + head) * p.dv;
        for (int x = 0; x < p.dv; ++x) go[x] = __float2bfloat16(NAN);
      }
    }
  }
  // every role reaches this point warp-converged
  fence_before();
  __syncthreads();
  if (warp == 9) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// Joins the records of the items that were cut along the keys: with w_s = 2^(m_s - max m),
// o = sum_s w_s O_s / sum_s w_s l_s. A block joins 32 rows (a lane a row, a warp every eighth column) and writes them
// through shared memory. For few records an item, whose loads it issues record by record. Launched as a programmatic
// dependent of the attention (one query on 4000 keys 24.9 -> 22.4 us one call after another).
__global__ void __launch_bounds__(256) palu_prefill_merge_kernel(const PfMerge* merges, const PfParams p) {
  __shared__ float s_o[32][129];
  const PfMerge w = merges[blockIdx.x];
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.y * 32 + lane, c = r >> 7, row = r & 127, lpos = c * p.ppt + row / p.rep;
  if (c * p.ppt + (blockIdx.y * 32 & 127) / p.rep >= w.npos) return;  // the block's first row is behind the item
  const bool have = row / p.rep < p.ppt && lpos < w.npos, empty = w.vis0 + lpos <= 0;
  float m = -INFINITY;
  bool lost = false;
  for (int s = 0; s < w.n; ++s) {
    const float ms = have ? p.ws_ml[((size_t)(w.slot0 + s) * 2 * kRows + r) * 2] : -INFINITY;
    lost |= isnan(ms);
    m = fmaxf(m, ms);
  }
  float l = 0.f, o[16];
#pragma unroll
  for (int y = 0; y < 16; ++y) o[y] = 0.f;
  for (int s = 0; s < w.n; ++s) {
    const size_t rec = (size_t)(w.slot0 + s) * 2 * kRows + r;
    const float ms = have ? p.ws_ml[rec * 2] : -INFINITY;
    if (ms == -INFINITY) continue;  // the row saw nothing of this piece
    const float wt = fast_exp2(ms - m);
    l += wt * p.ws_ml[rec * 2 + 1];
    const float* po = p.ws_o + (((size_t)(w.slot0 + s) * 2 + c) * p.dv) * kRows + row;
#pragma unroll
    for (int y = 0; y < 16; ++y)
      if (warp + 8 * y < p.dv) o[y] += wt * po[(warp + 8 * y) * kRows];
  }
  const float inv = lost ? NAN : 1.f / l;
#pragma unroll
  for (int y = 0; y < 16; ++y)
    if (warp + 8 * y < p.dv) s_o[lane][warp + 8 * y] = empty ? 0.f : o[y] * inv;
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * (p.dv / 2); e += 256) {
    const int rr = e / (p.dv / 2), x = e - rr * (p.dv / 2), row2 = (blockIdx.y * 32 + rr) & 127, pos = row2 / p.rep, lp = c * p.ppt + pos;
    if (pos >= p.ppt || lp >= w.npos) continue;
    *reinterpret_cast<uint32_t*>(p.out + (((size_t)w.q0 + lp) * p.n_q + w.kvh * p.rep + row2 % p.rep) * p.dv + 2 * x) =
        pack_bf16(s_o[rr][2 * x], s_o[rr][2 * x + 1]);
  }
}

// The same for many records an item (few queries on many keys): a block joins 32 rows of 32 columns, its 8 warps take the
// records in turn, all of a record's loads at once, and meet in shared memory. Bound by latency. us, with this kernel and with
// the one above: 64 queries on 32768 keys (19 records) 64 and 69; 512 on 8192 (3 records) 77 and 66: from 8 records on.
constexpr int kDeepRecords = 8;
__global__ void __launch_bounds__(256) palu_prefill_merge_deep_kernel(const PfMerge* merges, const PfParams p) {
  __shared__ float s_o[8][32][33], s_l[8][32];
  const PfMerge w = merges[blockIdx.x];
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = (int)blockIdx.y >> 2, row0 = (int)(blockIdx.y & 3) * 32, row = row0 + lane, x0 = blockIdx.z * 32;
  if (c * p.ppt + row0 / p.rep >= w.npos) return;  // the block's first row is behind the item
  const int pos = row / p.rep, lpos = c * p.ppt + pos;
  const bool have = pos < p.ppt && lpos < w.npos;
  const float* ml = p.ws_ml + ((size_t)w.slot0 * 2 * kRows + c * kRows + row) * 2;
  float m = -INFINITY;
  bool lost = false;
#pragma unroll 4
  for (int s = 0; s < w.n; ++s) {
    const float ms = have ? ml[(size_t)s * 4 * kRows] : -INFINITY;
    lost |= isnan(ms);
    m = fmaxf(m, ms);
  }
  float l = 0.f, o[32];
#pragma unroll
  for (int y = 0; y < 32; ++y) o[y] = 0.f;
  for (int s = warp; s < w.n; s += 8) {
    const float ms = have ? ml[(size_t)s * 4 * kRows] : -INFINITY;
    if (ms == -INFINITY) continue;  // the row saw nothing of this piece
    const float wt = fast_exp2(ms - m);
    l += wt * ml[(size_t)s * 4 * kRows + 1];
    const float* po = p.ws_o + (((size_t)(w.slot0 + s) * 2 + c) * p.dv + x0) * kRows + row;
#pragma unroll
    for (int y = 0; y < 32; ++y)
      if (x0 + y < p.dv) o[y] += wt * po[y * kRows];
  }
#pragma unroll
  for (int y = 0; y < 32; ++y) s_o[warp][lane][y] = o[y];
  s_l[warp][lane] = l;
  __syncthreads();
  // a warp writes 4 rows: sums over the warps' parts, 8 lanes a row, 4 columns a lane
  const int r = warp * 4 + (lane >> 3), y0 = (lane & 7) * 4;
  float sum[4] = {0.f, 0.f, 0.f, 0.f}, total = 0.f;
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    total += s_l[x][r];
#pragma unroll
    for (int y = 0; y < 4; ++y) sum[y] += s_o[x][r][y0 + y];
  }
  const bool bad = __shfl_sync(0xffffffffu, (int)lost, r) != 0;
  const int rpos = (row0 + r) / p.rep, rl = c * p.ppt + rpos;
  if (rpos < p.ppt && rl < w.npos && x0 + y0 < p.dv) {
    const float inv = bad ? NAN : 1.f / total;
    const bool empty = w.vis0 + rl <= 0;
    const uint2 h = empty ? make_uint2(0u, 0u) : make_uint2(pack_bf16(sum[0] * inv, sum[1] * inv), pack_bf16(sum[2] * inv, sum[3] * inv));
    *reinterpret_cast<uint2*>(p.out + (((size_t)w.q0 + rl) * p.n_q + w.kvh * p.rep + (row0 + r) % p.rep) * p.dv + x0 + y0) = h;
  }
}

}  // namespace pf
}  // namespace palu
