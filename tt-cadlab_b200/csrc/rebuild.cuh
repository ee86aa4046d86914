// Packed keys and values of cached latents: for token t of a row's cached prefix and KV head h with latent head g(h),
//   K[t, h] = R_pos (c_k[g, pos] U_k[h]),   V[t, h] = c_v[g, pos] U_v[h]   (or c_v itself where V stays absorbed),
// with R_pos rotating the pairs (2f, 2f + 1) by the table's cos and sin. Products accumulate in fp32, the rotation is
// fp32, and each result is rounded to bf16 once (half a step, 2^-8).
//
// Bound by memory: at rank 64 a token and head reads 128 B and writes 256 B for 16 kFLOP. The products run on tcgen05, which
// reads its operands from shared memory by itself: with warp-level mma.sync the fragments' trips through the load/store
// pipe (144 wavefronts of 128 B per 16 x 64 results) were what bound, 316 us for 32 rows of 8192 tokens at rank 64.
//
// A unit is 128 tokens of a row and a run of heads; CTAs are persistent, one an SM. Per head: TMA brings the latents' tile
// (once per latent head; from a paged cache one box a page) and U_h, tcgen05.mma writes D = c U (128 x 128, f32) to one of
// four TMEM buffers, and 8 warps turn it into results: a thread has a token's row and 64 head dims (a warp reads the 32 TMEM
// lanes of its quarter), with the token's 32 frequencies of the table in registers for all heads of the unit. A warp of its
// own sends the rows on from shared memory by TMA, so that the result warps wait for no store (each of them issuing its own
// took 25 % of its time; stored by the lanes, half). Four warps bring the next unit's table rows to shared memory meanwhile
// (loaded by the warps that use them, between units, they cost as much as the unit's heads); neighbouring units of the same
// positions share them. Warps 0..7: results, 8: TMA producer, 9: MMA issuer, 10: stores, 12 to 15: table.
//
// 32 rows of 8192 tokens, 8 heads, rank 64: K 152 us (805 MB), with the copy of absorbed V 237. The 537 MB of results alone
// take 139 us at the rate at which this GPU writes without reading (3850 GB/s, a plain fill); without the table's loads K takes
// 143. Every wait is bounded; on expiry the plan's status word is set and the results not yet written become NaN.
#pragma once
#include "prefill_tc.cuh"

namespace palu {
namespace rb {

using namespace palu::tc;
using palu::pf::elect_one;
using palu::pf::touch16;
using palu::pf::tmem_ld32p;

constexpr int kTokens = 128, kThreads = 512, kDBufs = 4, kMaxRing = 4, kTableWarps = 4;
// Neighbouring units of a CTA. 32 rows of 8192 tokens, us, with 1 / 2 / 4 / 8: 259, 246, 241, 239.
constexpr int kBlock = 4;
constexpr int kRoleRegs = 72, kResultRegs = 184;  // of the 128 x 512 launched
static_assert(8 * 32 * kRoleRegs + 8 * 32 * kResultRegs <= kThreads * 128, "the warpgroups' shares of the launch's registers");
constexpr int kOutBytes = 32 * 128;          // a warp's 32 rows x 64 results
constexpr int kTableBytes = kTokens * 512;  // a token's 64 cosines, then its 64 sines (fp32)
constexpr int kFixedSmem = kTableBytes + 512 + 1024;  // and the rings, and one or two sets of the 8 warps' result buffers

struct Params {
  const __nv_bfloat16 *k_lat, *v_lat, *u_k, *u_v;  // u_v null: V is gathered
  const float *cos, *sin;                          // [>= positions][128], each frequency twice
  __nv_bfloat16 *k_out, *v_out;
  const int4* tiles;                               // row, first position, packed token, tokens (<= 128)
  const int32_t* page_table;                       // null: contiguous [B][n_groups][max_seq][r]
  int table_ld, blk_shift, n_blocks;
  int n_kv, n_groups, group, r_k, r_v, max_seq;    // group: KV heads of a latent head
  int jobs, per_unit, runs;                        // heads to multiply (K, then V), per unit, runs of them
  int waves, rest, rest_more;                      // whole rounds of kBlock units a CTA; of what is left, units a CTA, CTAs with one more
  int ring, a_bytes, u_bytes, out_bufs;            // slots of the latent and the U ring, bytes of one; result buffers a warp
  int* status;
  unsigned long long wait_ns;
  int starve;  // test of the timeout path: the producer loads no U
};

PALU_DEVINL void cp_async4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}

// The heads of a unit, one after another: K of all heads, then V. No division in the loops over them (of a single warp's time
// they took more than the products).
struct Jobs {
  int j0, j1, job, h, g, k, gs;  // k: the head's place in its group of gs
  PALU_DEVINL Jobs(const Params& p, int run) {
    j0 = job = run * p.per_unit;
    j1 = min(p.jobs, j0 + p.per_unit);
    gs = p.group;
    h = job >= p.n_kv ? job - p.n_kv : job;
    g = h / gs;
    k = h - g * gs;
  }
  PALU_DEVINL bool more() const { return job < j1; }
  PALU_DEVINL bool is_v(const Params& p) const { return job >= p.n_kv; }
  PALU_DEVINL bool new_a() const { return job == j0 || k == 0; }                // its latents differ from the job's before it
  PALU_DEVINL bool last_of_a() const { return job == j1 - 1 || k == gs - 1; }  // and from the one's behind it
  PALU_DEVINL void next(const Params& p) {
    ++job;
    if (job == p.n_kv) h = g = k = 0;
    else {
      ++h;
      if (++k == gs) {
        k = 0;
        ++g;
      }
    }
  }
};
// A CTA's units: kBlock neighbours of every kBlock * gridDim.x, and its share of what is left over. (The plan puts the tiles
// of the same positions of up to kBlock sequences next to one another, so neighbours share the table's rows, while the CTAs
// together stay in a small part of the caches and results.)
struct Walk {
  int tile, run, left, wave;  // left: units to go in the CTA's block
  PALU_DEVINL explicit Walk(const Params& p) {
    wave = 0;
    block(p);
  }
  PALU_DEVINL void block(const Params& p) {
    const int c = blockIdx.x, base = wave * (int)gridDim.x * kBlock;
    const int at = wave < p.waves ? base + c * kBlock : base + c * p.rest + min(c, p.rest_more);
    left = wave < p.waves ? kBlock : p.rest + (c < p.rest_more);
    tile = at / p.runs;
    run = at - tile * p.runs;
  }
  PALU_DEVINL bool more() const { return left > 0; }
  PALU_DEVINL void next(const Params& p) {
    if (++run == p.runs) {
      run = 0;
      ++tile;
    }
    if (--left == 0 && wave < p.waves) {
      ++wave;
      block(p);
    }
  }
};
// Whether the table's rows of a unit's tokens are those that the CTA holds already.
struct Held {
  int pos = -1, tokens = 0;
  PALU_DEVINL bool has(const int4& tile) {
    if (tile.y == pos && tile.w <= tokens) return true;
    pos = tile.y;
    tokens = tile.w;
    return false;
  }
};
// A place in a ring of `n`, and the parity of how often it has been passed.
struct Place {
  int at = 0, turn = 0;
  PALU_DEVINL void next(int n) {
    if (++at == n) {
      at = 0;
      ++turn;
    }
  }
};

__global__ void __launch_bounds__(kThreads, 1)
    palu_rebuild_kv_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const __grid_constant__ CUtensorMap tm_uk, const __grid_constant__ CUtensorMap tm_uv,
                           const __grid_constant__ CUtensorMap tm_ko, const __grid_constant__ CUtensorMap tm_vo, const Params p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int off_u = p.ring * p.a_bytes, off_out = off_u + p.ring * p.u_bytes,
            off_table = off_out + p.out_bufs * 8 * kOutBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + off_table + kTableBytes);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  constexpr int B_AF = 0, B_AE = kMaxRing, B_UF = 2 * kMaxRing, B_UE = 3 * kMaxRing, B_DF = 4 * kMaxRing, B_DE = B_DF + kDBufs,
                B_TF = B_DE + kDBufs, B_TE = B_TF + 1, B_OF = B_TE + 1, B_OE = B_OF + 2, B_DRAIN = B_OE + 2, B_COUNT = B_DRAIN + 1;
  static_assert(B_COUNT * 8 + 16 <= 512, "misc area");
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + B_COUNT);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  auto wait = [&](uint32_t b, uint32_t ph) -> bool { return mbar_wait(b, ph, s_abort, p.status, p.wait_ns); };
  auto wait_all = [&](uint32_t b, uint32_t ph) -> bool {
    if (__all_sync(0xffffffffu, mbar_try(b, ph))) return true;
    return __all_sync(0xffffffffu, mbar_wait_slow(b, ph, s_abort, p.status, p.wait_ns)) != 0;
  };
  // the same without a call, for the warps that hold the table's rows in registers
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
  if (threadIdx.x == 0) {
    for (int i = 0; i < B_DE; ++i) mbar_init(bar(i), 1);
    for (int i = 0; i < kDBufs; ++i) mbar_init(bar(B_DE + i), 8);
    mbar_init(bar(B_TF), kTableWarps);
    mbar_init(bar(B_TE), 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(B_OF + i), 8);
      mbar_init(bar(B_OE + i), 1);
    }
    mbar_init(bar(B_DRAIN), 1);
    *s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kRoleRegs));
    if (warp == 8) {
      if (lane == 0) {
        // ============================== TMA producer ==============================
        int na = 0, nu = 0;  // copies so far
        Place pa, pu;
        bool ok = true;
        for (Walk u(p); ok && u.more(); u.next(p)) {
          const int4 tile = p.tiles[u.tile];
          for (Jobs x(p, u.run); x.more(); x.next(p)) {
            const bool is_v = x.is_v(p);
            const int r = is_v ? p.r_v : p.r_k;
            if (x.new_a()) {
              const int s = pa.at;
              if (pa.turn >= 1 && !(ok = wait(bar(B_AE + s), (pa.turn - 1) & 1))) break;
              const CUtensorMap* tm = is_v ? &tm_v : &tm_k;
              const int nbox = (r + 63) >> 6;
              const uint32_t dst = sbase + s * p.a_bytes, full = bar(B_AF + s);
              mbar_expect_tx(full, nbox * kBox);
              if (!p.page_table) {
                for (int c = 0; c < nbox; ++c) tma_load_3d(dst + c * kBox, tm, full, c * 64, tile.y, tile.x * p.n_groups + x.g);
              } else {
                // one box a page (pages of 2^blk_shift rows; a whole number of swizzle atoms); pages that the table does not
                // name, and those behind the row, are read past the tensor: zeros
                const int sub = kTokens >> p.blk_shift, first = tile.y >> p.blk_shift, last = (tile.y + tile.w - 1) >> p.blk_shift;
                for (int i = 0; i < sub; ++i) {
                  int b = p.n_blocks;
                  if (first + i <= last) {
                    const int e = p.page_table[(int64_t)tile.x * p.table_ld + first + i];
                    if ((unsigned)e < (unsigned)p.n_blocks) b = e;
                  }
                  for (int c = 0; c < nbox; ++c)
                    tma_load_3d(dst + c * kBox + (i << p.blk_shift) * 128, tm, full, c * 64, 0, b * p.n_groups + x.g);
                }
              }
              ++na;
              pa.next(p.ring);
            }
            const int s = pu.at;
            if (pu.turn >= 1 && !(ok = wait(bar(B_UE + s), (pu.turn - 1) & 1))) break;
            if (p.starve) continue;
            const CUtensorMap* tm = is_v ? &tm_uv : &tm_uk;
            mbar_expect_tx(bar(B_UF + s), r * 256);
            for (int c = 0; c < 2; ++c)
              tma_load_2d(sbase + off_u + s * p.u_bytes + c * r * 128, tm, bar(B_UF + s), c * 64, x.h * r);
            ++nu;
            pu.next(p.ring);
          }
        }
        if (*s_abort) {  // let every copy already issued land before the CTA can exit
          for (int n = max(0, na - p.ring); n < na; ++n) mbar_drain(bar(B_AF + n % p.ring), (n / p.ring) & 1);
          for (int n = max(0, nu - p.ring); n < nu; ++n) mbar_drain(bar(B_UF + n % p.ring), (n / p.ring) & 1);
        }
      }
      __syncwarp();
    } else if (warp == 9) {
      // ============================== MMA issuer ==============================
      constexpr uint32_t ID = idesc_f16(128, 1, false, true);  // latents (K-major) x U (MN-major)
      int nu = 0;
      Place pa, pu;
      bool ok = true;
      for (Walk u(p); ok && u.more(); u.next(p)) {
        for (Jobs x(p, u.run); x.more(); x.next(p)) {
          const int r = x.is_v(p) ? p.r_v : p.r_k;
          const int sa = pa.at, su = pu.at, d = nu % kDBufs, use = nu / kDBufs;
          if (x.new_a() && !(ok = wait_all(bar(B_AF + sa), pa.turn & 1))) break;
          if (!(ok = wait_all(bar(B_UF + su), pu.turn & 1))) break;
          if (use >= 1 && !(ok = wait_all(bar(B_DE + d), (use - 1) & 1))) break;
          fence_after();
          const bool last = x.last_of_a();
          const uint64_t a = sdesc(sbase + sa * p.a_bytes, 16, 1024), b = sdesc(sbase + off_u + su * p.u_bytes, r * 128, 1024);
          if (elect_one()) {
            for (int kk = 0; kk < r >> 4; ++kk)
              mma_ss(tmem + d * 128, a + (((kk >> 2) * kBox + (kk & 3) * 32) >> 4), b + kk * (2048 >> 4), ID, kk > 0);
            mma_commit(bar(B_DF + d));
            mma_commit(bar(B_UE + su));
            if (last) mma_commit(bar(B_AE + sa));
          }
          __syncwarp();
          ++nu;
          pu.next(p.ring);
          if (last) pa.next(p.ring);
        }
      }
      if (elect_one()) mma_commit(bar(B_DRAIN));
      __syncwarp();
      mbar_drain(bar(B_DRAIN), 0);
    } else if (warp == 10) {
      // ============================== stores ==============================
      // A head's whole blocks of 32 rows, from the result warps' buffers, by TMA; blocks that the tile's end cuts were stored
      // by their warps. One group of stores a head.
      int n = 0;
      bool ok = true;
      for (Walk u(p); u.more(); u.next(p)) {
        const int4 tile = p.tiles[u.tile];
        for (Jobs x(p, u.run); x.more(); x.next(p), ++n) {
          const int b = n & (p.out_bufs - 1), use = p.out_bufs == 2 ? n >> 1 : n;
          const bool is_v = x.is_v(p);
          if (ok) ok = wait_all(bar(B_OF + b), use & 1);
          if (ok) {
            if (elect_one()) {
              const uint64_t map = reinterpret_cast<uint64_t>(is_v ? &tm_vo : &tm_ko);
              for (int w = 0; w < 8; ++w)
                if ((w & 3) * 32 + 32 <= tile.w)
                  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];\n" ::"l"(map),
                               "r"(sbase + off_out + (b * 8 + w) * kOutBytes), "r"(64 * (w >> 2)), "r"(x.h), "r"(tile.z + (w & 3) * 32)
                               : "memory");
              asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
              asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
              mbar_arrive(bar(B_OE + b));
            }
            __syncwarp();
          } else {  // what an expired wait kept from being computed
            __nv_bfloat16* dst = (is_v ? p.v_out : p.k_out) + ((int64_t)tile.z * p.n_kv + x.h) * kHeadDim;
            for (int i = lane; i < tile.w * kHeadDim; i += 32) dst[(int64_t)(i >> 7) * p.n_kv * kHeadDim + (i & 127)] = __float2bfloat16(NAN);
          }
        }
      }
      if (elect_one()) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
      __syncwarp();
    } else if (warp >= 12) {
      // ============================== table ==============================
      // The next unit's table rows, while its predecessor's heads are worked on: 4-byte copies, which leave out each
      // frequency's second place; a lane a frequency, 32 of them 128 bytes, whose 16-byte chunk k goes to k ^ (row & 7).
      const uint32_t table = sbase + off_table + (lane & 3) * 4;
      Held held;
      int n = 0;
      bool ok = true;
      for (Walk u(p); ok && u.more(); u.next(p)) {
        if (u.run * p.per_unit >= p.n_kv) continue;  // V heads only
        const int4 tile = p.tiles[u.tile];
        if (held.has(tile)) continue;
        if (n >= 1 && !(ok = wait_all(bar(B_TE), (n - 1) & 1))) break;
        ++n;
#pragma unroll 4
        for (int r = warp - 12; r < kTokens; r += kTableWarps) {
          const int64_t at = (int64_t)(tile.y + min(r, tile.w - 1)) * kHeadDim + 2 * lane;
          const uint32_t to = table + r * 512 + (((lane >> 2) ^ (r & 7)) << 4);
          cp_async4(to, p.cos + at);
          cp_async4(to + 128, p.cos + at + 64);
          cp_async4(to + 256, p.sin + at);
          cp_async4(to + 384, p.sin + at + 64);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_TF));
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kResultRegs));
    // ============================== results ==============================
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t tD = tmem + ((uint32_t)(quarter * 32) << 16) + 64 * half;
    float cs[32], sn[32];  // the token's frequencies 32 half .. + 31
    Held held;
    int nu = 0, n_t = 0;
    bool ok = true;
    for (Walk u(p); ok && u.more(); u.next(p)) {
      const int4 tile = p.tiles[u.tile];
      Jobs x(p, u.run);
      if (x.j0 < p.n_kv && !held.has(tile)) {
        if (!(ok = wait_all_inline(bar(B_TF), n_t & 1))) break;
        ++n_t;
        const unsigned char* at = smem + off_table + row * 512 + half * 128;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 c = *reinterpret_cast<const float4*>(at + ((i ^ (row & 7)) << 4));
          const float4 s = *reinterpret_cast<const float4*>(at + 256 + ((i ^ (row & 7)) << 4));
          cs[4 * i] = c.x;
          cs[4 * i + 1] = c.y;
          cs[4 * i + 2] = c.z;
          cs[4 * i + 3] = c.w;
          sn[4 * i] = s.x;
          sn[4 * i + 1] = s.y;
          sn[4 * i + 2] = s.z;
          sn[4 * i + 3] = s.w;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_TE));
      }
      for (; x.more(); x.next(p)) {
        const bool is_v = x.is_v(p);
        const int d = nu % kDBufs, b = nu & (p.out_bufs - 1), use = p.out_bufs == 2 ? nu >> 1 : nu;
        if (!(ok = wait_all_inline(bar(B_DF + d), (nu / kDBufs) & 1))) break;
        fence_after();
        uint32_t v[64];
        tmem_ld32p(tD + d * 128, v);
        tmem_ld32p(tD + d * 128 + 32, v + 32);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) touch16(v + 16 * i);
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_DE + d));
        if (!is_v) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float a = __uint_as_float(v[2 * i]), b = __uint_as_float(v[2 * i + 1]);
            v[2 * i] = __float_as_uint(a * cs[i] - b * sn[i]);
            v[2 * i + 1] = __float_as_uint(b * cs[i] + a * sn[i]);
          }
        }
        // the warp's 32 rows x 128 bytes, in the layout that a swizzled TMA store takes
        if (use >= 1 && !(ok = wait_all_inline(bar(B_OE + b), (use - 1) & 1))) break;
        unsigned char* stage = smem + off_out + (b * 8 + warp) * kOutBytes;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t h[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) h[q] = pack_bf16(__uint_as_float(v[8 * i + 2 * q]), __uint_as_float(v[8 * i + 2 * q + 1]));
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_proxy_async();
        __syncwarp();
        if (quarter * 32 + 32 > tile.w) {
          __nv_bfloat16* dst = (is_v ? p.v_out : p.k_out) + ((int64_t)(tile.z + quarter * 32) * p.n_kv + x.h) * kHeadDim + 64 * half;
          const int64_t step = (int64_t)p.n_kv * kHeadDim;
          const int k = lane & 7;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3);
            if (quarter * 32 + r < tile.w)
              *reinterpret_cast<uint4*>(dst + r * step + 8 * k) = *reinterpret_cast<const uint4*>(stage + r * 128 + ((k ^ (r & 7)) << 4));
          }
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(bar(B_OF + b));
        ++nu;
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

// Absorbed V: the cached latents of a tile's tokens as they are, 8 lanes 128 bytes of a token and latent head. A copy: bound by
// reading and writing it once (32 rows of 8192 tokens, 8 latent heads of 64: 84 us, 6400 GB/s).
constexpr int kGatherThreads = 256;
__global__ void __launch_bounds__(kGatherThreads) palu_gather_latents_kernel(const Params p) {
  const int4 tile = p.tiles[blockIdx.x];
  const int t8 = threadIdx.x >> 3, c8 = threadIdx.x & 7, ch = p.r_v >> 3;
  int64_t at[4];  // cache rows of the tokens t8, t8 + 32, ... for latent head 0; each further head `step` rows on
  const int step = p.page_table ? 1 << p.blk_shift : p.max_seq;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t8 + 32 * i, pos = tile.y + t;
    at[i] = -1;
    if (t < tile.w) {
      if (!p.page_table) {
        at[i] = (int64_t)tile.x * p.n_groups * p.max_seq + pos;
      } else {
        const int b = p.page_table[(int64_t)tile.x * p.table_ld + (pos >> p.blk_shift)];
        if ((unsigned)b < (unsigned)p.n_blocks) at[i] = (((int64_t)b * p.n_groups) << p.blk_shift) + (pos & (step - 1));
      }
    }
  }
  for (int g = blockIdx.y; g < p.n_groups; g += gridDim.y)
    for (int c = c8; c < ch; c += 8) {
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = make_uint4(0, 0, 0, 0);
        if (at[i] >= 0) v[i] = *reinterpret_cast<const uint4*>(p.v_lat + (at[i] + (int64_t)g * step) * p.r_v + c * 8);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t8 + 32 * i < tile.w)
          *reinterpret_cast<uint4*>(p.v_out + ((int64_t)(tile.z + t8 + 32 * i) * p.n_groups + g) * p.r_v + c * 8) = v[i];
    }
}

}  // namespace rb
}  // namespace palu
