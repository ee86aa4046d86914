// Packed keys and values of cached latents: for token t of a row's cached prefix and KV head h with latent head g(h),
//   K[t, h] = R_pos (c_k[g, pos] U_k[h]),   V[t, h] = c_v[g, pos] U_v[h]   (or c_v itself where V stays absorbed),
// with R_pos rotating the pairs (2f, 2f + 1) by the table's cos and sin. Products accumulate in fp32, the rotation is
// fp32, and each result is rounded to bf16 once (half a step, 2^-8).
//
// Bound by memory: at rank 64 a token and head reads 128 B and writes 256 B for 16 kFLOP, a sixth of what the tensor
// cores could do meanwhile, so warp-level mma.sync reaches the same bound as tcgen05 would and keeps the accumulators in
// registers, where a rotation pair sits in one thread and the rotation is free. What it takes is loads in flight: a CTA
// takes 64 tokens and half of the head dims for all its heads (with all 128 dims, accumulators and table rows left room
// for 8 warps an SM, and 32 rows of 8192 tokens took 610 us), copies latents and U (cp.async) two heads ahead of the products, keeps its tokens' table rows in registers for all heads, and writes whole 128-byte lines.
// Gathered values are a copy by CTAs of their own. The CTAs of a tile are neighbours, so that its latents and table
// rows come from DRAM once.
#pragma once
#include "palu_common.cuh"

namespace palu {
namespace rb {

constexpr int kTokens = 64, kThreads = 128;

struct Params {
  const __nv_bfloat16 *k_lat, *v_lat, *u_k, *u_v;  // u_v null: V is gathered
  const float *cos, *sin;                          // [>= positions][128], each frequency twice
  __nv_bfloat16 *k_out, *v_out;
  const int4* tiles;                               // row, first position, packed token, tokens (<= 64)
  const int32_t* page_table;                       // null: contiguous [B][n_groups][max_seq][r]
  int table_ld, blk_shift, n_blocks;
  int n_kv, n_groups, r_k, r_v, max_seq;
  int jobs, per_cta, runs;                         // heads to multiply (K, then V), of a CTA, and runs of them
  int units;                                       // CTAs of a tile: 2 halves of each run, then one for gathered values
};

// Rows of a staged tile are padded by 16 bytes: 8 rows then start 4 banks apart (r / 2 + 4 or 36 words, odd multiples
// of 4).
__host__ __device__ constexpr int lat_stride(int r) { return r * 2 + 16; }
constexpr int kHalf = 64, kUStride = kHalf * 2 + 16;
constexpr int kStages = 3;
// A warp's results go where its 16 latent rows were: their room is the larger of the two.
__host__ __device__ constexpr int lat_bytes(int r) { return kTokens * (lat_stride(r) > kUStride ? lat_stride(r) : kUStride); }
__host__ __device__ constexpr int stage_bytes(int r) { return lat_bytes(r) + r * kUStride; }

// Row of a cached position in a cache of any width, for latent head 0 (each further head `step` rows on), or -1 where the
// page table names no block.
PALU_DEVINL int64_t cache_row(const Params& p, int row, int pos) {
  if (!p.page_table) return (int64_t)row * p.n_groups * p.max_seq + pos;
  const int b = p.page_table[(int64_t)row * p.table_ld + (pos >> p.blk_shift)];
  if ((unsigned)b >= (unsigned)p.n_blocks) return -1;
  return (((int64_t)b * p.n_groups) << p.blk_shift) + (pos & ((1 << p.blk_shift) - 1));
}
PALU_DEVINL void stsm_x4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// R: the K latents' width where it is at most 128 and values are not rebuilt, known to the compiler (the loops over it are
// then straight code); 0: any widths, K and V heads.
template <int R>
__global__ void __launch_bounds__(kThreads, 4) palu_rebuild_kv_kernel(const Params p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int4 tile = p.tiles[blockIdx.x / p.units];
  const int unit = blockIdx.x % p.units;
  const int row = tile.x, pos0 = tile.y, count = tile.w;
  const int64_t tok0 = tile.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // 8 threads copy a token's row, 16 bytes each: token tid / 8 and every 16th after it
  const int t8 = tid >> 3, c8 = tid & 7, step = p.page_table ? 1 << p.blk_shift : p.max_seq;
  int64_t at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = t8 + 16 * i < count ? cache_row(p, row, pos0 + t8 + 16 * i) : -1;

  if (unit == 2 * p.runs) {  // gathered V: the latent heads as they are
    const int ch = p.r_v >> 3;
    for (int g = 0; g < p.n_groups; ++g)
      for (int c = c8; c < ch; c += 8) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = make_uint4(0, 0, 0, 0);
          if (at[i] >= 0) v[i] = *reinterpret_cast<const uint4*>(p.v_lat + (at[i] + (int64_t)g * step) * p.r_v + c * 8);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t8 + 16 * i < count)
            *reinterpret_cast<uint4*>(p.v_out + ((tok0 + t8 + 16 * i) * p.n_groups + g) * p.r_v + c * 8) = v[i];
      }
    return;
  }

  const int half = unit & 1, j0 = (unit >> 1) * p.per_cta, j1 = min(p.jobs, j0 + p.per_cta);
  const int stage_sz = stage_bytes(R ? R : (p.u_v ? max(p.r_k, p.r_v) : p.r_k));
  const uint32_t sb = smem_u32(smem);
  const int gs = p.n_kv / p.n_groups;

  // The next head to copy: its latents (4 token rows) and U, as pointers that move from head to head.
  int h_l = 0, in_group = 0, r_l = 0;
  bool v_l = false;
  const __nv_bfloat16 *src_l[4], *u_l = nullptr;
  auto seek = [&](int job) {
    v_l = R == 0 && job >= p.n_kv;
    h_l = v_l ? job - p.n_kv : job;
    r_l = R ? R : (v_l ? p.r_v : p.r_k);
    const int g = h_l / gs;
    in_group = h_l - g * gs;
    const __nv_bfloat16* lat = v_l ? p.v_lat : p.k_lat;
#pragma unroll
    for (int i = 0; i < 4; ++i) src_l[i] = lat + (at[i] >= 0 ? (at[i] + (int64_t)g * step) * r_l + c8 * 8 : 0);
    u_l = (v_l ? p.u_v : p.u_k) + ((int64_t)h_l * r_l + t8) * kHeadDim + half * kHalf + c8 * 8;
  };
  auto copy_job = [&](int buf) {
    const int r = R ? R : r_l, ch = r >> 3;
    const uint32_t dl = sb + buf * stage_sz, ls = lat_stride(r), wl = lat_bytes(r) / 4, dt = dl + t8 * ls + c8 * 16;
    const uint32_t du = dl + lat_bytes(r) + t8 * kUStride + c8 * 16;
    if constexpr (R != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < R / 8; c += 8)
          if (c + 8 <= R / 8 || c + c8 < R / 8) cp_async16(dt + i * wl + c * 16, src_l[i] + c * 8, at[i] >= 0 ? 16 : 0);
#pragma unroll
      for (int k = 0; k < R; k += 16) cp_async16(du + k * kUStride, u_l + k * kHeadDim, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        for (int c = 0; c + c8 < ch; c += 8) cp_async16(dt + i * wl + c * 16, src_l[i] + c * 8, at[i] >= 0 ? 16 : 0);
#pragma unroll 4
      for (int k = 0; k < r; k += 16) cp_async16(du + k * kUStride, u_l + k * kHeadDim, 16);
    }
    cp_async_commit();
    ++h_l;
    u_l += (R ? R : r_l) * kHeadDim;
    if (R == 0 && h_l == p.n_kv) {
      if (!v_l && p.u_v) seek(p.n_kv);
    } else if (++in_group == gs) {
      in_group = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at[i] >= 0) src_l[i] += (int64_t)step * (R ? R : r_l);
    }
  };

  float cs[2][8], sn[2][8];  // frequency 32 half + 4 j + lane % 4 of rows lane / 4 and + 8 of the warp's 16 tokens
  seek(j0);
  copy_job(0);
  if (j0 + 1 < j1) copy_job(1);
  if (j0 < p.n_kv) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int t = warp * 16 + (lane >> 2) + 8 * y, pos = pos0 + min(t, count - 1);
      const int64_t at = (int64_t)pos * kHeadDim + kHalf * half + 2 * (lane & 3);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[y][j] = __ldg(p.cos + at + 8 * j);
        sn[y][j] = __ldg(p.sin + at + 8 * j);
      }
    }
  }
  const int64_t dst0 = (tok0 + warp * 16 + (lane >> 3)) * p.n_kv * kHeadDim + half * kHalf + (lane & 7) * 8;
  const int64_t dst_step = (int64_t)4 * p.n_kv * kHeadDim;
  int buf = 0;
  for (int job = j0; job < j1; ++job, buf = buf == kStages - 1 ? 0 : buf + 1) {
    if (job + 1 < j1) cp_async_wait<1>();
    else cp_async_wait<0>();
    __syncthreads();  // this head's copies have landed, and the stage of the head before it is free
    if (job + 2 < j1) copy_job(buf == 0 ? 2 : buf - 1);
    const bool is_v = R == 0 && job >= p.n_kv;
    const int h = is_v ? job - p.n_kv : job, r = R ? R : (is_v ? p.r_v : p.r_k);
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[j][x] = 0.f;
    const uint32_t sl = sb + buf * stage_sz, su = sl + lat_bytes(r);
    const uint32_t a_at = sl + warp * (lat_bytes(r) / 4) + (lane & 15) * lat_stride(r) + (lane >> 4) * 16;
    const uint32_t b_at = su + (lane & 15) * kUStride + (lane >> 4) * 16;
#pragma unroll(R ? R / 16 : 2)
    for (int k = 0; k < r; k += 16) {
      uint32_t a0, a1, a2, a3;
      ldsm_x4(a_at + k * 2, a0, a1, a2, a3);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(b_at + k * kUStride + j * 32, b0, b1, b2, b3);
        mma_bf16(acc[2 * j], a0, a1, a2, a3, b0, b1);
        mma_bf16(acc[2 * j + 1], a0, a1, a2, a3, b2, b3);
      }
    }
    if (!is_v) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float a = acc[j][2 * y], b = acc[j][2 * y + 1];
          acc[j][2 * y] = a * cs[y][j] - b * sn[y][j];
          acc[j][2 * y + 1] = b * cs[y][j] + a * sn[y][j];
        }
    }
    // 16 rows of 64 results through shared memory: 8 x 8 blocks (rows 0..7 and 8..15 of columns 8 j, then 8 j + 8)
    __syncwarp();
    unsigned char* out = smem + buf * stage_sz + warp * (lat_bytes(r) / 4);
    const uint32_t so = smem_u32(out) + (lane & 15) * kUStride + (lane >> 4) * 16;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      uint32_t w[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int jj = j + (x >> 1), y = x & 1;
        const float a = acc[jj][2 * y], b = acc[jj][2 * y + 1];
        w[x] = pack_bf16(a, b);
      }
      stsm_x4(so + j * 16, w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
    __nv_bfloat16* dst = (is_v ? p.v_out : p.k_out) + dst0 + h * kHeadDim;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (warp * 16 + i * 4 + (lane >> 3) < count)
        *reinterpret_cast<uint4*>(dst + i * dst_step) =
            *reinterpret_cast<const uint4*>(out + (i * 4 + (lane >> 3)) * kUStride + (lane & 7) * 16);
  }
}

}  // namespace rb
}  // namespace palu
