// Packed keys and values of cached latents: for token t of a row's cached prefix and KV head h with latent head g(h),
//   K[t, h] = R_pos (c_k[g, pos] U_k[h]),   V[t, h] = c_v[g, pos] U_v[h]   (or c_v itself where V stays absorbed),
// with R_pos rotating the pairs (2f, 2f + 1) by the table's cos and sin. Products accumulate in fp32, the rotation is
// fp32, and each result is rounded to bf16 once (half a step, 2^-8).
//
// Bound by memory: at rank 64 a token and head reads 128 B and writes 256 B for 16 kFLOP, a sixth of what the tensor
// cores could do meanwhile, so warp-level mma.sync reaches the same bound as tcgen05 would and keeps the accumulators in
// registers, where a rotation pair sits in one thread and the rotation is free. What it takes is loads in flight: a CTA
// takes 64 tokens and half of the head dims for all its heads (with all 128 dims, accumulators and table rows left room
// for 8 warps an SM, and 32 rows of 8192 tokens took 610 us), copies latents and U of the next head (cp.async) while the
// current one is multiplied, keeps its tokens' table rows in registers for all heads, and writes whole 128-byte lines.
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
__host__ __device__ constexpr int stage_bytes(int r) { return kTokens * lat_stride(r) + r * kUStride; }
constexpr int kOutBytes = kTokens * kUStride;

// Source row of a cached position, or null where the page table names no block.
PALU_DEVINL const __nv_bfloat16* lat_row(const Params& p, const __nv_bfloat16* base, int r, int row, int g, int pos) {
  if (!p.page_table) return base + (((int64_t)row * p.n_groups + g) * p.max_seq + pos) * r;
  const int b = p.page_table[(int64_t)row * p.table_ld + (pos >> p.blk_shift)];
  if ((unsigned)b >= (unsigned)p.n_blocks) return nullptr;
  return base + ((((int64_t)b * p.n_groups + g) << p.blk_shift) + (pos & ((1 << p.blk_shift) - 1))) * r;
}

__global__ void __launch_bounds__(kThreads, 4) palu_rebuild_kv_kernel(const Params p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int4 tile = p.tiles[blockIdx.x / p.units];
  const int unit = blockIdx.x % p.units;
  const int row = tile.x, pos0 = tile.y, count = tile.w;
  const int64_t tok0 = tile.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (unit == 2 * p.runs) {  // gathered V: the latent heads as they are
    const int ch = p.r_v >> 3, total = count * p.n_groups * ch;
    for (int e0 = tid; e0 < total; e0 += 4 * kThreads) {
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e0 + i * kThreads, t = e / (p.n_groups * ch), x = e - t * p.n_groups * ch, g = x / ch;
        v[i] = make_uint4(0, 0, 0, 0);
        if (e < total) {
          const __nv_bfloat16* src = lat_row(p, p.v_lat, p.r_v, row, g, pos0 + t);
          if (src) v[i] = *reinterpret_cast<const uint4*>(src + (x - g * ch) * 8);
        }
      }
      uint4* dst = reinterpret_cast<uint4*>(p.v_out + tok0 * p.n_groups * p.r_v);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e0 + i * kThreads < total) dst[e0 + i * kThreads] = v[i];
    }
    return;
  }

  const int half = unit & 1, j0 = (unit >> 1) * p.per_cta, j1 = min(p.jobs, j0 + p.per_cta);
  const int r_max = p.u_v ? max(p.r_k, p.r_v) : p.r_k, stage_sz = stage_bytes(r_max);
  const uint32_t sb = smem_u32(smem);
  const int gs = p.n_kv / p.n_groups;

  auto copy_job = [&](int job, int buf) {  // latents and half of U of a K or V head
    const bool is_v = job >= p.n_kv;
    const int h = is_v ? job - p.n_kv : job, g = h / gs, r = is_v ? p.r_v : p.r_k, ch = r >> 3;
    const __nv_bfloat16* lat = is_v ? p.v_lat : p.k_lat;
    const __nv_bfloat16* u = (is_v ? p.u_v : p.u_k) + (int64_t)h * r * kHeadDim + half * kHalf;
    const uint32_t dl = sb + buf * stage_sz, du = dl + kTokens * lat_stride(r);
    for (int e = tid; e < kTokens * ch; e += kThreads) {
      const int t = e / ch, c = e - t * ch;
      const __nv_bfloat16* src = t < count ? lat_row(p, lat, r, row, g, pos0 + t) : nullptr;
      cp_async16(dl + t * lat_stride(r) + c * 16, src ? src + c * 8 : lat, src ? 16 : 0);
    }
    for (int e = tid; e < r * 8; e += kThreads)
      cp_async16(du + (e >> 3) * kUStride + (e & 7) * 16, u + (e >> 3) * kHeadDim + (e & 7) * 8, 16);
    cp_async_commit();
  };

  float cs[2][8], sn[2][8];  // frequency 32 half + 4 j + lane % 4 of rows lane / 4 and + 8 of the warp's 16 tokens
  copy_job(j0, 0);
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
  for (int job = j0; job < j1; ++job) {
    const int buf = (job - j0) & 1;
    if (job + 1 < j1) {
      copy_job(job + 1, buf ^ 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    const bool is_v = job >= p.n_kv;
    const int h = is_v ? job - p.n_kv : job, r = is_v ? p.r_v : p.r_k;
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int x = 0; x < 4; ++x) acc[j][x] = 0.f;
    const uint32_t sl = sb + buf * stage_sz, su = sl + kTokens * lat_stride(r);
    const uint32_t a_at = sl + (warp * 16 + (lane & 15)) * lat_stride(r) + (lane >> 4) * 16;
    const uint32_t b_at = su + (lane & 15) * kUStride + (lane >> 4) * 16;
#pragma unroll 2
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
    unsigned char* out = smem + 2 * stage_sz + warp * 16 * kUStride;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float a = acc[j][2 * y], b = acc[j][2 * y + 1];
        const uint32_t w = is_v ? pack_bf16(a, b) : pack_bf16(a * cs[y][j] - b * sn[y][j], b * cs[y][j] + a * sn[y][j]);
        *reinterpret_cast<uint32_t*>(out + ((lane >> 2) + 8 * y) * kUStride + (8 * j + 2 * (lane & 3)) * 2) = w;
      }
    __syncwarp();
    __nv_bfloat16* dst = (is_v ? p.v_out : p.k_out) + half * kHalf;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = i * 4 + (lane >> 3), c = lane & 7;
      if (warp * 16 + t < count)
        *reinterpret_cast<uint4*>(dst + ((tok0 + warp * 16 + t) * p.n_kv + h) * kHeadDim + c * 8) =
            *reinterpret_cast<const uint4*>(out + t * kUStride + c * 16);
    }
    __syncthreads();  // the stage and the out rows are free
  }
}

}  // namespace rb
}  // namespace palu
