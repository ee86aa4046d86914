// C ABI of the operators around the decode step: packed prompts (plan, attention, rebuilt keys and values), scores of tokens,
// pages. Validation, planning and dispatch on the host; the kernels live in the .cuh files next to it.
#include <algorithm>
#include <atomic>
#include <exception>
#include <functional>
#include <utility>
#include <vector>

#include "../../include/palu_b200.h"
#include "abi_common.h"
#include "logprobs.cuh"
#include "pages.cuh"
#include "prefill_tc.cuh"
#include "rebuild.cuh"

using namespace palu::abi;

namespace {

// cudaFuncSetAttribute's dynamic shared memory limit, set once per kernel and device (`done`: one word per kernel, a bit per
// device; racing threads set the same value). Kernels whose size varies are given the largest they can need.
int allow_smem(const void* kern, int bytes, std::atomic<uint64_t>& done, const char* what) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return cuda_check(what);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return PALU_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return cuda_check(what);
  done.fetch_or(bit, std::memory_order_relaxed);
  return PALU_OK;
}

// ---- the plan of a packed batch -----------------------------------------------------------------------

constexpr int64_t kPlanHeader = 256;  // the blob starts with the status word
// Cost model of a piece, in key tiles: its tiles plus the pipeline's fill and the epilogue. Cutting items along the
// keys costs a merge launch, worth about kMergeTiles tiles of one CTA.
constexpr int kPieceTiles = 2, kMergeTiles = 6, kMinCut = 4;

struct Item {
  int32_t q0, npos, vis0, k0, tiles;
};

int64_t up16(int64_t x) { return (x + 15) / 16 * 16; }

// The work lists of a packed batch; see palu_prefill_plan in the header.
struct Lists {
  std::vector<int32_t> start;
  std::vector<palu::pf::PfPiece> pieces;
  std::vector<palu::pf::PfMerge> merges;
  std::vector<int4> tiles;
  int slots = 0;
};

// Whole items, heaviest first, each to the CTA with the least so far. Returns the largest CTA's cost.
int64_t deal_whole(const std::vector<Item>& items, int n_kv, int ctas, Lists* out) {
  typedef std::pair<int64_t, int> Load;
  std::vector<Load> heap(ctas);  // the least on top
  for (int c = 0; c < ctas; ++c) heap[c] = {0, c};
  std::vector<std::vector<palu::pf::PfPiece>> per(out ? ctas : 0);
  int64_t most = 0;
  for (const Item& it : items)
    for (int h = 0; h < n_kv; ++h) {
      std::pop_heap(heap.begin(), heap.end(), std::greater<Load>());
      const int c = heap.back().second;
      most = std::max(most, heap.back().first += it.tiles + kPieceTiles);
      std::push_heap(heap.begin(), heap.end(), std::greater<Load>());
      if (out) per[c].push_back({it.q0, it.npos, it.vis0, it.k0, h, 0, it.tiles, -1});
    }
  if (out) {
    out->start.assign(1, 0);
    for (auto& v : per) {
      out->pieces.insert(out->pieces.end(), v.begin(), v.end());
      out->start.push_back((int32_t)out->pieces.size());
    }
  }
  return most;
}

// Items cut along the keys so that no CTA gets more than `share`; false if that takes more than `ctas` CTAs.
bool deal_cut(const std::vector<Item>& items, int n_kv, int ctas, int64_t share, Lists* out) {
  int c = 0, slots = 0;
  int64_t left = share;
  if (out) out->start.assign(1, 0);
  auto close = [&]() {
    ++c;
    left = share;
    if (out) out->start.push_back((int32_t)out->pieces.size());
  };
  for (const Item& it : items)
    for (int h = 0; h < n_kv; ++h) {
      int t = 0, first = -1, n = 0;
      do {
        const int rest = it.tiles - t;
        int take = rest;
        if (rest + kPieceTiles > left) {
          take = (int)std::max<int64_t>(0, left - kPieceTiles);
          // no crumbs on either side of a cut
          if (rest - take < kMinCut) take = rest - kMinCut;
          if (take < kMinCut) {
            if (left < share) {
              close();
              continue;
            }
            take = rest;
          }
        }
        if (c >= ctas) return false;
        const bool whole = t == 0 && take == it.tiles;
        if (out) out->pieces.push_back({it.q0, it.npos, it.vis0, it.k0, h, t, t + take, whole ? -1 : slots});
        if (!whole) {
          if (first < 0) first = slots;
          ++slots;
          ++n;
        }
        left -= take + kPieceTiles;
        t += take;
        if (left <= kPieceTiles) close();
        if (it.tiles == 0) break;
      } while (t < it.tiles);
      if (out && first >= 0) out->merges.push_back({it.q0, it.npos, it.vis0, h, first, n});
    }
  if (out) {
    while ((int)out->start.size() < ctas + 1) out->start.push_back((int32_t)out->pieces.size());
    out->start.resize(ctas + 1);
    out->start[ctas] = (int32_t)out->pieces.size();
    out->slots = slots;
  }
  return c < ctas || (c == ctas && left == share);
}

void make_lists(const int32_t* q_lens, const int32_t* k_lens, const int32_t* rows, int n_seq, int n_kv, int ppt,
                int ctas, Lists& out) {
  std::vector<Item> items;
  int32_t q0 = 0, k0 = 0;
  size_t group = 0;
  for (int s = 0; s < n_seq; ++s) {
    const int ql = q_lens[s], kl = k_lens[s], step = 2 * ppt;
    for (int a = 0; a < ql; a += step) {
      const int n = std::min(step, ql - a), vis0 = kl - ql + a + 1, last = vis0 + n - 1;
      items.push_back({q0 + a, n, vis0, k0, last > 0 ? (last + palu::pf::kKeys - 1) / palu::pf::kKeys : 0});
    }
    for (int a = 0; a < kl; a += palu::rb::kTokens)
      out.tiles.push_back(make_int4(rows ? rows[s] : s, a, k0 + a, std::min(palu::rb::kTokens, kl - a)));
    q0 += ql;
    k0 += kl;
    if (s % palu::rb::kBlock == palu::rb::kBlock - 1 || s == n_seq - 1) {  // the same positions of some sequences next to one another
      std::stable_sort(out.tiles.begin() + group, out.tiles.end(), [](const int4& a, const int4& b) { return a.y < b.y; });
      group = out.tiles.size();
    }
  }
  std::stable_sort(items.begin(), items.end(), [](const Item& a, const Item& b) { return a.tiles > b.tiles; });
  int64_t total = 0;
  for (const Item& it : items) total += (int64_t)(it.tiles + kPieceTiles) * n_kv;
  const int64_t n = (int64_t)items.size() * n_kv;
  const int used = (int)std::min<int64_t>(ctas, n);
  if (used == 0) {
    out.start.assign(1, 0);
    return;
  }
  const int64_t whole = deal_whole(items, n_kv, used, nullptr);
  int64_t share = std::max<int64_t>((total + ctas - 1) / ctas, kMinCut + kPieceTiles);
  // cuts add pieces: grow the share until the pieces fit the CTAs
  while (share < whole && !deal_cut(items, n_kv, ctas, share, nullptr)) share += std::max<int64_t>(1, share / 32);
  if (share + kMergeTiles < whole) {
    deal_cut(items, n_kv, ctas, share, &out);
  } else {
    deal_whole(items, n_kv, used, &out);
  }
}

// ---- pages --------------------------------------------------------------------------------------------

int check_pool(const palu_page_pool* q, palu::pg::Pool& p) {
  if (!q) return fail(PALU_ERR_INVALID, "pool is NULL");
  if (!q->table || !q->refs || !q->mapped || !q->status) return fail(PALU_ERR_INVALID, "pool: table, refs, mapped and status must be set");
  if (q->rows <= 0 || q->blocks_per_row <= 0 || q->n_blocks <= 0 || q->block_size <= 0)
    return fail(PALU_ERR_INVALID, "pool: rows, blocks_per_row, n_blocks and block_size must be positive (got %d, %d, %d, %d)", q->rows,
                q->blocks_per_row, q->n_blocks, q->block_size);
  if ((int64_t)q->rows * q->blocks_per_row > INT32_MAX) return fail(PALU_ERR_INVALID, "pool: a table of more than 2^31 - 1 entries");
  p = {q->table, q->refs, q->mapped, q->status, q->rows, q->blocks_per_row, q->n_blocks, q->block_size};
  return PALU_OK;
}

int check_rows(const char* what, const int32_t* rows, const int32_t* lens, int n, const palu::pg::Pool& p) {
  if (n < 0 || (n > 0 && !rows)) return fail(PALU_ERR_INVALID, "%s must hold n entries", what);
  for (int i = 0; i < n; ++i) {
    if (rows[i] < 0 || rows[i] >= p.rows) return fail(PALU_ERR_INVALID, "%s: row %d is outside [0, %d)", what, rows[i], p.rows);
    if (lens && (lens[i] < 0 || lens[i] > (int64_t)p.per_row * p.page_size))
      return fail(PALU_ERR_INVALID, "%s: a row of %d blocks of %d cannot hold %d positions", what, p.per_row, p.page_size, lens[i]);
  }
  std::vector<int32_t> s(rows, rows + n);
  std::sort(s.begin(), s.end());
  for (int i = 1; i < n; ++i)
    if (s[i] == s[i - 1]) return fail(PALU_ERR_INVALID, "%s: row %d is named twice", what, s[i]);
  return PALU_OK;
}

// Caches of one launch, and whether all of them take 16-byte accesses.
int check_caches(const palu_page_cache* caches, int n, int n_blocks) {
  if (n < 0 || (n > 0 && !caches)) return fail(PALU_ERR_INVALID, "caches must hold n_caches entries");
  for (int i = 0; i < n; ++i)
    if (!caches[i].base || caches[i].block_bytes <= 0 || (n_blocks > 1 && caches[i].block_stride < caches[i].block_bytes))
      return fail(PALU_ERR_INVALID, "cache %d: blocks of %lld bytes every %lld bytes", i, (long long)caches[i].block_bytes,
                  (long long)caches[i].block_stride);
  return PALU_OK;
}
bool fill_caches(const palu_page_cache* caches, int n, palu::pg::Caches& a, int64_t& most) {
  a.n = n;
  most = 0;
  bool wide = true;
  for (int i = 0; i < n; ++i) {
    a.c[i] = {static_cast<unsigned char*>(caches[i].base), caches[i].block_stride, caches[i].block_bytes};
    most = std::max(most, caches[i].block_bytes);
    wide &= (reinterpret_cast<uintptr_t>(caches[i].base) | caches[i].block_stride | caches[i].block_bytes) % 16 == 0;
  }
  return wide;
}
// Thread blocks per cache: kCopyCtas for every SM over all caches, no more than there are units.
int copy_grid(int n_caches, int64_t moves, int64_t most) {
  const int64_t units = moves * ((most + palu::pg::kPart - 1) / palu::pg::kPart);
  const int64_t fill = ((int64_t)palu::pg::kCopyCtas * device_sms() + n_caches - 1) / std::max(1, n_caches);
  return (int)std::max<int64_t>(1, std::min(units, fill));
}

template <class K, class... A>
int launch_dependent(const char* what, K kern, dim3 grid, int threads, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) return cuda_check(what);
  return cuda_check(what);
}

// The move list behind a state change, applied to every cache (and the table, with a target array).
int apply_moves(const palu::pg::Pool& p, const palu::pg::Moves& mv, const int32_t* target, const palu_page_cache* caches, int n_caches,
                int64_t most_moves, cudaStream_t stream) {
  for (int i = 0; i < n_caches || (i == 0 && target); i += palu::pg::kMaxCaches) {
    palu::pg::Caches a;
    int64_t most;
    const int n = std::min(palu::pg::kMaxCaches, n_caches - i);
    const bool wide = fill_caches(caches + i, n, a, most);
    const dim3 grid(copy_grid(n, most_moves, std::max<int64_t>(most, 1)), std::max(1, n));
    const int32_t* t = i == 0 ? target : nullptr;
    const int st = wide ? launch_dependent("page move launch", palu::pg::palu_move_pages_kernel<uint4>, grid, palu::pg::kCopyThreads, stream, p, mv, t, a)
                        : launch_dependent("page move launch", palu::pg::palu_move_pages_kernel<uint8_t>, grid, palu::pg::kCopyThreads, stream, p, mv, t, a);
    if (st) return st;
  }
  return PALU_OK;
}

// Runs f and turns a C++ exception (all that can throw is a list's allocation) into a status.
template <class F>
int guarded(F f) {
  g_err.clear();
  try {
    return f();
  } catch (const std::exception& e) {
    return fail(PALU_ERR_INVALID, "out of host memory (%s)", e.what());
  }
}

}  // namespace

extern "C" {

int palu_plan_prefill(const int32_t* q_lens, const int32_t* k_lens, const int32_t* rows, int32_t n_seq, int32_t n_q_heads,
                      int32_t n_kv_heads, int32_t n_ctas, void* buf, size_t buf_bytes, palu_prefill_plan* plan) {
  g_err.clear();
  if (!plan) return fail(PALU_ERR_INVALID, "plan is NULL");
  if (n_seq < 0 || (n_seq > 0 && (!q_lens || !k_lens))) return fail(PALU_ERR_INVALID, "q_lens and k_lens must hold n_seq lengths");
  if (n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0)
    return fail(PALU_ERR_INVALID, "KV head count %d must divide the %d query heads", n_kv_heads, n_q_heads);
  const int rep = n_q_heads / n_kv_heads;
  if (n_q_heads > 65536) return fail(PALU_ERR_INVALID, "at most 65536 query heads are supported, got %d", n_q_heads);
  if (rep > palu::pf::kRows) return fail(PALU_ERR_INVALID, "at most 128 query heads per KV head are supported, got %d", rep);
  if (n_ctas < 0 || n_ctas > 4096) return fail(PALU_ERR_INVALID, "n_ctas must be in [0, 4096], got %d", n_ctas);
  int64_t tq = 0, tk = 0, items = 0;
  const int step = 2 * (palu::pf::kRows / rep);  // query positions of a work item
  int32_t longest = 0, last_row = -1;
  for (int s = 0; s < n_seq; ++s) {
    if (q_lens[s] < 0 || k_lens[s] < 0)
      return fail(PALU_ERR_INVALID, "sequence %d: lengths must not be negative (got %d queries, %d keys)", s, q_lens[s], k_lens[s]);
    if (rows && rows[s] < 0) return fail(PALU_ERR_INVALID, "sequence %d: cache row %d is negative", s, rows[s]);
    tq += q_lens[s];
    items += (q_lens[s] + (int64_t)step - 1) / step;
    tk += k_lens[s];
    longest = std::max(longest, k_lens[s]);
    last_row = std::max(last_row, rows ? rows[s] : s);
  }
  if (tq > (1 << 28) || tk > (1 << 28)) return fail(PALU_ERR_INVALID, "at most 2^28 packed tokens are supported");
  if (items * n_kv_heads > (1 << 28)) return fail(PALU_ERR_INVALID, "at most 2^28 work items (query tiles x KV heads) are supported");
  try {
    Lists l;
    const int ppt = palu::pf::kRows / rep;
    make_lists(q_lens, k_lens, rows, n_seq, n_kv_heads, ppt, n_ctas ? n_ctas : device_sms(), l);
    plan->q_tokens = tq;
    plan->k_tokens = tk;
    plan->n_seq = n_seq;
    plan->max_k_len = longest;
    plan->max_row = last_row;
    plan->n_q_heads = n_q_heads;
    plan->n_kv_heads = n_kv_heads;
    plan->pos_per_chain = ppt;
    plan->n_ctas = (int32_t)l.start.size() - 1;
    plan->n_pieces = (int32_t)l.pieces.size();
    plan->n_merges = (int32_t)l.merges.size();
    plan->n_slots = l.slots;
    plan->n_tiles = (int32_t)l.tiles.size();
    plan->off_start = kPlanHeader;
    plan->off_pieces = plan->off_start + up16((int64_t)l.start.size() * 4);
    plan->off_merges = plan->off_pieces + up16((int64_t)l.pieces.size() * sizeof(palu::pf::PfPiece));
    plan->off_tiles = plan->off_merges + up16((int64_t)l.merges.size() * sizeof(palu::pf::PfMerge));
    plan->bytes = plan->off_tiles + up16((int64_t)l.tiles.size() * sizeof(int4));
    if (!buf) return PALU_OK;
    if ((int64_t)buf_bytes < plan->bytes)
      return fail(PALU_ERR_WORKSPACE, "plan buffer of %zu bytes is smaller than the plan's %lld", buf_bytes, (long long)plan->bytes);
    char* b = static_cast<char*>(buf);
    std::fill(b, b + kPlanHeader, 0);
    std::copy(l.start.begin(), l.start.end(), reinterpret_cast<int32_t*>(b + plan->off_start));
    std::copy(l.pieces.begin(), l.pieces.end(), reinterpret_cast<palu::pf::PfPiece*>(b + plan->off_pieces));
    std::copy(l.merges.begin(), l.merges.end(), reinterpret_cast<palu::pf::PfMerge*>(b + plan->off_merges));
    std::copy(l.tiles.begin(), l.tiles.end(), reinterpret_cast<int4*>(b + plan->off_tiles));
    return PALU_OK;
  } catch (const std::exception& e) {
    return fail(PALU_ERR_INVALID, "out of host memory while planning (%s)", e.what());
  }
}

size_t palu_prefill_workspace_bytes(const palu_prefill_plan* plan, int32_t d_v) {
  return plan ? (size_t)plan->n_slots * 2 * palu::pf::kRows * (d_v + 2) * 4 : 0;
}

int palu_prefill_attn(const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok, int64_t k_head,
                      const void* v, int64_t v_tok, int64_t v_head, void* out, int32_t d_v, const palu_prefill_plan* plan,
                      void* plan_data, void* workspace, size_t workspace_bytes, float scale, palu_stream_t stream) {
  g_err.clear();
  if (!plan || !plan_data) return fail(PALU_ERR_INVALID, "prefill: plan and its device data must be set");
  if (d_v < 16 || d_v > 128 || d_v % 16 != 0) return fail(PALU_ERR_INVALID, "d_v must be a multiple of 16 in [16, 128], got %d", d_v);
  if (!(scale > 0.f) || !(scale * palu::kLog2e < INFINITY)) return fail(PALU_ERR_INVALID, "scale must be positive and finite (also times log2 e)");
  if (plan->q_tokens == 0) return PALU_OK;
  if (!q || !out || (plan->k_tokens > 0 && (!k || !v))) return fail(PALU_ERR_INVALID, "prefill: q, k, v and out must be set");
  auto aligned = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(out) || !aligned(plan_data) || !aligned(workspace))
    return fail(PALU_ERR_INVALID, "prefill: q, k, v, out, plan and workspace must be 16-byte aligned");
  const int64_t strides[6] = {q_tok, q_head, k_tok, k_head, v_tok, v_head};
  for (int64_t s : strides)
    if (s <= 0 || s % 8 != 0 || s >= (int64_t)1 << 38)
      return fail(PALU_ERR_INVALID, "prefill: token and head strides must be positive multiples of 8 elements");
  const size_t need = palu_prefill_workspace_bytes(plan, d_v);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(PALU_ERR_WORKSPACE, "prefill: workspace of %zu bytes needed, got %zu", need, workspace ? workspace_bytes : 0);
  const int rep = plan->n_q_heads / plan->n_kv_heads, ppt = plan->pos_per_chain;
  CUtensorMap mq, mk, mv;
  {
    const cuuint64_t dims[3] = {128, (cuuint64_t)plan->n_q_heads, (cuuint64_t)plan->q_tokens};
    const cuuint64_t str[2] = {(cuuint64_t)q_head * 2, (cuuint64_t)q_tok * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)rep, (cuuint32_t)ppt};
    if (int st = encode(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q, dims, str, box, "q")) return st;
  }
  if (plan->k_tokens > 0) {
    const cuuint64_t dims[3] = {128, (cuuint64_t)plan->n_kv_heads, (cuuint64_t)plan->k_tokens};
    const cuuint64_t str[2] = {(cuuint64_t)k_head * 2, (cuuint64_t)k_tok * 2};
    const cuuint32_t box[3] = {64, 1, palu::pf::kKeys};
    if (int st = encode(&mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, k, dims, str, box, "k")) return st;
    const cuuint64_t dv[3] = {(cuuint64_t)d_v, (cuuint64_t)plan->n_kv_heads, (cuuint64_t)plan->k_tokens};
    const cuuint64_t sv[2] = {(cuuint64_t)v_head * 2, (cuuint64_t)v_tok * 2};
    if (int st = encode(&mv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, v, dv, sv, box, "v")) return st;
  } else {  // no key anywhere: no tile is loaded
    mk = mv = mq;
  }
  char* data = static_cast<char*>(plan_data);
  palu::pf::PfParams p;
  p.pieces = reinterpret_cast<const palu::pf::PfPiece*>(data + plan->off_pieces);
  p.cta_start = reinterpret_cast<const int32_t*>(data + plan->off_start);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ws_o = static_cast<float*>(workspace);
  p.ws_ml = p.ws_o + (size_t)plan->n_slots * 2 * palu::pf::kRows * d_v;
  p.status = reinterpret_cast<int*>(data);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.v_tok = v_tok;
  p.v_head = v_head;
  p.n_q = plan->n_q_heads;
  p.rep = rep;
  p.ppt = ppt;
  p.dv = d_v;
  p.sl2 = scale * palu::kLog2e;
  p.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
  p.starve = g_starve_v.load(std::memory_order_relaxed);
  auto launch = [&](auto alias) -> int {
    constexpr bool A = decltype(alias)::value;
    auto kern = palu::pf::palu_prefill_tc_kernel<A>;
    const int smem = palu::pf::PfLayout<A>::TOTAL;
    static std::atomic<uint64_t> done{0};
    if (int st = allow_smem((const void*)kern, smem, done, "cudaFuncSetAttribute(prefill)")) return st;
    kern<<<plan->n_ctas, palu::pf::kPfThreads, smem, stream>>>(mq, mk, mv, p);
    return cuda_check("prefill kernel launch");
  };
  if (int st = d_v > 64 ? launch(std::true_type{}) : launch(std::false_type{})) return st;
  if (plan->n_merges > 0) {
    const auto* merges = reinterpret_cast<const palu::pf::PfMerge*>(data + plan->off_merges);
    if (plan->n_slots >= palu::pf::kDeepRecords * plan->n_merges)
      return launch_dependent("prefill merge launch", palu::pf::palu_prefill_merge_deep_kernel, dim3(plan->n_merges, 8, (d_v + 31) / 32), 256, stream, merges, p);
    return launch_dependent("prefill merge launch", palu::pf::palu_prefill_merge_kernel, dim3(plan->n_merges, 8), 256, stream, merges, p);
  }
  return PALU_OK;
}

int palu_rebuild_kv(const void* k_lat, const void* v_lat, const void* u_k, const void* u_v, const float* cos, const float* sin,
                    const palu_page_table* pages, const palu_prefill_plan* plan, const void* plan_data, void* k_out, void* v_out,
                    int32_t n_groups, int32_t r_k, int32_t r_v, int32_t max_seq, palu_stream_t stream) {
  g_err.clear();
  if (!plan || !plan_data) return fail(PALU_ERR_INVALID, "rebuild: plan and its device data must be set");
  if (n_groups <= 0 || plan->n_kv_heads % n_groups != 0)
    return fail(PALU_ERR_INVALID, "heads_per_group: %d latent heads do not divide %d KV heads", n_groups, plan->n_kv_heads);
  if (r_k < 16 || r_k > 256 || r_k % 16 != 0) return fail(PALU_ERR_INVALID, "r_k must be a multiple of 16 in [16, 256], got %d", r_k);
  if (r_v < 16 || r_v > 256 || r_v % 16 != 0) return fail(PALU_ERR_INVALID, "r_v must be a multiple of 16 in [16, 256], got %d", r_v);
  if (n_groups != plan->n_kv_heads && !u_v)
    return fail(PALU_ERR_INVALID, "grouped latents (%d groups for %d KV heads) need u_v", n_groups, plan->n_kv_heads);
  if (max_seq <= 0 || plan->max_k_len > max_seq)
    return fail(PALU_ERR_INVALID, "rebuild: max_seq %d must be positive and hold the longest sequence's %d keys", max_seq, plan->max_k_len);
  if (plan->n_tiles == 0) return PALU_OK;
  if (!k_lat || !v_lat || !u_k || !cos || !sin || !k_out || !v_out) return fail(PALU_ERR_INVALID, "rebuild: every pointer must be set");
  for (const void* x : {k_lat, v_lat, u_k, u_v, plan_data, (const void*)k_out, (const void*)v_out})
    if (reinterpret_cast<uintptr_t>(x) % 16 != 0) return fail(PALU_ERR_INVALID, "rebuild: pointers must be 16-byte aligned");
  palu::rb::Params p;
  p.page_table = nullptr;
  p.table_ld = p.blk_shift = p.n_blocks = 0;
  if (pages) {
    const int bs = pages->block_size;
    if (!pages->table || pages->n_blocks <= 0 || (bs != 16 && bs != 32 && bs != 64 && bs != 128) ||
        (int64_t)pages->table_ld * bs < max_seq)
      return fail(PALU_ERR_INVALID, "page table: blocks of 16, 32, 64 or 128 and rows that hold max_seq positions");
    p.page_table = pages->table;
    p.table_ld = pages->table_ld;
    p.n_blocks = pages->n_blocks;
    while ((1 << p.blk_shift) < bs) ++p.blk_shift;
  }
  p.k_lat = static_cast<const __nv_bfloat16*>(k_lat);
  p.v_lat = static_cast<const __nv_bfloat16*>(v_lat);
  p.u_k = static_cast<const __nv_bfloat16*>(u_k);
  p.u_v = static_cast<const __nv_bfloat16*>(u_v);
  p.cos = cos;
  p.sin = sin;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.tiles = reinterpret_cast<const int4*>(static_cast<const char*>(plan_data) + plan->off_tiles);
  p.n_kv = plan->n_kv_heads;
  p.n_groups = n_groups;
  p.group = p.n_kv / n_groups;
  p.r_k = r_k;
  p.r_v = r_v;
  p.max_seq = max_seq;
  p.status = reinterpret_cast<int*>(const_cast<void*>(plan_data));
  p.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
  p.starve = g_starve_v.load(std::memory_order_relaxed);
  p.jobs = u_v ? 2 * p.n_kv : p.n_kv;
  // runs of heads: as many as it takes to give every SM a unit (a unit reads its tokens' table rows once)
  const int sms = device_sms();
  const int runs = (int)std::min<int64_t>(p.jobs, std::max<int64_t>(1, (sms + plan->n_tiles - 1) / plan->n_tiles));
  p.per_unit = (p.jobs + runs - 1) / runs;
  p.runs = (p.jobs + p.per_unit - 1) / p.per_unit;
  if ((int64_t)plan->n_tiles * p.runs > (1 << 30)) return fail(PALU_ERR_INVALID, "rebuild: too many tiles");
  const int units = plan->n_tiles * p.runs, ctas = std::min(units, sms);
  p.waves = units / (ctas * palu::rb::kBlock);
  p.rest = (units - p.waves * ctas * palu::rb::kBlock) / ctas;
  p.rest_more = (units - p.waves * ctas * palu::rb::kBlock) % ctas;
  const int r_max = u_v ? std::max(r_k, r_v) : r_k;
  p.a_bytes = (r_max + 63) / 64 * palu::tc::kBox;
  p.u_bytes = (r_max * 256 + 1023) / 1024 * 1024;
  const int slot = p.a_bytes + p.u_bytes, outs = 8 * palu::rb::kOutBytes, room = palu::tc::kSmemBudget - palu::rb::kFixedSmem;
  p.out_bufs = room - 2 * outs >= slot ? 2 : 1;
  p.ring = std::min(palu::rb::kMaxRing, (room - p.out_bufs * outs) / slot);
  const int smem = palu::rb::kFixedSmem + p.out_bufs * outs + p.ring * slot;
  // tensor maps: latents by (row of the cache, latent head) or (page, latent head), U by rows of 128
  CUtensorMap mk, mv, muk, muv, mko, mvo;
  const int64_t items = pages ? (int64_t)pages->n_blocks * n_groups : (int64_t)(plan->max_row + 1) * n_groups;
  const int64_t seq = pages ? pages->block_size : max_seq;
  auto latents = [&](CUtensorMap* m, const void* base, int r, const char* what) -> int {
    const cuuint64_t dims[3] = {(cuuint64_t)r, (cuuint64_t)seq, (cuuint64_t)items};
    const cuuint64_t str[2] = {(cuuint64_t)r * 2, (cuuint64_t)seq * r * 2};
    const cuuint32_t box[3] = {64, pages ? (cuuint32_t)pages->block_size : (cuuint32_t)palu::rb::kTokens, 1};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, str, box, what);
  };
  auto factors = [&](CUtensorMap* m, const void* base, int r, const char* what) -> int {
    const cuuint64_t dims[2] = {128, (cuuint64_t)p.n_kv * r};
    const cuuint64_t str[1] = {256};
    const cuuint32_t box[2] = {64, (cuuint32_t)r};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, str, box, what);
  };
  if (int st = latents(&mk, k_lat, r_k, "k_lat")) return st;
  if (int st = factors(&muk, u_k, r_k, "u_k")) return st;
  auto results = [&](CUtensorMap* m, void* base, const char* what) -> int {
    const cuuint64_t dims[3] = {128, (cuuint64_t)p.n_kv, (cuuint64_t)plan->k_tokens};
    const cuuint64_t str[2] = {256, (cuuint64_t)p.n_kv * 256};
    const cuuint32_t box[3] = {64, 1, 32};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, str, box, what);
  };
  if (int st = results(&mko, k_out, "k_out")) return st;
  mv = mk;
  muv = muk;
  mvo = mko;
  if (u_v) {
    if (int st = results(&mvo, v_out, "v_out")) return st;
    if (int st = latents(&mv, v_lat, r_v, "v_lat")) return st;
    if (int st = factors(&muv, u_v, r_v, "u_v")) return st;
  }
  static std::atomic<uint64_t> done{0};
  if (int st = allow_smem((const void*)palu::rb::palu_rebuild_kv_kernel, palu::tc::kSmemBudget, done, "cudaFuncSetAttribute(rebuild)")) return st;
  palu::rb::palu_rebuild_kv_kernel<<<ctas, palu::rb::kThreads, smem, stream>>>(mk, mv, muk, muv, mko, mvo, p);
  if (int st = cuda_check("rebuild kernel launch")) return st;
  if (u_v) return PALU_OK;
  const int heads = (int)std::min<int64_t>(n_groups, std::max<int64_t>(1, 4LL * sms / plan->n_tiles));
  palu::rb::palu_gather_latents_kernel<<<dim3(plan->n_tiles, heads), palu::rb::kGatherThreads, 0, stream>>>(p);
  return cuda_check("gather kernel launch");
}

int palu_token_logprobs(const void* logits, int64_t ld, int32_t dtype, int64_t rows, int32_t vocab, const void* tokens, int32_t tokens64,
                        int32_t top, float* logprob, float* entropy, float* top_logprob, int64_t* top_id, palu_stream_t stream) {
  g_err.clear();
  if (rows < 0 || vocab <= 0) return fail(PALU_ERR_INVALID, "logprobs: rows must not be negative and vocab positive (got %lld, %d)", (long long)rows, vocab);
  if (dtype != PALU_BF16 && dtype != PALU_F32) return fail(PALU_ERR_INVALID, "logits dtype must be bf16 or f32");
  if (top < 0 || top > palu::lp::kMaxTop || top > vocab)
    return fail(PALU_ERR_INVALID, "top must be in [0, 32] and at most the vocabulary's %d, got %d", vocab, top);
  if (rows > 1 && ld < vocab) return fail(PALU_ERR_INVALID, "logits rows of %lld elements cannot hold %d", (long long)ld, vocab);
  if (rows == 0) return PALU_OK;
  if (!logits || !tokens || !logprob || !entropy || (top > 0 && (!top_logprob || !top_id)))
    return fail(PALU_ERR_INVALID, "logprobs: every pointer must be set");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == PALU_F32 ? 4 : 2) != 0) return fail(PALU_ERR_INVALID, "logits are not aligned to their type");
  const palu::lp::Params p{logits, ld, rows, vocab, top, tokens, tokens64, logprob, entropy, top_logprob, top_id};
  // CTAs a row (a cluster) while there are few rows. In a graph, us, with 1 / 2 / 4 / 8 a row (top 1): 1 x 128256 bf16 20 / 14 /
  // 11 / 10, 129 x 128256 21 / 16 / 15 / 22, 300 x 128256 28 / 24 / 30 / 43, 600 x 128256 40 / 41 / 57 / 89: worth it up to
  // about 4.3 CTAs an SM, and as long as a thread has 16 elements.
  const int slots = palu::lp::kCtas * device_sms();
  int c = 1;
  while (c < 8 && rows * c * 2 * 3 <= 13 * device_sms() && vocab >= palu::lp::kThreads * 16 * c * 2) c *= 2;
  const int smem = palu::lp::kStages * palu::lp::kStageBytes;
  auto kern = dtype == PALU_F32 ? palu::lp::palu_token_logprobs_kernel<float> : palu::lp::palu_token_logprobs_kernel<__nv_bfloat16>;
  static std::atomic<uint64_t> done[2];
  if (int st = allow_smem((const void*)kern, smem, done[dtype == PALU_F32], "cudaFuncSetAttribute(logprobs)")) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(rows, std::max(1, slots / c)) * c));
  cfg.blockDim = dim3(palu::lp::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)c, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) return cuda_check("logprobs kernel launch");
  return cuda_check("logprobs kernel launch");
}

size_t palu_page_workspace_bytes(int32_t n_blocks) { return n_blocks > 0 ? 16 + (size_t)n_blocks * 12 : 0; }

int palu_reserve_pages(const palu_page_pool* pool, const int32_t* rows, const int32_t* lens, int32_t n, palu_stream_t stream) {
  return guarded([&]() -> int {
    palu::pg::Pool p;
    if (int st = check_pool(pool, p)) return st;
    if (n > 0 && !lens) return fail(PALU_ERR_INVALID, "lens must hold n entries");
    if (int st = check_rows("rows", rows, lens, n, p)) return st;
    for (int i = 0; i < n; i += palu::pg::kMaxPairs) {
      palu::pg::RowLens a;
      a.n = std::min(palu::pg::kMaxPairs, n - i);
      std::copy(rows + i, rows + i + a.n, a.row);
      std::copy(lens + i, lens + i + a.n, a.len);
      palu::pg::palu_reserve_pages_kernel<<<1, palu::pg::kPlanThreads, 0, stream>>>(p, a);
      if (int st = cuda_check("reserve pages launch")) return st;
    }
    return PALU_OK;
  });
}

int palu_fork_pages(const palu_page_pool* pool, const palu_page_cache* caches, int32_t n_caches, const int32_t* parents,
                    const int32_t* children, const int32_t* lens, int32_t n, void* workspace, size_t workspace_bytes, palu_stream_t stream) {
  return guarded([&]() -> int {
    palu::pg::Pool p;
    if (int st = check_pool(pool, p)) return st;
    if (int st = check_caches(caches, n_caches, p.n_pages)) return st;
    if (n > 0 && (!lens || !parents)) return fail(PALU_ERR_INVALID, "parents and lens must hold n entries");
    if (int st = check_rows("children", children, lens, n, p)) return st;
    std::vector<int32_t> kids(children, children + n);
    std::sort(kids.begin(), kids.end());
    for (int i = 0; i < n; ++i) {
      if (parents[i] < 0 || parents[i] >= p.rows) return fail(PALU_ERR_INVALID, "parents: row %d is outside [0, %d)", parents[i], p.rows);
      if (std::binary_search(kids.begin(), kids.end(), parents[i]))
        return fail(PALU_ERR_INVALID, "row %d is a parent and a child of the same fork", parents[i]);
    }
    if (!workspace || workspace_bytes < palu_page_workspace_bytes(p.n_pages) || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return fail(PALU_ERR_WORKSPACE, "page workspace of %zu bytes (16-byte aligned) needed", palu_page_workspace_bytes(p.n_pages));
    const palu::pg::Moves mv{static_cast<int32_t*>(workspace), reinterpret_cast<int2*>(static_cast<char*>(workspace) + 16)};
    for (int i = 0; i < n; i += palu::pg::kMaxPairs) {
      palu::pg::ForkList a;
      a.n = std::min(palu::pg::kMaxPairs, n - i);
      int copies = 0;
      for (int x = 0; x < a.n; ++x) {
        a.parent[x] = parents[i + x];
        a.child[x] = children[i + x];
        a.len[x] = lens[i + x];
        copies += lens[i + x] % p.page_size != 0;
      }
      palu::pg::palu_fork_pages_kernel<<<1, palu::pg::kPlanThreads, 0, stream>>>(p, mv, a);
      if (int st = cuda_check("fork pages launch")) return st;
      if (copies > 0)
        if (int st = apply_moves(p, mv, nullptr, caches, n_caches, copies, stream)) return st;
    }
    return PALU_OK;
  });
}

int palu_free_pages(const palu_page_pool* pool, const int32_t* rows, int32_t n, palu_stream_t stream) {
  return guarded([&]() -> int {
    palu::pg::Pool p;
    if (int st = check_pool(pool, p)) return st;
    if (int st = check_rows("rows", rows, nullptr, n, p)) return st;
    for (int i = 0; i < n; i += palu::pg::kMaxPairs) {
      palu::pg::RowList a;
      a.n = std::min(palu::pg::kMaxPairs, n - i);
      std::copy(rows + i, rows + i + a.n, a.row);
      palu::pg::palu_free_pages_kernel<<<a.n, 256, 0, stream>>>(p, a);
      if (int st = cuda_check("free pages launch")) return st;
    }
    return PALU_OK;
  });
}

int palu_compact_pages(const palu_page_pool* pool, const palu_page_cache* caches, int32_t n_caches, void* workspace,
                       size_t workspace_bytes, palu_stream_t stream) {
  return guarded([&]() -> int {
    palu::pg::Pool p;
    if (int st = check_pool(pool, p)) return st;
    if (int st = check_caches(caches, n_caches, p.n_pages)) return st;
    if (!workspace || workspace_bytes < palu_page_workspace_bytes(p.n_pages) || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return fail(PALU_ERR_WORKSPACE, "page workspace of %zu bytes (16-byte aligned) needed", palu_page_workspace_bytes(p.n_pages));
    const palu::pg::Moves mv{static_cast<int32_t*>(workspace), reinterpret_cast<int2*>(static_cast<char*>(workspace) + 16)};
    int32_t* target = reinterpret_cast<int32_t*>(mv.list + p.n_pages);
    palu::pg::palu_compact_pages_kernel<<<1, palu::pg::kPlanThreads, 0, stream>>>(p, mv, target);
    if (int st = cuda_check("compact pages launch")) return st;
    return apply_moves(p, mv, target, caches, n_caches, p.n_pages / 2 + 1, stream);
  });
}

int palu_copy_pages(const palu_page_cache* caches, int32_t n_caches, int32_t n_blocks, const int32_t* src, const int32_t* dst, int32_t n,
                    palu_stream_t stream) {
  return guarded([&]() -> int {
    if (n_blocks <= 0) return fail(PALU_ERR_INVALID, "n_blocks must be positive, got %d", n_blocks);
    if (int st = check_caches(caches, n_caches, n_blocks)) return st;
    if (n < 0 || (n > 0 && (!src || !dst))) return fail(PALU_ERR_INVALID, "src and dst must hold n entries");
    for (int i = 0; i < n; ++i)
      if (src[i] < 0 || src[i] >= n_blocks || dst[i] < 0 || dst[i] >= n_blocks)
        return fail(PALU_ERR_INVALID, "copy %d -> %d is outside [0, %d)", src[i], dst[i], n_blocks);
    std::vector<int32_t> to(dst, dst + n);
    std::sort(to.begin(), to.end());
    for (int i = 1; i < n; ++i)
      if (to[i] == to[i - 1]) return fail(PALU_ERR_INVALID, "block %d is copied to twice", to[i]);
    for (int i = 0; i < n; ++i)
      if (src[i] != dst[i] && std::binary_search(to.begin(), to.end(), src[i]))
        return fail(PALU_ERR_INVALID, "block %d is copied from and copied to by the same call", src[i]);
    for (int i = 0; i < n; i += palu::pg::kMaxCopies) {
      palu::pg::CopyList l;
      l.n = std::min(palu::pg::kMaxCopies, n - i);
      for (int x = 0; x < l.n; ++x) l.move[x] = make_int2(src[i + x], dst[i + x]);
      for (int c = 0; c < n_caches; c += palu::pg::kMaxCaches) {
        palu::pg::Caches a;
        int64_t most;
        const int m = std::min(palu::pg::kMaxCaches, n_caches - c);
        const bool wide = fill_caches(caches + c, m, a, most);
        const dim3 grid(copy_grid(m, l.n, most), m);
        if (wide) palu::pg::palu_copy_pages_kernel<uint4><<<grid, palu::pg::kCopyThreads, 0, stream>>>(n_blocks, l, a);
        else palu::pg::palu_copy_pages_kernel<uint8_t><<<grid, palu::pg::kCopyThreads, 0, stream>>>(n_blocks, l, a);
        if (int st = cuda_check("copy pages launch")) return st;
      }
    }
    return PALU_OK;
  });
}

}  // extern "C"
