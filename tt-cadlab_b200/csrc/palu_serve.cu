// C ABI of the operators around the decode step: the plan and attention of packed prompts. Validation, planning and
// dispatch on the host; the kernels live in the .cuh files next to it.
#include <algorithm>
#include <new>
#include <vector>

#include "../../include/palu_b200.h"
#include "abi_common.h"
#include "prefill_tc.cuh"

using namespace palu::abi;

namespace {

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

// Whole items, heaviest first, dealt to the CTAs in alternating direction. Returns the largest CTA's cost.
int64_t deal_whole(const std::vector<Item>& items, int n_kv, int ctas, Lists* out) {
  std::vector<int64_t> load(ctas, 0);
  std::vector<std::vector<palu::pf::PfPiece>> per(out ? ctas : 0);
  int64_t n = 0;
  for (const Item& it : items)
    for (int h = 0; h < n_kv; ++h, ++n) {
      const int64_t round = n / ctas, x = n % ctas;
      const int c = (int)(round & 1 ? ctas - 1 - x : x);
      load[c] += it.tiles + kPieceTiles;
      if (out) per[c].push_back({it.q0, it.npos, it.vis0, it.k0, h, 0, it.tiles, -1});
    }
  if (out) {
    out->start.assign(1, 0);
    for (auto& v : per) {
      out->pieces.insert(out->pieces.end(), v.begin(), v.end());
      out->start.push_back((int32_t)out->pieces.size());
    }
  }
  return load.empty() ? 0 : *std::max_element(load.begin(), load.end());
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
  for (int s = 0; s < n_seq; ++s) {
    const int ql = q_lens[s], kl = k_lens[s], step = 2 * ppt;
    for (int a = 0; a < ql; a += step) {
      const int n = std::min(step, ql - a), vis0 = kl - ql + a + 1, last = vis0 + n - 1;
      items.push_back({q0 + a, n, vis0, k0, last > 0 ? (last + palu::pf::kKeys - 1) / palu::pf::kKeys : 0});
    }
    for (int a = 0; a < kl; a += 64) out.tiles.push_back(make_int4(rows ? rows[s] : s, a, k0 + a, std::min(64, kl - a)));
    q0 += ql;
    k0 += kl;
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
  if (rep > palu::pf::kRows) return fail(PALU_ERR_INVALID, "at most 128 query heads per KV head are supported, got %d", rep);
  if (n_ctas < 0 || n_ctas > 4096) return fail(PALU_ERR_INVALID, "n_ctas must be in [0, 4096], got %d", n_ctas);
  int64_t tq = 0, tk = 0;
  for (int s = 0; s < n_seq; ++s) {
    if (q_lens[s] < 0 || k_lens[s] < 0)
      return fail(PALU_ERR_INVALID, "sequence %d: lengths must not be negative (got %d queries, %d keys)", s, q_lens[s], k_lens[s]);
    if (rows && rows[s] < 0) return fail(PALU_ERR_INVALID, "sequence %d: cache row %d is negative", s, rows[s]);
    tq += q_lens[s];
    tk += k_lens[s];
  }
  if (tq > (1 << 28) || tk > (1 << 28)) return fail(PALU_ERR_INVALID, "at most 2^28 packed tokens are supported");
  try {
    Lists l;
    const int ppt = palu::pf::kRows / rep;
    make_lists(q_lens, k_lens, rows, n_seq, n_kv_heads, ppt, n_ctas ? n_ctas : device_sms(), l);
    plan->q_tokens = tq;
    plan->k_tokens = tk;
    plan->n_seq = n_seq;
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
  } catch (const std::bad_alloc&) {
    return fail(PALU_ERR_INVALID, "out of host memory while planning");
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
  if (!(scale > 0.f) || !(scale < INFINITY)) return fail(PALU_ERR_INVALID, "scale must be positive and finite");
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
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return cuda_check("cudaFuncSetAttribute(prefill)");
    kern<<<plan->n_ctas, palu::pf::kPfThreads, smem, stream>>>(mq, mk, mv, p);
    return cuda_check("prefill kernel launch");
  };
  if (int st = d_v > 64 ? launch(std::true_type{}) : launch(std::false_type{})) return st;
  if (plan->n_merges > 0) {
    palu::pf::palu_prefill_merge_kernel<<<dim3(plan->n_merges, 8), 256, 0, stream>>>(
        reinterpret_cast<const palu::pf::PfMerge*>(data + plan->off_merges), p);
    return cuda_check("prefill merge launch");
  }
  return PALU_OK;
}

}  // extern "C"
