// Attention over the paged 4-bit cache: the entry points.  Calls whose new tokens times query heads per kv head fit 16 rows go to the
// split kernel on mma.sync (hq_paged_decode.cu), longer ones to the tile kernel on tcgen05 (hq_paged_tile.cu), whose query tiles
// have 256 rows whatever they are filled with.  Both at the rule's border and below it, split kernel and tile kernel: one request of 512
// tokens, four rows 7.2 and 16.0 us; of 32768 16.7 and 40.2; 16 of 16384, eight rows 70 and 177; 4 of 65536, sixteen rows
// 39 and 62; sixteen rows, 2 of 20000 20 and 34, 16 of 4096 22 and 26, 64 of 512 13 and 23.  The rule goes by the call's longest request: one
// that passes it takes the others along, which then cost what the second figures say.
#include "hq_paged.cuh"

namespace hq {
namespace paged {

static int shift_of(int page_size) { return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7; }

static bool few_rows(const hq_paged_attention_args* a) { return (int64_t)a->max_q_len * (a->H_Q / a->H_KV) <= 16; }

// Rows of 128 at i * si + j * sj that share nothing: one index's rows all lie within a step of the other.  (Strides below 2^56: no
// overflow in what is compared; an index of one value has no stride.)
static bool rows_apart(int64_t ni, int64_t si, int64_t nj, int64_t sj) {
  constexpr int64_t kMost = (int64_t)1 << 56;
  if (ni == 1) si = 128;
  if (nj == 1) sj = 128;
  if (si < 128 || sj < 128 || si > kMost || sj > kMost) return false;
  auto within = [](int64_t n, int64_t s, int64_t step) { return n == 1 || (step - 128) / s >= n - 1; };
  return ni == 1 || nj == 1 || within(nj, sj, si) || within(ni, si, sj);
}

static int check(const hq_paged_attention_args* a) {
  HQ_REQUIRE(a != nullptr, HQ_ERR_INVALID, "hq_paged_attention: null argument block");
  HQ_REQUIRE(a->struct_bytes == (int)sizeof(hq_paged_attention_args), HQ_ERR_INVALID, "hq_paged_attention: struct_bytes %d, expected %d",
             a->struct_bytes, (int)sizeof(hq_paged_attention_args));
  HQ_REQUIRE(a->R >= 0 && a->T >= 0 && a->H_Q >= 1 && a->H_KV >= 1 && a->max_pages >= 0 && a->num_pages >= 0 && a->max_q_len >= 1, HQ_ERR_INVALID,
             "hq_paged_attention: bad size");
  HQ_REQUIRE(a->head_dim == 128, HQ_ERR_UNSUPPORTED, "hq_paged_attention: head_dim %d is not built (128 only)", a->head_dim);
  HQ_REQUIRE(a->H_Q % a->H_KV == 0 && a->H_Q / a->H_KV <= 16, HQ_ERR_UNSUPPORTED,
             "hq_paged_attention: %d query heads over %d kv heads (a multiple of 1 to 16 is built)", a->H_Q, a->H_KV);
  HQ_REQUIRE(page_size_ok(a->page_size), HQ_ERR_UNSUPPORTED, "hq_paged_attention: page_size must be 16, 32, 64 or 128, got %d", a->page_size);
  HQ_REQUIRE((int64_t)a->max_pages * a->page_size <= 0x7FFFFF00, HQ_ERR_UNSUPPORTED, "hq_paged_attention: tables of %d pages of %d tokens",
             a->max_pages, a->page_size);
  HQ_REQUIRE(a->dtype == HQ_BF16 || a->dtype == HQ_F16, HQ_ERR_UNSUPPORTED, "hq_paged_attention: dtype %d (bf16 and fp16 are built)", a->dtype);
  HQ_REQUIRE(a->sm_scale >= 0.f && a->sm_scale < 1e30f, HQ_ERR_INVALID, "hq_paged_attention: sm_scale must be finite and not negative");
  HQ_REQUIRE(a->cu_q || (a->R == a->T && a->max_q_len == 1), HQ_ERR_INVALID, "hq_paged_attention: without cu_q every request has one token");
  HQ_REQUIRE((int64_t)a->R * a->H_KV <= 0x7FFFFFFF, HQ_ERR_UNSUPPORTED, "hq_paged_attention: %d requests of %d kv heads", a->R, a->H_KV);
  HQ_REQUIRE(a->num_pages * a->H_KV <= 0x7FFFFFFF, HQ_ERR_UNSUPPORTED, "hq_paged_attention: %lld pages of %d kv heads", (long long)a->num_pages, a->H_KV);
  HQ_REQUIRE((int64_t)a->T * (a->H_Q / a->H_KV) < (1 << 27), HQ_ERR_UNSUPPORTED, "hq_paged_attention: %d tokens of %d query heads a kv head", a->T,
             a->H_Q / a->H_KV);
  // Places in the row of all requests' keys are 32-bit numbers (at most kTilePerKey a cached token and kTilePerItem more for each query tile
  // of 256 rows, or a unit of 32 tokens and two more for each kv head): tables this long, for this many rows, are refused.
  const double items = few_rows(a) ? (double)a->R : (double)a->R + (double)a->T * (a->H_Q / a->H_KV) / 256;
  const double each = (double)a->max_pages * a->page_size * (few_rows(a) ? 1. / 32 : kTilePerKey) + (few_rows(a) ? 2 : kTilePerItem);
  HQ_REQUIRE(items * a->H_KV * each < 2147483647.0, HQ_ERR_UNSUPPORTED,
             "hq_paged_attention: %d requests, %d tokens and tables of %d pages of %d tokens are too much for one call", a->R, a->T, a->max_pages, a->page_size);
  if (a->R == 0 || a->T == 0) return HQ_OK;
  HQ_REQUIRE(a->q && a->out && a->kv_lens && (a->page_table || a->max_pages == 0) && (a->pages || a->num_pages == 0), HQ_ERR_INVALID,
             "hq_paged_attention: null pointer");
  HQ_REQUIRE(a->table_stride >= a->max_pages, HQ_ERR_INVALID, "hq_paged_attention: table rows of %d pages overlap at stride %lld", a->max_pages,
             (long long)a->table_stride);
  const int64_t strides = (a->T > 1 ? a->q_st | a->o_st : 0) | (a->H_Q > 1 ? a->q_sh | a->o_sh : 0);
  HQ_REQUIRE(aligned16(a->q) && aligned16(a->out) && aligned16(a->pages) && strides % 8 == 0, HQ_ERR_ALIGNMENT,
             "hq_paged_attention: q, out and pages must be 16-byte aligned, strides multiples of 8 elements");
  HQ_REQUIRE(((uintptr_t)a->page_table | (uintptr_t)a->kv_lens | (uintptr_t)a->cu_q) % 4 == 0, HQ_ERR_ALIGNMENT,
             "hq_paged_attention: page_table, kv_lens and cu_q must be 4-byte aligned");
  HQ_REQUIRE(rows_apart(a->T, a->o_st, a->H_Q, a->o_sh), HQ_ERR_INVALID, "hq_paged_attention: rows of out overlap at strides %lld and %lld",
             (long long)a->o_st, (long long)a->o_sh);
  return HQ_OK;
}

static AttnParams params_of(const hq_paged_attention_args* a) {
  AttnParams p{};
  p.R = a->R; p.T = a->T; p.H_Q = a->H_Q; p.H_KV = a->H_KV; p.G = a->H_Q / a->H_KV;
  p.g_inv = (uint32_t)(0x100000000ull / (uint64_t)p.G) + 1u;      // G == 1 is not looked up
  p.page_shift = shift_of(a->page_size); p.max_pages = a->max_pages; p.max_q_len = a->max_q_len;
  p.sml = a->sm_scale * 1.44269504f;
  p.num_pages = (int)a->num_pages; p.page_bytes = kBlockBytes << (p.page_shift - 4); p.blocks_mask = (1 << (p.page_shift - 4)) - 1;
  p.q = a->q; p.q_st = a->q_st; p.q_sh = a->q_sh; p.pages = (const uint8_t*)a->pages;
  p.table = a->page_table; p.table_stride = a->table_stride; p.kv_lens = a->kv_lens; p.cu_q = a->cu_q;
  p.ws = (float*)a->workspace;
  p.out = a->out; p.o_st = a->o_st; p.o_sh = a->o_sh; p.dtype = a->dtype;
  return p;
}
static int64_t workspace_of(const hq_paged_attention_args* a, const AttnParams& p) { return few_rows(a) ? decode_workspace(p) : tile_workspace(p); }

}  // namespace paged
}  // namespace hq

extern "C" int hq_paged_attention_workspace_bytes(const hq_paged_attention_args* a, int64_t* bytes) {
  using namespace hq;
  if (int rc = paged::check(a)) return rc;
  HQ_REQUIRE(bytes, HQ_ERR_INVALID, "hq_paged_attention_workspace_bytes: null pointer");
  const paged::AttnParams p = paged::params_of(a);
  *bytes = a->R > 0 && a->T > 0 ? paged::workspace_of(a, p) : 0;
  return HQ_OK;
}

extern "C" int hq_paged_attention(const hq_paged_attention_args* a, void* stream) {
  using namespace hq;
  using namespace hq::paged;
  if (int rc = check(a)) return rc;
  if (a->R == 0 || a->T == 0) return HQ_OK;
  const AttnParams p = params_of(a);
  const int64_t need = workspace_of(a, p);
  HQ_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need), HQ_ERR_WORKSPACE, "hq_paged_attention: %lld bytes of workspace, %lld needed",
             (long long)a->workspace_bytes, (long long)need);
  HQ_REQUIRE(aligned16(a->workspace), HQ_ERR_ALIGNMENT, "hq_paged_attention: the workspace must be 16-byte aligned");
  return few_rows(a) ? decode_launch(p, (cudaStream_t)stream) : tile_launch(p, (cudaStream_t)stream);
}
