// Attention over the paged 4-bit cache.
#include "hq_paged.cuh"

namespace hq {
namespace paged {

// One block per new token and kv head; 128 threads.  Keys in tiles of 32: four threads a key for the scores, then a thread per
// channel for the values.
__global__ void __launch_bounds__(128)
attn_simple_kernel(const AttnParams p) {
  __shared__ float sq[16][128], sp[16][32], smx[16], sl[16], sal[16];
  const int r = blockIdx.z, h = blockIdx.y, i = blockIdx.x, tid = threadIdx.x;
  const Request rq = request_of(p, r);
  if (i >= rq.nq) return;
  const int q0 = rq.q0, n_keys = max(0, min(rq.len, rq.past + i + 1));
  const int t = q0 + i, G = p.G;
  for (int x = tid; x < G * 128; x += 128) {
    const int64_t at = t * p.q_st + (h * G + x / 128) * p.q_sh + x % 128;
    sq[x / 128][x % 128] = (p.dtype == HQ_BF16 ? __bfloat162float(((const __nv_bfloat16*)p.q)[at]) : __half2float(((const __half*)p.q)[at])) * p.sml;
  }
  if (tid < 16) { smx[tid] = -INFINITY; sl[tid] = 0.f; }
  __syncthreads();
  float acc[16];
#pragma unroll
  for (int g = 0; g < 16; ++g) acc[g] = 0.f;
  for (int j0 = 0; j0 < n_keys; j0 += 32) {
    const int jj = tid >> 2, part = tid & 3, j = j0 + jj;
    const int page = j < n_keys ? p.table[r * p.table_stride + (j >> p.page_shift)] : -1;
    const bool live = page >= 0 && page < p.num_pages;
    float kx[32];
    if (live) {
      const int64_t slot = ((int64_t)page << p.page_shift) + (j & ((1 << p.page_shift) - 1));
      const uint8_t* b = p.pages + block_offset(slot, h, p.H_KV, p.page_shift);
      const float s = __uint_as_float((uint32_t)((const uint16_t*)(b + kKsOff))[j & 15] << 16);
      const uint4 c = *reinterpret_cast<const uint4*>(b + (j & 15) * 64 + part * 16);
      const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int x = 0; x < 32; ++x) kx[x] = (float)((int)(w[x >> 3] << (28 - 4 * (x & 7))) >> 28) * s;
    }
    for (int g = 0; g < G; ++g) {
      float d = 0.f;
      if (live)
#pragma unroll
        for (int x = 0; x < 32; ++x) d += kx[x] * sq[g][part * 32 + x];
      d += __shfl_xor_sync(0xffffffffu, d, 1);
      d += __shfl_xor_sync(0xffffffffu, d, 2);
      if (part == 0) sp[g][jj] = live ? d : -INFINITY;
    }
    __syncthreads();
    if (tid < G) {
      float m = smx[tid];
      for (int x = 0; x < 32; ++x) m = fmaxf(m, sp[tid][x]);
      const float mu = m == -INFINITY ? 0.f : m;
      const float alpha = ex2f(smx[tid] - mu);
      float l = sl[tid] * alpha;
      for (int x = 0; x < 32; ++x) { const float e = ex2f(sp[tid][x] - mu); sp[tid][x] = e; l += e; }
      sal[tid] = alpha; smx[tid] = m; sl[tid] = l;
    }
    __syncthreads();
    for (int g = 0; g < G; ++g) acc[g] *= sal[g];
    for (int x = 0; x < 32 && j0 + x < n_keys; ++x) {
      const int pg = p.table[r * p.table_stride + ((j0 + x) >> p.page_shift)];
      if (pg < 0 || pg >= p.num_pages) continue;
      const int64_t slot = ((int64_t)pg << p.page_shift) + ((j0 + x) & ((1 << p.page_shift) - 1));
      const uint8_t* b = p.pages + block_offset(slot, h, p.H_KV, p.page_shift);
      const int row = (j0 + x) & 15;
      const float s = __uint_as_float((uint32_t)((const uint16_t*)(b + kVsOff))[row] << 16);
      const int c = b[kVOff + row * 64 + (tid >> 1)];
      const float vv = (float)((int)((uint32_t)c << (tid & 1 ? 24 : 28)) >> 28) * s;
      for (int g = 0; g < G; ++g) acc[g] += sp[g][x] * vv;
    }
    __syncthreads();
  }
  for (int g = 0; g < G; ++g) {
    const float l = sl[g], o = l > 0.f ? acc[g] / l : 0.f;
    store_out(p.out, t * p.o_st + (h * G + g) * p.o_sh + tid, o, p.dtype);
  }
}

static int shift_of(int page_size) { return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7; }

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
  if (a->R == 0 || a->T == 0) return HQ_OK;
  HQ_REQUIRE(a->q && a->out && a->kv_lens && (a->page_table || a->max_pages == 0) && (a->pages || a->num_pages == 0), HQ_ERR_INVALID,
             "hq_paged_attention: null pointer");
  HQ_REQUIRE(a->table_stride >= a->max_pages, HQ_ERR_INVALID, "hq_paged_attention: table rows of %d pages overlap at stride %lld", a->max_pages,
             (long long)a->table_stride);
  HQ_REQUIRE(aligned16(a->q) && aligned16(a->out) && aligned16(a->pages) && (a->q_st | a->q_sh | a->o_st | a->o_sh) % 8 == 0, HQ_ERR_ALIGNMENT,
             "hq_paged_attention: q, out and pages must be 16-byte aligned, strides multiples of 8 elements");
  return HQ_OK;
}

static AttnParams params_of(const hq_paged_attention_args* a) {
  AttnParams p{};
  p.R = a->R; p.T = a->T; p.H_Q = a->H_Q; p.H_KV = a->H_KV; p.G = a->H_Q / a->H_KV;
  p.page_shift = shift_of(a->page_size); p.max_pages = a->max_pages; p.max_q_len = a->max_q_len;
  p.sml = a->sm_scale * 1.44269504f;
  p.num_pages = a->num_pages;
  p.q = a->q; p.q_st = a->q_st; p.q_sh = a->q_sh; p.pages = (const uint8_t*)a->pages;
  p.table = a->page_table; p.table_stride = a->table_stride; p.kv_lens = a->kv_lens; p.cu_q = a->cu_q;
  p.ws = (float*)a->workspace;
  p.out = a->out; p.o_st = a->o_st; p.o_sh = a->o_sh; p.dtype = a->dtype;
  return p;
}
static bool few_rows(const AttnParams& p) { return (int64_t)p.max_q_len * p.G <= 16; }

}  // namespace paged
}  // namespace hq

extern "C" int hq_paged_attention_workspace_bytes(const hq_paged_attention_args* a, int64_t* bytes) {
  using namespace hq;
  if (int rc = paged::check(a)) return rc;
  HQ_REQUIRE(bytes, HQ_ERR_INVALID, "hq_paged_attention_workspace_bytes: null pointer");
  const paged::AttnParams p = paged::params_of(a);
  *bytes = paged::few_rows(p) && a->R > 0 && a->T > 0 ? paged::decode_workspace(p) : 0;
  return HQ_OK;
}

extern "C" int hq_paged_attention(const hq_paged_attention_args* a, void* stream) {
  using namespace hq;
  using namespace hq::paged;
  if (int rc = check(a)) return rc;
  if (a->R == 0 || a->T == 0) return HQ_OK;
  const AttnParams p = params_of(a);
  if (few_rows(p)) {
    HQ_REQUIRE(a->workspace && a->workspace_bytes >= decode_workspace(p), HQ_ERR_WORKSPACE, "hq_paged_attention: %lld bytes of workspace, %lld needed",
               (long long)a->workspace_bytes, (long long)decode_workspace(p));
    HQ_REQUIRE(aligned16(a->workspace), HQ_ERR_ALIGNMENT, "hq_paged_attention: the workspace must be 16-byte aligned");
    return decode_launch(p, (cudaStream_t)stream);
  }
  HQ_REQUIRE(a->R <= 65535 && a->H_KV <= 65535, HQ_ERR_UNSUPPORTED, "hq_paged_attention: too many requests");
  attn_simple_kernel<<<dim3(a->max_q_len, a->H_KV, a->R), 128, 0, (cudaStream_t)stream>>>(p);
  HQ_CUDA(cudaGetLastError());
  return HQ_OK;
}
