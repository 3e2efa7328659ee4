// The paged 4-bit cache: layout, row quantiser and address arithmetic shared by its kernels.
//
// A page holds `page` tokens (16, 32, 64 or 128) of every kv head; a head's part of it is a run of blocks of sixteen
// tokens, and a block lies in one piece:
//   16 x 64 bytes K codes | 16 x 64 bytes V codes | 16 bf16 K scales | 16 bf16 V scales      = 2112 bytes
// so that any run of tokens inside a page is one contiguous range: attention fetches it with one request, whatever the
// page size.  Codes are two's-complement nibbles, even channel in the low one (as hq_quant_pack at 4 bits).
//
// Row quantiser: scale = max|x| / 7 rounded UP to bf16, within [2^-17, 9344]; code = rint(x / scale), half to even, clamped
// to +-7.  A value code * scale then has at most 3 + 8 significant bits, a lowest bit of 2^-24 or more and a magnitude of 65408
// at most: it IS an fp16 number, and the tensor core's 16-bit operands hold the cache without another rounding (with an
// 11-bit scale the product is rounded: 1e-4 of a value, half of what fp16 outputs are rounded by).  The price is a step up to
// 2^-7 wider, 0.3 % on average.  Larger values and infinities saturate; a NaN takes the lowest code and does not count for
// the scale.
#pragma once
#include "hq_common.cuh"

namespace hq {
namespace paged {

constexpr int kTok = HQ_PAGED_BLOCK;                    // tokens of a block
constexpr int kBlockBytes = HQ_PAGED_BLOCK_BYTES;
constexpr int kVOff = kTok * 64, kKsOff = 2 * kTok * 64, kVsOff = kKsOff + 2 * kTok;
static_assert(kVsOff + 2 * kTok == kBlockBytes && kBlockBytes % 16 == 0, "block layout");

struct AttnParams {
  int R, T, H_Q, H_KV, G, page_shift, max_pages, max_q_len;
  uint32_t g_inv;                              // row / G == __umulhi(row, g_inv) for rows below 2^27 (G > 1)
  float sml;                                   // sm_scale * log2(e)
  int dtype;
  int num_pages, page_bytes, blocks_mask;      // bytes of a page of one head; its blocks - 1
  const void* q; int64_t q_st, q_sh;
  const uint8_t* pages;
  const int* table; int64_t table_stride;
  const int* kv_lens; const int* cu_q;
  void* out; int64_t o_st, o_sh;
  float* ws;
};

// positions that the tile kernel gives a key tile of 64 that both halves of its softmax work on, one that a half has to itself, and a
// query tile beside them, in 400 clocks: 1930, 1300 to 1500, and some 12000 for queries, first reference, masks and results.
// With nothing for the query tiles six chunks of 1 to 700 tokens took 238 us, with this 145 at that time.
constexpr int kFullCost = 5, kSplitCost = 4, kItemCost = 30;
constexpr double kTilePerKey = kFullCost / 64., kTilePerItem = kItemCost + kFullCost;

int64_t decode_workspace(const AttnParams& p);                 // bytes; hq_paged_decode.cu
int decode_launch(const AttnParams& p, cudaStream_t st);
int64_t tile_workspace(const AttnParams& p);                   // hq_paged_tile.cu
int tile_launch(const AttnParams& p, cudaStream_t st);

inline bool page_size_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128; }

#if defined(__CUDACC__)
__device__ __forceinline__ float scale_of(float amax) {
  const float s = fminf(fmaxf(__fdiv_rn(amax, 7.0f), 0x1p-17f), 9344.0f);
  return __uint_as_float((__float_as_uint(s) + 0xFFFFu) & 0xFFFF0000u);
}

// Eight lanes hold one row, sixteen channels each (all 32 lanes call).  Returns the row's scale; the lane's codes in channel order.
// The common lane multiplies by the rounded reciprocal and corrects the product once by its remainder, which leaves it on the
// IEEE quotient's side of every half-integer h (h * scale has 12 bits at most, so it and the remainder are exact: the argument
// at quant_row16 holds with fewer bits), and adds 1.5 * 2^23, which rounds to the integer, ties to even.  Lanes that hold a NaN, and
// rows whose scale is saturated, divide and clamp.
__device__ __forceinline__ float quant_row(const float (&v)[16], uint32_t (&code)[2]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) top = fmax3_abs_nan(top, v[i], v[i + 1]);
  bool rare = top != top;
  if (rare) {
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) top = fmax3_abs(top, v[i], v[i + 1]);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = scale_of(top);
  rare |= !(top <= 65408.0f);
  const float rcp = __frcp_rn(s);
  constexpr uint32_t kOnes = 0x11111111u, kTop = 0x88888888u, kMagic = 0x4B400000u;
  const float2 rcp2 = make_float2(rcp, rcp), ns2 = make_float2(-s, -s), magic2 = make_float2(12582912.f, 12582912.f);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint32_t c = kTop - kMagic * kOnes;              // + 8 per digit: no borrows between digits
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 x = make_float2(v[8 * w + i], v[8 * w + i + 1]);
      const float2 t = fmul2(x, rcp2);
      const float2 r = fadd2(ffma2(ffma2(t, ns2, x), rcp2, t), magic2);
      c += __float_as_uint(r.x) << (4 * i);
      c += __float_as_uint(r.y) << (4 * i + 4);
    }
    code[w] = c ^ kTop;
  }
  if (__builtin_expect(rare, 0)) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint32_t c = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = fminf(fmaxf(rintf(__fdiv_rn(v[8 * w + i], s)), -7.f), 7.f);      // a NaN becomes -7
        c |= ((uint32_t)__float2int_rn(q) & 15u) << (4 * i);
      }
      code[w] = c;
    }
  }
  return s;
}

// Eight codes -> eight values in the order 0 4 1 5 2 6 3 7.  Nibbles in the low mantissa bits are 1024 + 8 + code, or 1024 + 16 (8 + code)
// four bits up; the code is taken out exactly and its product with the scale is an fp16 number.
struct Unpack { uint32_t lo, hi, lo8, hi8; };
__device__ __forceinline__ uint4 values8(const Unpack& k, uint32_t w, __half2 s) {
  const uint32_t w8 = w >> 8;
  auto h2 = [](uint32_t x) { return *reinterpret_cast<const __half2*>(&x); };
  auto u32 = [](__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); };
  const __half2 c1032 = h2(0xE408E408u), c16th = h2(0x2C002C00u), c72 = h2(0xD480D480u);       // -1032, 1 / 16, -72
  return make_uint4(u32(__hmul2(__hadd2(h2(lop3_and_xor(w, k.lo, k.lo8)), c1032), s)),
                    u32(__hmul2(__hfma2(h2(lop3_and_xor(w, k.hi, k.hi8)), c16th, c72), s)),
                    u32(__hmul2(__hadd2(h2(lop3_and_xor(w8, k.lo, k.lo8)), c1032), s)),
                    u32(__hmul2(__hfma2(h2(lop3_and_xor(w8, k.hi, k.hi8)), c16th, c72), s)));
}
// the masks, kept in registers: as constants they are loaded again beside every use
__device__ __forceinline__ Unpack unpack_masks() {
  Unpack k;
  asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(k.lo));
  asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(k.hi));
  asm volatile("mov.b32 %0, 0x64086408;" : "=r"(k.lo8));
  asm volatile("mov.b32 %0, 0x64806480;" : "=r"(k.hi8));
  return k;
}

// Request r of a call: its first row of q, its rows, its cached tokens, and those before its first new one.  Starts outside q and
// lengths past the table are cut, so that no address is formed from them.
struct Request { int q0, nq, len, past; };
__device__ __forceinline__ Request request_of(const AttnParams& p, int r) {
  Request x;
  int n = 1;
  x.q0 = r;
  if (p.cu_q) {
    x.q0 = min(max(__ldg(p.cu_q + r), 0), p.T);
    n = max(min(max(__ldg(p.cu_q + r + 1), 0), p.T) - x.q0, 0);
  }
  x.nq = min(n, p.max_q_len);
  x.len = max(0, min(__ldg(p.kv_lens + r), p.max_pages << p.page_shift));
  x.past = x.len - n;
  return x;
}

// token of a row (token, head of the group)
__device__ __forceinline__ int token_of(const AttnParams& p, int row) { return p.G == 1 ? row : (int)__umulhi((uint32_t)row, p.g_inv); }

// Even cuts of `total` positions (below 2^31) over the blocks of a launch: block b has `share` of them from share * b + min(b, more)
// on, the first `more` blocks one more.
struct Cuts {
  int total, blocks, share, more;
  __device__ __forceinline__ Cuts(int t, int n) : total(t), blocks(n) { share = (int)((uint32_t)t / (uint32_t)n); more = t - share * n; }
  __device__ __forceinline__ int begin(int b) const { return share * b + min(b, more); }
  __device__ __forceinline__ int block_of(int pos) const {
    const int cut = (share + 1) * more;
    return pos < cut ? (int)((uint32_t)pos / (uint32_t)(share + 1)) : more + (int)((uint32_t)(pos - cut) / (uint32_t)share);
  }
};

// Sums of weights stop at 2^31 - 1.  Starts that rise never get there (the entry point sees to that); starts that rise and fall can hand the
// same rows to many requests, and their positions past that number are left out.
__device__ __forceinline__ int add_sat(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7FFFFFFFu); }

// The requests' weights in a row.  Up to 64 requests every warp adds them up by itself; more go through shared memory (part: threads + 1
// words, s_warp: a word per warp), a run of requests per thread.  All threads call the constructor, whole warps `seek`.
template <int kThreads, class Weight>
struct Prefix {
  const AttnParams& p;
  Weight weight;
  int total, w0, w1;                             // up to 64 requests: running sums at request `lane` and 32 + `lane`
  const int* s_part;
  int per;
  __device__ __forceinline__ static int scan(int x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x = add_sat(x, y); }
    return x;
  }
  __device__ __forceinline__ Prefix(const AttnParams& pp, Weight w, int* part, int* s_warp) : p(pp), weight(w), s_part(part) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (p.R <= 64) {
      w0 = scan(lane < p.R ? weight(request_of(p, lane)) : 0);
      total = __shfl_sync(0xffffffffu, w0, 31);
      if (p.R > 32) {
        w1 = add_sat(scan(32 + lane < p.R ? weight(request_of(p, 32 + lane)) : 0), total);
        total = __shfl_sync(0xffffffffu, w1, 31);
      }
      return;
    }
    per = (p.R + kThreads - 1) / kThreads;
    int mine = 0;
    for (int r = tid * per; r < min(p.R, (tid + 1) * per); ++r) mine = add_sat(mine, weight(request_of(p, r)));
    const int x = scan(mine);
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    const int sums = scan(lane < kThreads / 32 ? s_warp[lane] : 0), before = __shfl_sync(0xffffffffu, sums, (warp + 31) & 31);
    total = __shfl_sync(0xffffffffu, sums, 31);
    part[tid + 1] = add_sat(x, warp ? before : 0);
    if (tid == 0) part[0] = 0;
    __syncthreads();
  }
  // the request that position pos < total lies in, and the position in it
  __device__ __forceinline__ int seek(int pos, int& in) const {
    if (p.R <= 64) {
      int r = __popc(__ballot_sync(0xffffffffu, w0 <= pos));
      int below = __shfl_sync(0xffffffffu, w0, max(r - 1, 0));
      if (r == 32) {
        const int b = __popc(__ballot_sync(0xffffffffu, w1 <= pos)), y = __shfl_sync(0xffffffffu, w1, max(b - 1, 0));
        if (b) below = y;
        r += b;
      }
      in = r ? pos - below : pos;
      return r;
    }
    int lo = 0, hi = kThreads;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (s_part[mid] <= pos) lo = mid; else hi = mid; }
    in = pos - s_part[lo];
    for (int r = lo * per;; ++r) {
      const int w = weight(request_of(p, r));
      if (in < w) return r;
      in -= w;
    }
  }
};

// first byte of the sixteen-token block of `slot` (page * page_size + position in the page) of head `h`
__device__ __forceinline__ int64_t block_offset(int64_t slot, int h, int H, int page_shift) {
  const int64_t page = slot >> page_shift;
  const int blocks = 1 << (page_shift - 4), in_page = (int)(slot & ((1 << page_shift) - 1));
  return ((page * H + h) * blocks + (in_page >> 4)) * kBlockBytes;
}
#endif

}  // namespace paged
}  // namespace hq
