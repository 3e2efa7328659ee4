// Attention of a few new tokens per request over the paged 4-bit cache: calls whose new tokens times query heads per kv head
// fit 16 rows (one token at every group size, drafts of a few).
//
// 132 bytes a cached token and kv head, read once: 32 tokens are 4224 bytes, 95 ns of an SM's share of 6.54 TB/s.  A unit of them takes an SM
// 131 ns (16 requests of 4096 to 65536 tokens, 64 query heads over 8), and a call takes 12 us beside its units: finding the part, first copy,
// queries, the merges, the merge kernel.  16 requests of up to 32768 tokens 61 us, 3.8 TB/s; one request of 517 tokens 8.0 us, of 32768
// 16.4.  Counters of the long batch: 547 instructions a unit with all that runs once, issue slots 50 %, ALU pipe 49 % (unpacking, masks),
// warps wait for a math pipe (0.88 of every issue) and for an instruction's result (1.58) more than for data (0.29).
// Nine to sixteen rows a head double the products and exponentials, not the unpacking: 213 ns a unit and 16 us; 4 requests of up to 131072
// tokens, 2 heads, 49 us, issue slots 37 %.
// O += P V beside the next unit's scores in one stretch of code, in order or interleaved, gave nothing (61 us where the batch took 58).
//
// Work split.  A kv head of a request is a run of units of 32 tokens and one closing unit, so that heads without tokens cost
// something too; all runs in a row (requests, then heads) are cut evenly over the blocks, one per SM, and a block's part evenly over its
// warps, whatever the lengths are: they are only known on the device.  A warp walks its part alone: no barrier inside, and a run that lies within one warp's part is written out by that warp.  Runs that several warps share are
// merged through shared memory at the block's end, runs that several blocks share by the merge kernel.  Everything goes by
// position, nothing by arrival: results do not depend on timing, and no counter has to be zero beforehand.
//
// Per warp a ring of three units in shared memory, each one bulk copy (two for pages of sixteen tokens).  Products on mma.sync
// m16n8k16 in fp16: S^T = K Q^T, tokens on M and the rows (token, head of the group) on N, then O^T = V^T P^T.  Codes enter as fp16
// subnormals (one logic operation for two of them): the nibble + 8 as mantissa bits is (code + 8) 2^-24, or 2^-20 for a nibble four
// bits up.  The power of two goes into the query operand and the epilogue, the 8 into the accumulators' start (K) and a row sum
// of P (V, one more product).  The tensor core cuts what does not fit 24 bits beside its largest term off towards zero, and all terms of
// P (code + 8) are positive: summed in its accumulators over a part's length they came out 1.2e-5 v_scale too small for 16 requests of 32768
// tokens, 3e-5 for 64 of 16384, where flat attention is 0.02 of it.  So a unit's products start at zero and are added outside, rounded
// to nearest, and the row sum is formed of eights of the codes' own two kinds, which lose what they lose: the errors are those of
// P's and the output's rounding now, at every length (batch 16: 60.2 -> 61.2 us, sixteen rows 47.5 -> 49.1).  Queries are scaled by a power of two of their own so that fp16 holds them
// exactly.  P v_scale is rounded to fp16, 11 bits against bf16's 8, relative to the row's largest product so far: a row's one reference is
// the maximum of score and log2 of v_scale together, so that a key with all the weight and a small value keeps its bits beside large
// values without weight.  The row sum of P, in 32 bits, is relative to it too.
#include "hq_paged.cuh"

namespace hq {
namespace paged {

constexpr int kUnit = 32, kUnitBytes = 2 * kBlockBytes, kSlots = 3;
constexpr int kRowPad = 132;                    // floats of a row of a piece
constexpr float kShift = 9.0f;                  // P~ v_scale = 2^(s - m + 9) v_scale: at most 2^10 when a reference is set, 2^15 before it moves
constexpr float kNone = 1e30f;                  // a shift under which nothing is 0 and any key calls for a reference
constexpr float kFirst = 3.0f, kLeast = 256.0f; // the reference that a run's first unit is tried with, and the least sum of 32 P~ v_scale that lets it stay
// Warps of a block: few enough for their registers (167; more than eight rows 255, with 16 bytes spilled), and as many on every scheduler.
// The 32768 tokens, the batch and 200 short requests: 16 warps 17.3, 62.2, 29.6 us, 14 18.1, 67.2, 30.3, 12 16.4, 61.1, 25.9, 11 17.7, 66.3,
// 26.0, 8 17.8, 72.3, 28.4.  More than eight rows: 12 warps 51.9 us, 11 53.7, 10 57.1, 8 49.1.
__host__ __device__ constexpr int warps_of(int NT) { return NT == 1 ? 12 : 8; }
__host__ __device__ constexpr int piece_floats(int NT) { return 8 * NT * kRowPad + 16 * NT; }

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void add4(float (&a)[4], const float (&b)[4]) {
  const float2 x = fadd2(make_float2(a[0], a[1]), make_float2(b[0], b[1])), y = fadd2(make_float2(a[2], a[3]), make_float2(b[2], b[3]));
  a[0] = x.x; a[1] = x.y; a[2] = y.x; a[3] = y.y;
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma16816_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float2 c) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y));
}
// nibbles 0..3 of each 16-bit half as fp16 subnormals: (code + 8) 2^-24 for 0 and 2, 2^-20 for 1 and 3.  The masks stay in registers:
// as constants they are loaded again beside every use.
struct Masks { uint32_t lo, hi, lo8, hi8; };
__device__ __forceinline__ Masks masks() {
  Masks k;
  asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(k.lo));
  asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(k.hi));
  asm volatile("mov.b32 %0, 0x00080008;" : "=r"(k.lo8));
  asm volatile("mov.b32 %0, 0x00800080;" : "=r"(k.hi8));
  return k;
}
__device__ __forceinline__ void nibbles(const Masks& k, uint32_t w, uint32_t (&h)[4]) {
  const uint32_t w8 = w >> 8;
  h[0] = lop3_and_xor(w, k.lo, k.lo8);
  h[1] = lop3_and_xor(w, k.hi, k.hi8);
  h[2] = lop3_and_xor(w8, k.lo, k.lo8);
  h[3] = lop3_and_xor(w8, k.hi, k.hi8);
}
__device__ __forceinline__ float over_g(float v, bool max) {      // over the eight lanes with the same lane % 4
#pragma unroll
  for (int o = 4; o <= 16; o <<= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, v, o);
    v = max ? fmaxf(v, x) : v + x;
  }
  return v;
}
__device__ __forceinline__ float bf16_bits(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// A place in the row of runs; u == units is the closing unit.
struct Walk { int r, h, u, units; };
__device__ __forceinline__ int units_of(const Request& x) { return x.nq > 0 ? (x.len + kUnit - 1) / kUnit : -1; }     // -1: no run at all
// true where the next run is another request's
__device__ __forceinline__ bool next_run(const AttnParams& p, Walk& w) {
  w.u = 0;
  if (++w.h < p.H_KV) return false;
  w.h = 0;
  do {
    if (++w.r >= p.R) break;
    w.units = units_of(request_of(p, w.r));
  } while (w.units < 0);
  return true;
}

// Workspace: pieces of runs that begin before a warp's part and end in it; two pieces per block; what the merge kernel has to
// do for each block.
struct Merge { int q0, nq, h, first, go, unused[3]; };
template <int NT> __host__ __device__ inline int64_t ws_block_pieces(int blocks) { return (int64_t)blocks * warps_of(NT) * piece_floats(NT); }
template <int NT> __host__ __device__ inline int64_t ws_merge(int blocks) { return ws_block_pieces<NT>(blocks) + (int64_t)blocks * 2 * piece_floats(NT); }

template <bool kBf16>
__device__ __forceinline__ void store_row4(const AttnParams& p, int64_t at, float4 v, float inv) {
  v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
  uint2 o;
  if (kBf16) {
    __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    o = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  } else {
    __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    o = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  }
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) = o;
}
__device__ __forceinline__ int64_t out_row(const AttnParams& p, const Request& q, int h, int n) {
  const int i = token_of(p, n);
  return (int64_t)(q.q0 + i) * p.o_st + (int64_t)(h * p.G + n - i * p.G) * p.o_sh;
}

// a block has at least one position for every warp: fewer blocks take part in short calls
__device__ __forceinline__ int blocks_of(int total, int warps) { return max(1, min((int)gridDim.x, total / warps)); }
template <int NT>
__device__ __forceinline__ Merge* todo_of(const AttnParams& p) { return reinterpret_cast<Merge*>(p.ws + ws_merge<NT>(gridDim.x)) + blockIdx.x; }

template <int NT, bool kBf16>
__global__ void __launch_bounds__(warps_of(NT) * 32, 1)
decode_kernel(const AttnParams p, bool whole) {
  constexpr int kWarps = warps_of(NT), kThreads = kWarps * 32;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_before;                                   // units of the block's first run that lie before it
  __shared__ uint64_t bars[kWarps * kSlots];
  __shared__ int s_live[kWarps * kSlots];                    // which of a unit's two blocks lie in the pool
  __shared__ int2 s_page[kWarps][32];                        // pages of a unit's blocks, 32 units ahead
  __shared__ int s_cut[2];                             // where the block's part begins, all positions
  __shared__ int s_part[kThreads + 1], s_warp[kWarps];
  __shared__ int s_seg[32];                                  // run (r * H_KV + h) of a warp's first and last piece, or -1
  __shared__ int4 s_run[32];                                 // its first row of q, rows, head
  __shared__ float s_max[8 * NT][32], s_sum[8 * NT][32];     // (log2) maximum and sum of a piece's rows
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
  if (tid < kWarps * kSlots) { mbar_init(bars + tid, 1); fence_mbar_init(); }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- where this warp's part lies
  const int block = blockIdx.x;
  Walk c{0, 0, 0, -1};
  int left = 0;
  auto weight = [&](const Request& q) { return p.H_KV * (units_of(q) + 1); };
  if (whole) {                                               // one run a block
    __syncthreads();
    c.r = block / p.H_KV; c.h = block - c.r * p.H_KV;
    c.units = units_of(request_of(p, c.r));
    if (c.units < 0) return;
    const int n = c.units + 1;
    c.u = n * warp / kWarps;
    left = n * (warp + 1) / kWarps - c.u;
  } else {
    const Prefix<kThreads, decltype(weight)> prefix(p, weight, s_part, s_warp);
    if (p.R <= 64) __syncthreads();
    const Cuts cuts(prefix.total, blocks_of(prefix.total, kWarps));
    if (block >= cuts.blocks) { if (tid == 0) todo_of<NT>(p)->go = 0; return; }
    const int b0 = cuts.begin(block), n = cuts.begin(block + 1) - b0, each = n / kWarps, rest = n - each * kWarps;
    if (tid == 0) { s_cut[0] = b0; s_cut[1] = prefix.total; }
    left = each + (warp < rest ? 1 : 0);
    if (left > 0) {
      int in;
      c.r = prefix.seek(b0 + each * warp + min(warp, rest), in);
      c.units = units_of(request_of(p, c.r));
      c.h = (int)((uint32_t)in / (uint32_t)(c.units + 1));
      c.u = in - c.h * (c.units + 1);
    }
  }
  const int start_u = c.u;                                   // the part begins inside a run if start_u > 0

  if (warp == 0 && lane == 0) s_before = start_u;

  // ---- the ring
  uint8_t* ring = smem + warp * (kSlots * kUnitBytes);
  uint64_t* bar = bars + warp * kSlots;
  int slot = 0, ahead = 0;                                   // the slot that is read next; units under way
  uint32_t parity = 0;
  Walk f = c;                                                // the unit that is fetched next
  int f_left = left, tab_r = -1, tab_u = 0;                  // pages of the units tab_u .. + 31 of request tab_r are at hand
  bool lost = false;                                         // a copy never came: from there on the part's rows are NaN
  auto fetch = [&]() {                                       // asks for the next unit, if there is one; all lanes
    while (f_left > 0 && f.u >= f.units) { if (--f_left > 0) next_run(p, f); }
    if (f_left <= 0) return;
    if (f.r != tab_r || f.u - tab_u >= 32 || f.u < tab_u) {
      tab_r = f.r; tab_u = f.u;
      const int64_t tok = ((int64_t)tab_u + lane) * kUnit;
      const int* row = p.table + (int64_t)f.r * p.table_stride;
      const int len = request_of(p, f.r).len;
      __syncwarp();
      s_page[warp][lane] = make_int2(tok < len ? __ldg(row + (tok >> p.page_shift)) : -1, tok + kTok < len ? __ldg(row + ((tok + kTok) >> p.page_shift)) : -1);
      __syncwarp();
    }
    if (lane == 0) {
      const int at = slot + ahead >= kSlots ? slot + ahead - kSlots : slot + ahead;
      const int2 pg = s_page[warp][f.u - tab_u];
      const bool la = (uint32_t)pg.x < (uint32_t)p.num_pages, lb = (uint32_t)pg.y < (uint32_t)p.num_pages;
      s_live[warp * kSlots + at] = (la ? 1 : 0) | (lb ? 2 : 0);
      uint8_t* dst = ring + at * kUnitBytes;
      const uint8_t* src = p.pages + (int64_t)(pg.x * p.H_KV + f.h) * p.page_bytes + ((f.u << 1) & p.blocks_mask) * kBlockBytes;
      mbar_expect_tx(bar + at, ((la ? 1 : 0) + (lb ? 1 : 0)) * kBlockBytes);
      if (la && lb && p.page_shift > 4) bulk_g2s(dst, src, kUnitBytes, bar + at);
      else {
        if (la) bulk_g2s(dst, src, kBlockBytes, bar + at);
        if (lb) bulk_g2s(dst + kBlockBytes, p.page_shift > 4 ? src + kBlockBytes : p.pages + (int64_t)(pg.y * p.H_KV + f.h) * p.page_bytes, kBlockBytes,
                         bar + at);
      }
    }
    ++f.u; --f_left;
  };

  // ---- the state of the run in hand
  uint32_t qf[NT][16];                                       // query operand: word w, nibble k at 4 w + k
  uint4 raw[4];                                              // a tile's rows as they lie: channels 32 t4 .. + 31
  float2 fac[NT], start[NT];                                 // factor of a score, start of the accumulators: columns 2 t4, 2 t4 + 1
  float2 l[NT], shift[NT];                                   // P = 2^(score + shift); kNone: no key so far
  const Masks km = masks();
  float O[NT][8][4], Ls[NT][4];
  int lim0 = 0;                                              // keys that the run's first token sees
  auto ask_q = [&](const Request& q, int nt) {
    const int n = 8 * nt + g, i = token_of(p, n);
    const uint4* at = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + (int64_t)(q.q0 + i) * p.q_st +
                                                     (int64_t)(c.h * p.G + n - i * p.G) * p.q_sh + 32 * t4);
#pragma unroll
    for (int w = 0; w < 4; ++w) raw[w] = n < q.nq * p.G ? at[w] : make_uint4(0u, 0u, 0u, 0u);      // (not __ldg: out may be q)
    lim0 = q.past + 1;
  };
  auto open = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt > 0) ask_q(request_of(p, c.r), nt);
      uint32_t top2 = 0u;                                    // magnitudes of 16-bit numbers order like integers
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint4 u = raw[w];
        top2 = __vmaxu2(__vmaxu2(__vmaxu2(top2, u.x & 0x7FFF7FFFu), u.y & 0x7FFF7FFFu), __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
      }
      top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, 1));
      top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, 2));
      auto value = [&](uint32_t u, int hi) {
        if (kBf16) return __uint_as_float(hi ? u & 0xFFFF0000u : u << 16);
        return __half2float(__ushort_as_half((unsigned short)(hi ? u >> 16 : u & 0xFFFFu)));
      };
      // the largest magnitude to [2^13, 2^14): below it fp16 has 37 bits
      const int ex = (int)(__float_as_uint(value(max(top2 & 0xFFFFu, top2 >> 16), 0)) >> 23);      // 0: zero or below the normal numbers, 255: infinite
      const int up = ex == 255 ? 0 : 140 - max(ex, 14);      // at most 2^126, a normal number
      const float scale = __uint_as_float((uint32_t)(127 + up) << 23), scale16 = scale * 0.0625f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t u[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {                        // channels k and k + 4 of the eight
          const float2 x = fmul2(make_float2(value(u[k >> 1], k & 1), value(u[2 + (k >> 1)], k & 1)),
                                 k & 1 ? make_float2(scale16, scale16) : make_float2(scale, scale));
          const __half2 hh = __floats2half2_rn(x.x, x.y);
          qf[nt][4 * w + k] = *reinterpret_cast<const uint32_t*>(&hh);
        }
      }
      // what codes of zero give: the 8 that is in every nibble, to be taken off
      float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 8; ++w) mma16816(zero, km.lo8, km.lo8, km.hi8, km.hi8, qf[nt][2 * w], qf[nt][2 * w + 1]);
      start[nt] = make_float2(-zero[0], -zero[1]);
      shift[nt] = make_float2(kShift - kFirst, kShift - kFirst);
      // sml 2^24 / scale.  Where that is no number (queries from 2^117 on) the largest one serves: scores are 2^60 apart then, or equal.
      const float back = fminf(p.sml * __uint_as_float((uint32_t)min(127 + 24 - up, 254) << 23), 0x1.fffffep127f);
      fac[nt] = make_float2(__shfl_sync(0xffffffffu, back, 8 * t4), __shfl_sync(0xffffffffu, back, 8 * t4 + 4));
    }
  };
  // The run's rows so far: the 8 of the codes taken off, their powers of two put back.  To the output (piece == nullptr) or as a piece.
  auto finish = [&](float* piece, int at_piece, const Request& q) {
    const int rows = q.nq * p.G;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float ls[2] = {over_g(l[nt].x, false), over_g(l[nt].y, false)};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = 8 * nt + 2 * t4 + j;
        const float f = piece ? 1.f : ls[j] == 0.f ? 0.f : 1.f / ls[j], f24 = f * 0x1p24f, f20 = f * 0x1p20f, eight = -Ls[nt][j] * f24, eight20 = -Ls[nt][2 + j] * f20;
        float v[16];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          v[4 * q4] = fmaf(O[nt][2 * q4][j], f24, eight); v[4 * q4 + 1] = fmaf(O[nt][2 * q4 + 1][j], f20, eight20);
          v[4 * q4 + 2] = fmaf(O[nt][2 * q4][2 + j], f24, eight); v[4 * q4 + 3] = fmaf(O[nt][2 * q4 + 1][2 + j], f20, eight20);
        }
        if (n >= rows) continue;
        if (piece) {
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<float4*>(piece + n * kRowPad + 16 * g + 4 * q4) = make_float4(v[4 * q4], v[4 * q4 + 1], v[4 * q4 + 2], v[4 * q4 + 3]);
          if (g == 0) { s_max[n][at_piece] = -(j ? shift[nt].y : shift[nt].x); s_sum[n][at_piece] = ls[j]; }
        } else {
          uint32_t w[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (kBf16) { const __nv_bfloat162 hh = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]); w[k] = *reinterpret_cast<const uint32_t*>(&hh); }
            else { const __half2 hh = __floats2half2_rn(v[2 * k], v[2 * k + 1]); w[k] = *reinterpret_cast<const uint32_t*>(&hh); }
          }
          uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + out_row(p, q, c.h, n) + 16 * g);
          to[0] = make_uint4(w[0], w[1], w[2], w[3]);
          to[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
      }
    }
  };

  const int tau = (g >> 1) + 4 * (g & 1);                    // token of score row g (and + 8): the four tokens of a V fragment's
                                                             // load are neighbours then, on both halves of the banks
  auto unit = [&](bool fresh) {                              // fresh: the run's first one here
    const bool late = lost || !mbar_wait_bounded(bar + slot, parity);
    const uint8_t* u0 = ring + slot * kUnitBytes;
    const int there = s_live[warp * kSlots + slot];
    float S[NT][2][4];
    float ks[2][2], vs[2][2];
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      const uint8_t* b = u0 + cb * kBlockBytes;
      const uint4 ka = *reinterpret_cast<const uint4*>(b + tau * 64 + 16 * t4), kb = *reinterpret_cast<const uint4*>(b + (tau + 8) * 64 + 16 * t4);
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t ha[4], hb[4];
        nibbles(km, wa[w], ha);
        nibbles(km, wb[w], hb);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (w == 0) mma16816_from(S[nt][cb], ha[0], hb[0], ha[1], hb[1], qf[nt][0], qf[nt][1], start[nt]);
          else mma16816(S[nt][cb], ha[0], hb[0], ha[1], hb[1], qf[nt][4 * w], qf[nt][4 * w + 1]);
          mma16816(S[nt][cb], ha[2], hb[2], ha[3], hb[3], qf[nt][4 * w + 2], qf[nt][4 * w + 3]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[cb][i] = bf16_bits(*reinterpret_cast<const uint16_t*>(b + kKsOff + 2 * (tau + 8 * i)));
        vs[cb][i] = bf16_bits(*reinterpret_cast<const uint16_t*>(b + kVsOff + 2 * (tau + 8 * i)));
      }
    }
    // scores in powers of two
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float2 y = fmul2(make_float2(S[nt][cb][2 * i], S[nt][cb][2 * i + 1]), make_float2(ks[cb][i], ks[cb][i]));
          y = fmul2(y, fac[nt]);
          S[nt][cb][2 * i] = y.x; S[nt][cb][2 * i + 1] = y.y;
        }
    const int tok0 = c.u * kUnit;
    if (__builtin_expect(tok0 + kUnit > lim0 || there != 3, 0)) {        // keys behind a row's last one, pages that are not there
      const Request q = request_of(p, c.r);
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int tok = tok0 + 16 * cb + tau + 8 * i;
          const bool here = (there >> cb) & 1;
          if (!here || tok >= q.len) vs[cb][i] = 0.f;                    // what lies there may be anything, NaN too
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (!here || tok >= lim0 + min(token_of(p, 8 * nt + 2 * t4 + j), q.nq - 1)) S[nt][cb][2 * i + j] = -INFINITY;
        }
    }
    // P v_scale against the rows' references as they stand.  Nothing is compared beforehand: a term that fp16 could not hold shows
    // in the sum of the terms.  Only then the maxima are taken, the references move and the unit's P is formed again.  A run's first unit is
    // tried with a reference of kFirst, which fits if every row's sum comes out large enough for fp16's lower end, too.
    uint32_t P[NT][2][2];
    float2 le[NT];
    auto form = [&](bool first) {                            // true where the references do not fit
      float most = 0.f;
      bool fits = true;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        le[nt] = make_float2(0.f, 0.f);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 y = fadd2(make_float2(S[nt][cb][2 * i], S[nt][cb][2 * i + 1]), shift[nt]);
            const float2 e = make_float2(ex2f(y.x), ex2f(y.y));
            le[nt] = fadd2(le[nt], e);
            const float2 pv = fmul2(e, make_float2(vs[cb][i], vs[cb][i]));
            sum = fadd2(sum, pv);
            const __half2 hh = __floats2half2_rn(pv.x, pv.y);
            P[nt][cb][i] = *reinterpret_cast<const uint32_t*>(&hh);
          }
        most += sum.x + sum.y;
        if (first) {
          const int n = 8 * nt + 2 * t4, rows = request_of(p, c.r).nq * p.G;
          const float x0 = over_g(sum.x, false), x1 = over_g(sum.y, false);
          fits = fits && (x0 >= kLeast || n >= rows) && (x1 >= kLeast || n + 1 >= rows);
        }
      }
      return !(most <= 32768.f) || !fits;
    };
    if (__builtin_expect(__any_sync(0xffffffffu, form(fresh) || late), 0)) {
      if (!lost && __any_sync(0xffffffffu, late)) {
        // Barriers of slots that are asked for again would be a phase behind: nothing more is fetched or waited for, only what is
        // under way, once more, since its places are used for other things later.
        lost = true;
        f_left = 0;
        for (int i = 0; i < ahead; ++i)
          mbar_wait_bounded(bar + (slot + i >= kSlots ? slot + i - kSlots : slot + i), slot + i >= kSlots ? parity ^ 1u : parity, 1u << 16);
      }
      float ve[2][2];                                        // exponents of the V scales; a row that was never written (0) counts like the least scale
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int i = 0; i < 2; ++i) ve[cb][i] = (float)((int)max(__float_as_uint(vs[cb][i]) >> 23, 127u - 17u) - 127);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        auto top = [&](int j) {
          return over_g(fmaxf(fmaxf(S[nt][0][j] + ve[0][0], S[nt][0][2 + j] + ve[0][1]), fmaxf(S[nt][1][j] + ve[1][0], S[nt][1][2 + j] + ve[1][1])), true);
        };
        // the reference rises to the maximum, or falls to it if there was none; P so far is of 2^(new - old)
        const float2 old = fresh ? make_float2(kNone, kNone) : shift[nt];
        const float2 ns = make_float2(fminf(old.x, kShift - top(0)), fminf(old.y, kShift - top(1)));
        const float2 al = make_float2(old.x == kNone ? 0.f : ex2f(ns.x - old.x), old.y == kNone ? 0.f : ex2f(ns.y - old.y));
        l[nt] = fmul2(l[nt], al);
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) { O[nt][mt][0] *= al.x; O[nt][mt][1] *= al.y; O[nt][mt][2] *= al.x; O[nt][mt][3] *= al.y; }
        Ls[nt][0] *= al.x; Ls[nt][1] *= al.y; Ls[nt][2] *= al.x; Ls[nt][3] *= al.y;
        shift[nt] = ns;
      }
      form(false);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt] = fadd2(l[nt], le[nt]);
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) { P[nt][cb][0] = movmatrix(P[nt][cb][0]); P[nt][cb][1] = movmatrix(P[nt][cb][1]); }
    }
    if (lost) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) l[nt] = make_float2(__int_as_float(0x7FC00000), __int_as_float(0x7FC00000));
    }
    uint2 vw[2][4];
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
      for (int i = 0; i < 4; ++i) vw[cb][i] = *reinterpret_cast<const uint2*>(u0 + cb * kBlockBytes + kVOff + 8 * g + (t4 + 4 * i) * 64);
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {                         // channels 16 g + 4 q4 .. + 3: a 16-bit half of each token's word
      const uint32_t sel = q4 & 1 ? 0x7632u : 0x5410u;
      float d[NT][2][4];                                     // the unit's own products
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) {
        uint32_t ha[4], hb[4];
        nibbles(km, prmt(q4 < 2 ? vw[cb][0].x : vw[cb][0].y, q4 < 2 ? vw[cb][1].x : vw[cb][1].y, sel), ha);
        nibbles(km, prmt(q4 < 2 ? vw[cb][2].x : vw[cb][2].y, q4 < 2 ? vw[cb][3].x : vw[cb][3].y, sel), hb);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (cb == 0) {
            mma16816_from(d[nt][0], ha[0], ha[2], hb[0], hb[2], P[nt][0][0], P[nt][0][1], make_float2(0.f, 0.f));
            mma16816_from(d[nt][1], ha[1], ha[3], hb[1], hb[3], P[nt][0][0], P[nt][0][1], make_float2(0.f, 0.f));
          } else {
            mma16816(d[nt][0], ha[0], ha[2], hb[0], hb[2], P[nt][1][0], P[nt][1][1]);
            mma16816(d[nt][1], ha[1], ha[3], hb[1], hb[3], P[nt][1][0], P[nt][1][1]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) add4(O[nt][2 * q4 + k], d[nt][k]);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {                        // 8 P in the units of nibbles 0 and 2 (the first two sums), of 1 and 3
      float d[4];
      mma16816_from(d, km.lo8, km.hi8, km.lo8, km.hi8, P[nt][0][0], P[nt][0][1], make_float2(0.f, 0.f));
      mma16816(d, km.lo8, km.hi8, km.lo8, km.hi8, P[nt][1][0], P[nt][1][1]);
      add4(Ls[nt], d);
    }
    __syncwarp();
    if (++slot == kSlots) { slot = 0; parity ^= 1u; }
  };

  if (tid < 32) s_seg[tid] = -1;
  __syncthreads();
  bool inside = start_u > 0;                                 // the run in hand began before this part
  // the first unit is asked for before anything else, the others of the ring behind the queries: a copy takes the SM's copy engine some
  // 25 ns, 12 warps' rings 0.9 us
  if (left > 0) { ask_q(request_of(p, c.r), 0); fetch(); ++ahead; }
#pragma unroll 1
  while (left > 0) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      shift[nt] = make_float2(kNone, kNone);
      l[nt] = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) Ls[nt][i] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) O[nt][mt][i] = 0.f;
    }
    const int n = min(c.units - c.u, left);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      if (i == 0) open();
#pragma unroll 1
      for (; ahead < kSlots; ++ahead) fetch();               // the slot that has just been read
      unit(i == 0);
      --ahead;
      ++c.u;
    }
    left -= n;
    const bool ends = left > 0;                              // else it goes on in the next part
    float* mine = reinterpret_cast<float*>(ring);            // empty when it is the part's last
    float* piece = !ends ? mine : !inside ? nullptr : whole ? mine : p.ws + (int64_t)(block * kWarps + warp) * piece_floats(NT);
    const Request q = request_of(p, c.r);
    const int at = 2 * warp + (ends ? 0 : 1);
    finish(piece, at, q);
    if (piece && lane == 0) {
      s_seg[at] = c.r * p.H_KV + c.h;
      s_run[at] = make_int4(q.q0, q.nq, c.h, 0);
    }
    if (ends && --left > 0) { inside = false; next_run(p, c); ask_q(request_of(p, c.r), 0); }
  }

  // ---- runs that several warps share: pieces in order are the warps' first and last ones, a lane each; neighbours of the same
  // run are a group.  A warp takes half a row of a group at a time.
  __syncthreads();
  const int seg = s_seg[lane];
  const uint32_t valid = __ballot_sync(0xffffffffu, seg >= 0), below = valid & ((1u << lane) - 1u);
  const int prev = __shfl_sync(0xffffffffu, seg, below ? 31 - __clz(below) : 0);
  const uint32_t heads = __ballot_sync(0xffffffffu, seg >= 0 && (below == 0u || prev != seg));
  const bool first_before = !whole && s_before > 0;          // the first group's run began in another block
  float* to = whole ? nullptr : p.ws + ws_block_pieces<NT>(gridDim.x) + (int64_t)(2 * block) * piece_floats(NT);
  Merge todo{0, 0, 0, 0, 0, {0, 0, 0}};
  int turn = warp;                                           // items are dealt out over all groups
#pragma unroll 1
  for (uint32_t rest = heads; rest; rest &= rest - 1) {
    const int head = __ffs(rest) - 1;
    const uint32_t later = rest & (rest - 1);
    const uint32_t group = valid & ~((1u << head) - 1u) & (later ? (later & (0u - later)) - 1u : 0xffffffffu);
    const int4 run = s_run[head];
    const int items = 2 * run.y * p.G;
    const bool began_before = first_before && rest == heads, ends = ((31 - __clz(group)) & 1) == 0, in = (group >> lane) & 1u;
    if (began_before && ends) todo = Merge{run.x, run.y, run.z, 0, 1, {0, 0, 0}};
#pragma unroll 1
    for (; turn < items; turn += kWarps) {
      const int n = turn >> 1, ch = 64 * (turn & 1) + 2 * lane;
      const float mi = in ? s_max[n][lane] : -INFINITY;
      const int mb = __float_as_int(mi), top = __reduce_max_sync(0xffffffffu, mb >= 0 ? mb : mb ^ 0x7FFFFFFF);
      const float M = __int_as_float(top >= 0 ? top : top ^ 0x7FFFFFFF), w = ex2f(mi - M);
      float L = in ? w * s_sum[n][lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
      float2 acc = make_float2(0.f, 0.f);
      uint32_t x = group;
#pragma unroll 1
      while (x) {                                            // four pieces' loads at a time
        float2 v[4];
        float wi[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = x ? __ffs(x) - 1 : head;
          const float* piece = (j & 1) || whole ? reinterpret_cast<const float*>(smem + (j >> 1) * (kSlots * kUnitBytes))
                                                : p.ws + (int64_t)(block * kWarps + (j >> 1)) * piece_floats(NT);
          wi[k] = __shfl_sync(0xffffffffu, w, j);
          if (!x) wi[k] = 0.f;
          v[k] = *reinterpret_cast<const float2*>(piece + n * kRowPad + ch);
          x &= x - 1;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) { acc.x = fmaf(wi[k], v[k].x, acc.x); acc.y = fmaf(wi[k], v[k].y, acc.y); }
      }
      if (!began_before && ends) {
        const float inv = L == 0.f ? 0.f : 1.f / L;          // a row that saw no key: 0
        uint32_t o;
        if (kBf16) { const __nv_bfloat162 hh = __floats2bfloat162_rn(acc.x * inv, acc.y * inv); o = *reinterpret_cast<const uint32_t*>(&hh); }
        else { const __half2 hh = __floats2half2_rn(acc.x * inv, acc.y * inv); o = *reinterpret_cast<const uint32_t*>(&hh); }
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p.out) + out_row(p, Request{run.x, run.y, 0, 0}, run.z, n) + ch) = o;
      } else {
        float* mine = to + (began_before ? 0 : piece_floats(NT));
        *reinterpret_cast<float2*>(mine + n * kRowPad + ch) = acc;
        if (lane == 0) { mine[8 * NT * kRowPad + n] = M; mine[8 * NT * kRowPad + 8 * NT + n] = L; }      // (both halves write the same)
      }
    }
    turn -= items;
  }
  if (!whole && tid == kThreads - 1) {
    if (todo.go) todo.first = Cuts(s_cut[1], blocks_of(s_cut[1], kWarps)).block_of(s_cut[0] - s_before);
    *todo_of<NT>(p) = todo;
  }
}

// Runs that several blocks share.  Block (b, n) merges row n of the run that ends in block b of the decode kernel: eight warps take
// its pieces in turn, then each other's sums.
template <int NT>
__global__ void __launch_bounds__(256)
merge_kernel(const AttnParams p, int grid) {
  __shared__ float s_m[8], s_l[8], s_acc[8][128];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.x, n = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Merge todo = reinterpret_cast<const Merge*>(p.ws + ws_merge<NT>(grid))[b];
  if (!todo.go || n >= todo.nq * p.G) return;
  const float* base = p.ws + ws_block_pieces<NT>(grid);
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = todo.first + warp; i <= b; i += 8) {
    const float* x = base + (int64_t)(2 * i + (i == todo.first ? 1 : 0)) * piece_floats(NT);
    const float m = x[8 * NT * kRowPad + n], l = x[8 * NT * kRowPad + 8 * NT + n];
    const float4 v = *reinterpret_cast<const float4*>(x + n * kRowPad + 4 * lane);
    const float nm = fmaxf(M, m), ref = nm == -INFINITY ? 0.f : nm, wo = ex2f(M - ref), w = ex2f(m - ref);
    L = L * wo + l * w;
    acc.x = acc.x * wo + v.x * w; acc.y = acc.y * wo + v.y * w; acc.z = acc.z * wo + v.z * w; acc.w = acc.w * wo + v.w * w;
    M = nm;
  }
  if (lane == 0) { s_m[warp] = M; s_l[warp] = L; }
  *reinterpret_cast<float4*>(&s_acc[warp][4 * lane]) = acc;
  __syncthreads();
  if (warp) return;
  M = s_m[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) M = fmaxf(M, s_m[i]);
  const float ref = M == -INFINITY ? 0.f : M;
  L = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w = ex2f(s_m[i] - ref);
    const float4 v = *reinterpret_cast<const float4*>(&s_acc[i][4 * lane]);
    L += w * s_l[i];
    acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
  }
  const int64_t at = out_row(p, Request{todo.q0, todo.nq, 0, 0}, todo.h, n) + 4 * lane;
  const float inv = L == 0.f ? 0.f : 1.f / L;                // a row that saw no key: 0
  if (p.dtype == HQ_BF16) store_row4<true>(p, at, acc, inv);
  else store_row4<false>(p, at, acc, inv);
}

static int tiles_of(const AttnParams& p) { return p.max_q_len * p.G <= 8 ? 1 : 2; }

// Short tables and no more runs than SMs: a block per run, nothing to merge across blocks, one launch and no workspace.  Against the cut
// over all SMs: one request of 8 heads, 512 tokens 7.2 us and 10.1, 1024 9.5 and 9.5, 2048 13.4 and 9.8; eight requests 7.6 and
// 10.4, 10.4 and 11.3, 14.5 and 13.4; four of 2 heads with sixteen rows 11.5 and 15.1, 14.9 and 15.1, 21.6 and 15.1.  The rule asks the
// table's width, since lengths are only known on the device: a wide table takes the cut whatever is in it.
static bool block_per_run(const AttnParams& p) {
  return ((int64_t)p.max_pages << p.page_shift) <= 1024 && (int64_t)p.R * p.H_KV <= sm_count();
}

int64_t decode_workspace(const AttnParams& p) {
  if (block_per_run(p)) return 0;
  const int grid = sm_count();
  return (tiles_of(p) == 1 ? ws_merge<1>(grid) : ws_merge<2>(grid)) * 4 + grid * (int64_t)sizeof(Merge);
}

template <int NT, bool kBf16>
static int launch(const AttnParams& p, cudaStream_t st) {
  const bool whole = block_per_run(p);
  const int grid = whole ? p.R * p.H_KV : sm_count(), smem = warps_of(NT) * kSlots * kUnitBytes;
  static thread_local int attr_dev = -1;
  int dev = 0;
  HQ_CUDA(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    HQ_CUDA(cudaFuncSetAttribute(decode_kernel<NT, kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_dev = dev;
  }
  cudaLaunchAttribute after{};
  after.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  after.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid); cfg.blockDim = dim3(warps_of(NT) * 32); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cfg.attrs = &after; cfg.numAttrs = 1;
  HQ_CUDA(cudaLaunchKernelEx(&cfg, decode_kernel<NT, kBf16>, p, whole));
  if (whole) return HQ_OK;
  cfg.gridDim = dim3(grid, p.max_q_len * p.G); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = 0;
  HQ_CUDA(cudaLaunchKernelEx(&cfg, merge_kernel<NT>, p, grid));
  return HQ_OK;
}

int decode_launch(const AttnParams& p, cudaStream_t st) {
  if (tiles_of(p) == 1) return p.dtype == HQ_BF16 ? launch<1, true>(p, st) : launch<1, false>(p, st);
  return p.dtype == HQ_BF16 ? launch<2, true>(p, st) : launch<2, false>(p, st);
}

}  // namespace paged
}  // namespace hq
