// Attention of many new tokens over the paged 4-bit cache (prompt chunks, long drafts): tcgen05 products with accumulators in
// tensor memory.
//
// A query tile is 256 rows of one kv head of one request - rows are (token, head of the group) pairs, one behind the other, whatever the
// group size - in two halves of 128; keys come in tiles of 64.  Bound by the tensor pipe and the exponentials, which take about the
// same time: 8.4 MFLOP and 16384 exponentials a tile pair, some 1024 clocks of an SM each at their nominal rates.
//
// One block per SM, 15 warps:
//   0-3, 4-7   softmax of the two halves, a thread per row; they also load the queries and write the results
//   8-11       the cache: codes become fp16 values (exact: the format sees to that) in the swizzled operand tiles that both halves
//              read, so that 64 keys are unpacked once for 256 rows
//   12, 13     issue the products of a half each: S = Q K^T into one of two buffers of 64 columns, O += P V with P (fp16, over the
//              buffer just read) from tensor memory and V's rows as they lie.  Q K^T of tile t + 2 follows P V of tile t.
//   14         fetches the codes: a tile is four blocks of sixteen tokens, a bulk copy each, some tiles ahead
// Channels stand in the order in which the unpacking produces them (0 4 1 5 2 6 3 7 in every eight), in Q, K and V alike; the rows that
// are written put them back.
//
// All query tiles' keys in a row (requests, heads, query tiles) are cut evenly over the blocks, by position: lengths are only known
// on the device, and no block is left with a long tile at the end.  A query tile that several blocks share leaves softmax states,
// which the merge kernel joins.
#include "hq_paged.cuh"
#include "hq_tc05.cuh"

namespace hq {
namespace paged {

constexpr int kTileThreads = 480, kRows = 256, kKeys = 64;
constexpr int kIssue = 12, kFetch = 14;          // first issuing warp; the fetching one
constexpr int kStages = 3;                       // K tiles, and V tiles, in shared memory
constexpr int kAhead = 4;                        // tiles of codes in shared memory
constexpr int kCodeBytes = kKeys / kTok * kBlockBytes;
constexpr int kItemCost = 2;                     // what a query tile costs beside its key tiles, in key tiles
constexpr float kTShift = 9.0f, kTMost = 32768.0f;        // P~ = 2^(s - m + 9); a tile's row sum that calls for a new reference
constexpr uint32_t kTPolls = 400000u;

struct TileSmem {
  static constexpr int Q = 0, K = 65536, V = K + kStages * 16384, Codes = V + kStages * 16384, Bar = Codes + kAhead * kCodeBytes,
                       Rows = Bar + 320, Bad = Rows + 4 * kAhead, Total = Bad + 16;
};
static_assert(TileSmem::Bar % 16 == 0 && TileSmem::Total + 1024 <= 227 * 1024, "shared memory");

struct TileMerge { int q0, rows, h, qt, first, go, unused[2]; };

// A query tile and where in it a block's part begins
struct Item {
  int r, h, qt, n_qt, u, tiles;
  Request q;
};
__device__ __forceinline__ int query_tiles(const AttnParams& p, const Request& q) { return (q.nq * p.G + kRows - 1) / kRows; }
__device__ __forceinline__ int key_tiles(const AttnParams& p, const Request& q, int qt) {
  const int last = min(q.nq * p.G, (qt + 1) * kRows) - 1;
  const int keys = min(q.len, q.past + 1 + last / p.G);
  return keys > 0 ? (keys + kKeys - 1) / kKeys : 0;
}
__device__ __forceinline__ void next_item(const AttnParams& p, Item& x) {
  x.u = 0;
  if (++x.qt >= x.n_qt) {
    x.qt = 0;
    if (++x.h >= p.H_KV) {
      x.h = 0;
      do {
        if (++x.r >= p.R) return;
        x.q = request_of(p, x.r);
        x.n_qt = query_tiles(p, x.q);
      } while (x.n_qt == 0);
    }
  }
  x.tiles = key_tiles(p, x.q, x.qt);
}
// A block's part as pieces of query tiles: key tiles [t0, t1) of `it`
struct Pieces {
  Item it;
  long long left;
  int t0, t1;
  bool began, ends;                              // earlier, in another block; here
  __device__ __forceinline__ bool take(const AttnParams& p) {
    while (left > 0) {
      const bool some = it.tiles > 0 ? it.u < it.tiles : it.u == 0;
      if (some) {
        began = it.u > 0;
        t0 = it.u;
        t1 = (int)min((long long)it.tiles, it.u + left);
        ends = t1 == it.tiles;
        return true;
      }
      done(p);
    }
    return false;
  }
  __device__ __forceinline__ void done(const AttnParams& p) {
    left -= it.tiles + kItemCost - it.u;
    if (left > 0) next_item(p, it);
  }
};

__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, tc::mbar_wait_abortable(bar, parity, abort_flag, 0, kTPolls));
}

struct SlowState { float m, l; bool ok; };

// A tile that needs masks or a new reference: the scores are read again, the maximum taken, O rescaled where a row's reference
// moves (where the maximum passes it by `slack`), P formed.  `lim`: keys of the tile that the row sees; bad: blocks of sixteen keys that are not there.
__device__ __noinline__ SlowState slow_tile(uint32_t tS, uint32_t tO, float f, int lim, uint32_t bad, float slack, float m, float l,
                                            uint64_t* pv_bar, uint32_t pv_parity, volatile int* abort_flag) {
  SlowState out{m, l, true};
  float x[64];
  tc::tmem_ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
  tc::tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&x[32]));
  tc::tmem_wait_ld();
  float mx = -INFINITY;
#pragma unroll
  for (int c = 0; c < 64; ++c) {
    x[c] = (c < lim && !((bad >> (c >> 4)) & 1u)) ? x[c] * f : -INFINITY;
    mx = fmaxf(mx, x[c]);
  }
  const bool grow = mx > m + slack;
  if (__any_sync(0xffffffffu, grow)) {
    const float alpha = !grow ? 1.f : m == -INFINITY ? 0.f : ex2f(m - mx);
    if (pv_bar != nullptr) {                     // O must be quiescent
      if (!wait_warp(pv_bar, pv_parity, abort_flag)) { out.ok = false; return out; }
      tc::fence_after_sync();
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        uint32_t o[32];
        tc::tmem_ld32(tO + ch * 32, o);
        tc::tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
        tc::tmem_st32(tO + ch * 32, o);
      }
      tc::tmem_wait_st();
    }
    out.l *= alpha;
    if (grow) out.m = mx;
  }
  const float shift = out.m == -INFINITY ? 0.f : kTShift - out.m;
  uint32_t pk[32];
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < 64; c += 2) {
    const float p0 = ex2f(x[c] + shift), p1 = ex2f(x[c + 1] + shift);
    sum += p0 + p1;
    const __half2 hh = __floats2half2_rn(p0, p1);
    pk[c >> 1] = *reinterpret_cast<const uint32_t*>(&hh);
  }
  tc::tmem_st32(tS, pk);
  tc::tmem_wait_st();
  out.l += sum;
  return out;
}

// eight codes -> eight values in the order 0 4 1 5 2 6 3 7: the nibble at the top of the mantissa is 16 + (code + 8), one fma takes 24
// scales off.  24 * scale and the result have at most ten and eleven bits: exact for scales up to 2048 (24 * scale is an fp16 number).
__device__ __forceinline__ uint4 values8(uint32_t w, __half2 s, __half2 s24) {
  const uint32_t x0 = lop3_and_xor(w << 6, 0x03C003C0u, 0x4E004E00u), x1 = lop3_and_xor(w << 2, 0x03C003C0u, 0x4E004E00u);
  const uint32_t x2 = lop3_and_xor(w >> 2, 0x03C003C0u, 0x4E004E00u), x3 = lop3_and_xor(w >> 6, 0x03C003C0u, 0x4E004E00u);
  auto val = [&](uint32_t x) {
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&x), s, s24);
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  return make_uint4(val(x0), val(x1), val(x2), val(x3));
}
// the same for any scale: the code by itself first
__device__ __forceinline__ uint4 values8_any(uint32_t w, __half2 s) {
  const uint32_t x0 = lop3_and_xor(w << 6, 0x03C003C0u, 0x4E004E00u), x1 = lop3_and_xor(w << 2, 0x03C003C0u, 0x4E004E00u);
  const uint32_t x2 = lop3_and_xor(w >> 2, 0x03C003C0u, 0x4E004E00u), x3 = lop3_and_xor(w >> 6, 0x03C003C0u, 0x4E004E00u);
  const __half2 c24 = __float2half2_rn(24.f);
  auto val = [&](uint32_t x) {
    const __half2 v = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&x), c24), s);
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  return make_uint4(val(x0), val(x1), val(x2), val(x3));
}

template <bool kBf16>
__global__ void __launch_bounds__(kTileThreads, 1)
tile_kernel(const AttnParams p, int piece_rows) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + TileSmem::Bar);
  uint64_t* q_full = bars;                       // [half]
  uint64_t* k_full = bars + 2;                   // [stage]
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* c_full = v_empty + kStages;          // [kAhead]
  uint64_t* c_empty = c_full + kAhead;
  uint64_t* s_full = c_empty + kAhead;           // [half][2]
  uint64_t* p_ready = s_full + 4;
  uint64_t* pv_done = p_ready + 4;
  uint64_t* drained = pv_done + 4;               // [half]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ long long s_part[kTileThreads + 1], s_warp[kTileThreads / 32];
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (warp == kIssue) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) { mbar_init(q_full + i, 128); mbar_init(drained + i, 1); }
      for (int i = 0; i < kStages; ++i) { mbar_init(k_full + i, 4); mbar_init(k_empty + i, 2); mbar_init(v_full + i, 4); mbar_init(v_empty + i, 2); }
      for (int i = 0; i < kAhead; ++i) { mbar_init(c_full + i, 1); mbar_init(c_empty + i, 4); }
      for (int i = 0; i < 4; ++i) { mbar_init(s_full + i, 1); mbar_init(p_ready + i, 128); mbar_init(pv_done + i, 1); }
      *abort_flag = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tc::tmem_alloc(tmem_slot, 512);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- where this block's part lies
  auto weight = [&](const Request& q) {
    long long w = 0;
    for (int qt = 0, n = query_tiles(p, q); qt < n; ++qt) w += key_tiles(p, q, qt) + kItemCost;
    return w;
  };
  const int per = (p.R + kTileThreads - 1) / kTileThreads;
  long long mine = 0;
  for (int r = tid * per; r < min(p.R, (tid + 1) * per); ++r) mine += p.H_KV * weight(request_of(p, r));
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const long long y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < kTileThreads / 32; ++w) { if (w < warp) before += s_warp[w]; total += s_warp[w]; }
  s_part[tid + 1] = before + x;
  if (tid == 0) s_part[0] = 0;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const int blocks = (int)max(1ll, min((long long)gridDim.x, total / (kItemCost + 1))), block = blockIdx.x;
  const int64_t piece_floats = (int64_t)piece_rows * 130;
  TileMerge* todo = reinterpret_cast<TileMerge*>(p.ws + 2 * piece_floats * gridDim.x) + block;
  const long long b0 = block < blocks ? total * block / blocks : 0, b1 = block < blocks ? total * (block + 1) / blocks : 0;
  if (tid == 0) todo->go = 0;
  Pieces pc;
  pc.left = b1 - b0;
  if (pc.left > 0) {
    int lo = 0, hi = kTileThreads;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (s_part[mid] <= b0) lo = mid; else hi = mid; }
    long long at = s_part[lo];
    Item it;
    it.r = lo * per;
    long long w;
    for (;; ++it.r) {
      it.q = request_of(p, it.r);
      w = weight(it.q);
      if (b0 < at + w * p.H_KV) break;
      at += w * p.H_KV;
    }
    it.h = (int)((b0 - at) / w);
    long long in = b0 - at - it.h * w;
    it.n_qt = query_tiles(p, it.q);
    for (it.qt = 0;; ++it.qt) {
      it.tiles = key_tiles(p, it.q, it.qt);
      if (in < it.tiles + kItemCost) break;
      in -= it.tiles + kItemCost;
    }
    it.u = (int)in;
    pc.it = it;
  }

  int* key_rows = reinterpret_cast<int*>(smem + TileSmem::Rows);           // [kAhead] keys of a tile that are there, the last ones missing
  uint8_t* bads = smem + TileSmem::Bad;                                    // [16] blocks of a tile whose page is not there
  if (warp == kFetch) {
    // ------------------------------------------------------------ codes
    const int num_pages = (int)p.num_pages, page_bytes = kBlockBytes << (p.page_shift - 4), blocks_mask = (1 << (p.page_shift - 4)) - 1;
    int tab_r = -1, tab_t = 0, pg = -1;          // pages of eight tiles of request tab_r: lane 4 i + b, block b of tile tab_t + i
    int stage = 0;
    uint32_t par = 1u, tile = 0;                 // empty barriers: the first round passes
    bool ok = true;
    while (ok && pc.take(p)) {
#pragma unroll 1
      for (int t = pc.t0; t < pc.t1; ++t, ++tile) {
        if (pc.it.r != tab_r || t < tab_t || t >= tab_t + 8) {
          tab_r = pc.it.r; tab_t = t;
          const int64_t tok = ((int64_t)t + (lane >> 2)) * kKeys + kTok * (lane & 3);
          pg = tok < pc.it.q.len ? __ldg(p.table + (int64_t)tab_r * p.table_stride + (tok >> p.page_shift)) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, pg, 4 * (t - tab_t) + (lane & 3)), tok = t * kKeys + kTok * (lane & 3);
        const bool in = tok < pc.it.q.len && lane < 4, there = in && (uint32_t)page < (uint32_t)num_pages;
        const uint32_t have = __ballot_sync(0xffffffffu, there), gone = __ballot_sync(0xffffffffu, in && !there);
        ok = wait_warp(c_empty + stage, par, abort_flag);
        if (!ok) break;
        if (lane == 0) {
          key_rows[stage] = min(kKeys, pc.it.q.len - t * kKeys) | (int)(gone << 16);
          bads[tile & 15u] = (uint8_t)gone;
          mbar_expect_tx(c_full + stage, __popc(have) * kBlockBytes);
        }
        __syncwarp();
        if (there)
          bulk_g2s(smem + TileSmem::Codes + stage * kCodeBytes + lane * kBlockBytes,
                   p.pages + (int64_t)(page * p.H_KV + pc.it.h) * page_bytes + ((tok >> 4) & blocks_mask) * kBlockBytes, kBlockBytes, c_full + stage);
        if (++stage == kAhead) { stage = 0; par ^= 1u; }
      }
      pc.done(p);
    }
    // a block must not end with copies under way, also where it gives up: wait for the last load of every slot
    for (int i = 0; i < kAhead; ++i) mbar_wait_bounded(c_full + i, i < stage ? par ^ 1u : par, kTPolls);
  } else if (warp >= kIssue) {
    // ------------------------------------------------------------ products of one half
    const int half = warp - kIssue;
    const uint32_t idesc_qk = tc::make_idesc(1, 0, 0, 128, kKeys), idesc_pv = tc::make_idesc(1, 0, 0, 128, 128) | tc::kBMnMajor;
    const uint64_t dQ = tc::smem_desc_k128(smem + TileSmem::Q + half * 32768, 0);
    const uint64_t dK = tc::smem_desc_k128(smem + TileSmem::K, 0), dV = tc::smem_desc_mn128(smem + TileSmem::V, 8192);
    const uint32_t tS = tmem + 128u * half, tO = tmem + 256u + 128u * half;
    int ks = 0, vs = 0;
    uint32_t kpar = 0, vpar = 0, tile = 0, q_par = 0;       // tile: of this half, over all pieces
    bool ok = true;
    auto k_step = [&]() { if (++ks == kStages) { ks = 0; kpar ^= 1u; } };
    auto v_step = [&]() { if (++vs == kStages) { vs = 0; vpar ^= 1u; } };
    while (ok && pc.take(p)) {
      const int n = pc.t1 - pc.t0, rows = pc.it.q.nq * p.G - pc.it.qt * kRows - 128 * half;
      if (n > 0 && rows <= 0) {                  // the other half's tiles: handed back as they come
        for (int t = 0; ok && t < n; ++t) {
          ok = wait_warp(k_full + ks, kpar, abort_flag);
          if (ok && tc::elect_one()) tc::mbar_arrive(k_empty + ks);
          ok = ok && wait_warp(v_full + vs, vpar, abort_flag);
          if (ok && tc::elect_one()) tc::mbar_arrive(v_empty + vs);
          k_step(); v_step();
        }
      } else if (n > 0) {
        ok = wait_warp(q_full + half, q_par, abort_flag);
        q_par ^= 1u;
        uint32_t tq = tile;
        auto qk = [&]() {
          ok = ok && wait_warp(k_full + ks, kpar, abort_flag);
          if (!ok) return;
          tc::fence_after_sync();
          if (tc::elect_one()) {
            const uint32_t dS = tS + 64u * (tq & 1u);
            const uint64_t bK = dK + (uint64_t)(ks * 1024);
#pragma unroll
            for (int k = 0; k < 8; ++k) tc::mma_bf16_ss(dS, dQ + (k >> 2) * 1024 + 2 * (k & 3), bK + (k >> 2) * 512 + 2 * (k & 3), idesc_qk, k > 0);
            tc::mma_commit(k_empty + ks);
            tc::mma_commit(s_full + 2 * half + (tq & 1u));
          }
          __syncwarp();
          ++tq;
          k_step();
        };
        qk();
        if (n > 1) qk();
        for (int t = 0; ok && t < n; ++t, ++tile) {
          ok = wait_warp(v_full + vs, vpar, abort_flag) && wait_warp(p_ready + 2 * half + (tile & 1u), (tile >> 1) & 1u, abort_flag);
          if (!ok) break;
          tc::fence_after_sync();
          if (tc::elect_one()) {
            const uint32_t aP = tS + 64u * (tile & 1u);
            const uint64_t bV = dV + (uint64_t)(vs * 1024);
#pragma unroll
            for (int k = 0; k < 4; ++k) tc::mma_bf16_ts(tO, aP + 8 * k, bV + 128 * k, idesc_pv, (t > 0 || k > 0) ? 1u : 0u);
            tc::mma_commit(v_empty + vs);
            tc::mma_commit(pv_done + 2 * half + (tile & 1u));
          }
          __syncwarp();
          v_step();
          if (t + 2 < n) qk();
        }
      }
      pc.done(p);
    }
    // nothing may still write tensor memory or arrive on a barrier when the block ends
    if (tc::elect_one()) tc::mma_commit(drained + half);
    __syncwarp();
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(drained + half, 0, kTPolls)) || !ok) *abort_flag = 1;
  } else if (warp >= 8) {
    // ------------------------------------------------------------ the cache: codes to operand tiles
    // Lane: row lane / 4 of a group of eight keys, channels 32 (lane % 4) ..  A warp reads 512 bytes in one piece; the lanes of the
    // upper channels take their words two apart, so that no two of eight lanes write to the same banks either.
    const int w = warp - 8, rowl = lane >> 2, quarter = lane & 3, turn = quarter & 2;
    int n_all = 0;
    while (pc.take(p)) { n_all += pc.t1 - pc.t0; pc.done(p); }
    int ks = 0;
    uint32_t kpar = 1u;                          // empty barriers: the first round passes
    bool ok = true;
#pragma unroll 1
    for (int tile = 0; ok && tile < n_all; ++tile) {
      const int cs = tile % kAhead;
      ok = wait_warp(c_full + cs, (uint32_t)(tile / kAhead) & 1u, abort_flag);
      if (!ok) break;
      const uint8_t* block = smem + TileSmem::Codes + cs * kCodeBytes + w * kBlockBytes;       // keys 16 w .. + 15
      const int info = key_rows[cs], rows = ((info >> (16 + w)) & 1) ? 0 : (info & 0xFFFF) - kTok * w;
      uint8_t* to = smem + TileSmem::K + ks * 16384 + (quarter >> 1) * 8192 + (kTok * w + rowl) * 128;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        uint4 val[2][4];
        {
          uint4 c[2];
          float s[2];
#pragma unroll
          for (int g = 0; g < 2; ++g) {          // keys 16 w + 8 g .. + 7
            c[g] = *reinterpret_cast<const uint4*>(block + kv * kVOff + g * 512 + lane * 16);
            const uint16_t sb = *reinterpret_cast<const uint16_t*>(block + (kv ? kVsOff : kKsOff) + 2 * (8 * g + rowl));
            s[g] = 8 * g + rowl < rows ? __uint_as_float((uint32_t)sb << 16) : 0.f;        // keys that are not there: zeros, whatever lies here
          }
          const bool big = __any_sync(0xffffffffu, s[0] > 2048.f || s[1] > 2048.f);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const uint32_t cw[4] = {turn ? c[g].z : c[g].x, turn ? c[g].w : c[g].y, turn ? c[g].x : c[g].z, turn ? c[g].y : c[g].w};
            const __half2 s2 = __float2half2_rn(s[g]), s24 = __float2half2_rn(-24.f * s[g]);
            if (__builtin_expect(big, 0)) {
#pragma unroll
              for (int k = 0; k < 4; ++k) val[g][k] = values8_any(cw[k], s2);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) val[g][k] = values8(cw[k], s2, s24);
            }
          }
        }
        // the values are in registers before their place is free: from then on it takes eight stores
        ok = ok && wait_warp((kv ? v_empty : k_empty) + ks, kpar, abort_flag);
        if (ok) {
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<uint4*>(to + kv * (TileSmem::V - TileSmem::K) + g * 1024 + (((((quarter & 1) << 2) + (k ^ turn)) ^ rowl) << 4)) = val[g][k];
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (kv) tc::mbar_arrive(c_empty + cs);
            tc::mbar_arrive((kv ? v_full : k_full) + ks);
          }
        }
      }
      if (++ks == kStages) { ks = 0; kpar ^= 1u; }
    }
  } else {
    // ------------------------------------------------------------ softmax: a thread per row
    const int half = warp >> 2, wq = warp & 3, r = wq * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(wq * 32) << 16), tO = lane_base + 256u + 128u * half;
    uint8_t* sQ = smem + TileSmem::Q + half * 32768;
    uint32_t tile = 0, all = 0;                  // tiles of this half; of the block
    bool ok = true;
    while (pc.take(p)) {
      const Request& q = pc.it.q;
      const int n = pc.t1 - pc.t0, rows = min(128, q.nq * p.G - pc.it.qt * kRows - 128 * half);
      const int row = pc.it.qt * kRows + 128 * half + r, i = row / p.G, gh = pc.it.h * p.G + row - i * p.G;
      float m = -INFINITY, l = 0.f;
      if (n > 0 && rows > 0 && ok) {
        // queries: scaled by a power of two of the row so that fp16 holds them exactly, into the operand tile
        float f;
        {
          const uint16_t* from = reinterpret_cast<const uint16_t*>(p.q) + (int64_t)(q.q0 + i) * p.q_st + (int64_t)gh * p.q_sh;
          const bool live = r < rows;
          auto value = [&](uint32_t u, int hi) {
            if (kBf16) return __uint_as_float(hi ? u & 0xFFFF0000u : u << 16);
            return __half2float(__ushort_as_half((unsigned short)(hi ? u >> 16 : u & 0xFFFFu)));
          };
          float top = 0.f;
          uint4 raw[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) raw[c] = live ? __ldg(reinterpret_cast<const uint4*>(from) + c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const uint32_t u[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(fabsf(value(u[k], 0)), fabsf(value(u[k], 1))));
          }
          const int ex = (int)(__float_as_uint(top) >> 23), up = ex == 255 ? 0 : 140 - max(ex, 14);       // largest magnitude to [2^13, 2^14)
          const float scale = __uint_as_float((uint32_t)(127 + up) << 23);
          f = p.sml * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const uint32_t u[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {        // channels k and k + 4 of the eight
              const __half2 hh = __floats2half2_rn(value(u[k >> 1], k & 1) * scale, value(u[2 + (k >> 1)], k & 1) * scale);
              o[k] = *reinterpret_cast<const uint32_t*>(&hh);
            }
            *reinterpret_cast<uint4*>(sQ + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        fence_proxy_async_smem();
        tc::mbar_arrive(q_full + half);
        const int lim = r < rows ? min(q.len, q.past + 1 + i) : 0x7FFFFFFF;      // rows that are none see everything: finite, not written
        float shift = INFINITY;
        const float2 f2 = make_float2(f, f);
#pragma unroll 1
        for (int t = 0; t < n; ++t, ++tile) {
          const uint32_t slot = tile & 1u;
          ok = wait_warp(s_full + 2 * half + slot, (tile >> 1) & 1u, abort_flag);
          if (!ok) break;
          tc::fence_after_sync();
          const uint32_t tS = lane_base + 128u * half + 64u * slot;
          const uint32_t bad = bads[(all + t) & 15u];
          const int see = lim - (pc.t0 + t) * kKeys;
          const bool masks = __any_sync(0xffffffffu, see < kKeys || bad != 0u);
          bool need = false;
          uint32_t pk[32];
          float sum = 0.f;
          if (!masks) {
            uint32_t s[64];
            tc::tmem_ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
            tc::tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
            tc::tmem_wait_ld();
            const float2 sh2 = make_float2(shift, shift);
            float2 a = make_float2(0.f, 0.f), b = a;
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float2 y = ffma2(make_float2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), f2, sh2);
              const float2 e = make_float2(ex2f(y.x), ex2f(y.y));
              if (c & 1) b = fadd2(b, e); else a = fadd2(a, e);
              const __half2 hh = __floats2half2_rn(e.x, e.y);
              pk[c] = *reinterpret_cast<const uint32_t*>(&hh);
            }
            a = fadd2(a, b);
            sum = a.x + a.y;
            need = !(sum <= kTMost);
          }
          if (__builtin_expect(masks || __any_sync(0xffffffffu, need), 0)) {
            const SlowState x2 = slow_tile(tS, tO, f, see, bad, need ? 0.f : 4.f, m, l, t > 0 ? pv_done + 2 * half + (slot ^ 1u) : nullptr,
                                           ((tile - 1u) >> 1) & 1u, abort_flag);
            ok = x2.ok;
            if (!ok) break;
            m = x2.m; l = x2.l;
            shift = m == -INFINITY ? INFINITY : kTShift - m;
          } else {
            l += sum;
            tc::tmem_st32(tS, pk);
            tc::tmem_wait_st();
          }
          tc::fence_before_sync();
          tc::mbar_arrive(p_ready + 2 * half + slot);
        }
        if (ok) ok = wait_warp(pv_done + 2 * half + ((tile - 1u) & 1u), ((tile - 1u) >> 1) & 1u, abort_flag);
        tc::fence_after_sync();
      }
      all += (uint32_t)n;
      if (rows > 0) {
        // O leaves through the rows' own part of the query tile, 32 columns at a time, so that a store writes whole sectors
        const bool whole = !pc.began && pc.ends;
        if (!ok) { m = 0.f; l = __int_as_float(0x7FC00000); }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        float* piece = p.ws + (int64_t)(2 * block + (pc.began ? 0 : 1)) * piece_floats;
        uint8_t* stage = sQ + wq * 32 * 128;     // of the first half of the channels: 4 KB that only this warp touches
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          float o[32];
          if (n > 0 && ok) {
            tc::tmem_ld32(tO + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
            tc::tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          __syncwarp();
          // column 8 k + 2 j + b holds channel 8 k + 4 b + j
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = o[8 * k + 2 * j]; v[4 + j] = o[8 * k + 2 * j + 1]; }
            if (whole) {
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = ok ? v[j] * inv : __int_as_float(0x7FC00000);
              uint32_t u[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (kBf16) { const __nv_bfloat162 hh = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]); u[j] = *reinterpret_cast<const uint32_t*>(&hh); }
                else { const __half2 hh = __floats2half2_rn(v[2 * j], v[2 * j + 1]); u[j] = *reinterpret_cast<const uint32_t*>(&hh); }
              }
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((k ^ (lane & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
            } else {
              *reinterpret_cast<float4*>(stage + lane * 128 + (((2 * k) ^ (lane & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
              *reinterpret_cast<float4*>(stage + lane * 128 + (((2 * k + 1) ^ (lane & 7)) << 4)) = make_float4(v[4], v[5], v[6], v[7]);
            }
          }
          __syncwarp();
          if (whole) {                           // four lanes a row, 64 bytes
#pragma unroll
            for (int x8 = 0; x8 < 4; ++x8) {
              const int rr = 8 * x8 + (lane >> 2), part = lane & 3, orow = wq * 32 + rr;
              const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((part ^ (rr & 7)) << 4));
              if (orow < rows) {
                const int grow = pc.it.qt * kRows + 128 * half + orow, gi = grow / p.G;
                *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + (int64_t)(q.q0 + gi) * p.o_st +
                                          (int64_t)(pc.it.h * p.G + grow - gi * p.G) * p.o_sh + ch * 32 + part * 8) = v;
              }
            }
          } else {                               // eight lanes a row, 128 bytes
#pragma unroll
            for (int x4 = 0; x4 < 8; ++x4) {
              const int rr = 4 * x4 + (lane >> 3), part = lane & 7, orow = wq * 32 + rr;
              const float4 v = *reinterpret_cast<const float4*>(stage + rr * 128 + ((part ^ (rr & 7)) << 4));
              if (orow < rows) *reinterpret_cast<float4*>(piece + (int64_t)(128 * half + orow) * 128 + ch * 32 + part * 4) = v;
            }
          }
        }
        __syncwarp();
        if (!whole && r < rows) {
          piece[(int64_t)piece_rows * 128 + 128 * half + r] = m;
          piece[(int64_t)piece_rows * 129 + 128 * half + r] = l;
        }
      }
      if (pc.began && pc.ends && tid == 0) {
        const long long start = b0 - pc.t0;      // the block's first piece: its query tile began t0 positions before
        int first = (int)(start * blocks / total);
        while (total * first / blocks > start) --first;
        while (total * (first + 1) / blocks <= start) ++first;
        *todo = TileMerge{q.q0, min(kRows, q.nq * p.G - pc.it.qt * kRows), pc.it.h, pc.it.qt, first, 1, {0, 0}};
      }
      pc.done(p);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kIssue) tc::tmem_dealloc(tmem, 512);
}

// Query tiles that several blocks share: a warp a row, over the pieces of the blocks first .. b.
__global__ void __launch_bounds__(256)
tile_merge_kernel(const AttnParams p, int piece_rows, int grid) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.x, lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int64_t piece_floats = (int64_t)piece_rows * 130;
  const TileMerge todo = reinterpret_cast<const TileMerge*>(p.ws + 2 * piece_floats * grid)[b];
  if (!todo.go || row >= todo.rows) return;
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = todo.first; i <= b; ++i) {
    const float* x = p.ws + (int64_t)(2 * i + (i == todo.first ? 1 : 0)) * piece_floats;
    const float m = x[(int64_t)piece_rows * 128 + row], l = x[(int64_t)piece_rows * 129 + row];
    const float4 v = *reinterpret_cast<const float4*>(x + (int64_t)row * 128 + 4 * lane);
    const float nm = fmaxf(M, m), ref = nm == -INFINITY ? 0.f : nm, wo = ex2f(M - ref), w = ex2f(m - ref);
    L = L * wo + l * w;
    acc.x = acc.x * wo + v.x * w; acc.y = acc.y * wo + v.y * w; acc.z = acc.z * wo + v.z * w; acc.w = acc.w * wo + v.w * w;
    M = nm;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int grow = todo.qt * kRows + row, gi = grow / p.G;
  const int64_t at = (int64_t)(todo.q0 + gi) * p.o_st + (int64_t)(todo.h * p.G + grow - gi * p.G) * p.o_sh + 4 * lane;
  uint2 o;
  if (p.dtype == HQ_BF16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), c = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
    o = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
  } else {
    const __half2 a = __floats2half2_rn(acc.x * inv, acc.y * inv), c = __floats2half2_rn(acc.z * inv, acc.w * inv);
    o = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
  }
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) = o;
}

static int piece_rows_of(const AttnParams& p) { return (int)min((int64_t)kRows, (int64_t)p.max_q_len * p.G); }

int64_t tile_workspace(const AttnParams& p) {
  const int64_t grid = sm_count();
  return (2 * (int64_t)piece_rows_of(p) * 130 * 4 + (int64_t)sizeof(TileMerge)) * grid;
}

int tile_launch(const AttnParams& p, cudaStream_t st) {
  const int grid = sm_count(), smem = TileSmem::Total + 1024, rows = piece_rows_of(p);
  static thread_local int attr_dev = -1;
  int dev = 0;
  HQ_CUDA(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    HQ_CUDA(cudaFuncSetAttribute(tile_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    HQ_CUDA(cudaFuncSetAttribute(tile_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_dev = dev;
  }
  cudaLaunchAttribute after{};
  after.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  after.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid); cfg.blockDim = dim3(kTileThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cfg.attrs = &after; cfg.numAttrs = 1;
  if (p.dtype == HQ_BF16) HQ_CUDA(cudaLaunchKernelEx(&cfg, tile_kernel<true>, p, rows));
  else HQ_CUDA(cudaLaunchKernelEx(&cfg, tile_kernel<false>, p, rows));
  cfg.gridDim = dim3(grid, (rows + 7) / 8); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = 0;
  HQ_CUDA(cudaLaunchKernelEx(&cfg, tile_merge_kernel, p, rows, grid));
  return HQ_OK;
}

}  // namespace paged
}  // namespace hq
