// Attention of many new tokens over the paged 4-bit cache (prompt chunks, long drafts): tcgen05 products with accumulators in
// tensor memory.
//
// A query tile is 256 rows of one kv head of one request - rows are (token, head of the group) pairs, one behind the other, whatever the
// group size; keys come in tiles of 64.  The two halves of the softmax take 128 rows each, or, where a query tile has no more than
// 128 rows, the same rows and every other key tile, and join their states at the end.  A key tile of 256 rows is 8.4 MFLOP and 16384
// exponentials, some 1024 clocks of an SM each at their nominal rates; the products' operands and the unpacked tiles pass through
// shared memory in some 1600.  It takes 1850 with all that runs once (1.59 M clocks for 859 key tiles an SM): a prompt of 2048 tokens over
// 32768 cached ones, 32 heads over 8, 894 to 915 us in a short run, 1.18 PFLOP/s, 1024 in a long one at the power cap's clock.  Counters: tensor
// pipe 55 %, issue slots 53 %, ALU pipe 34 %.
// Exponentials moved to the FMA pipe (an eighth to a half of them, by polynomial) gave nothing, key tiles of 128 lost the second
// buffer of scores and took 1236 us where 64 took 1052.
//
// One block per SM, 15 warps:
//   0-3, 4-7   softmax of the two halves, a thread per row; they also load the queries and write the results
//   8-11       the cache: codes become fp16 values (exact: the format sees to that) in the swizzled operand tiles that both halves
//              read, so that 64 keys are unpacked once for 256 rows
//   12, 13     issue the products of a half each: S = Q K^T into one of two buffers of 64 columns, O += P V with P (fp16, over the
//              buffer just read) from tensor memory and V's rows as they lie.  Q K^T of the next tile but one follows P V.
//   14         fetches the codes: a tile is four blocks of sixteen tokens, a bulk copy each, some tiles ahead
// Channels stand in the order in which the unpacking produces them (0 4 1 5 2 6 3 7 in every eight), in Q, K and V alike; the rows that
// are written put them back.  What runs once per query tile is written as loops: straight-line code that is met cold costs more
// for its instructions' way to the SM than for their execution (results 10800 -> 5000 clocks).  480 threads leave 128 registers each, and 60
// bytes are spilled; registers moved between the roles took longer.
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
constexpr int kKStages = 3, kVStages = 4;        // K tiles and V tiles in shared memory
constexpr int kAhead = 4;                        // tiles of codes in shared memory
constexpr int kCodeBytes = kKeys / kTok * kBlockBytes;
constexpr float kTShift = 9.0f, kTMost = 32768.0f;        // P~ = 2^(s - m + 9); a tile's row sum that calls for a new reference
// Scores (log2) up to which a rounded reference will do: it is off by 2^-12 of a power of two at most.  Exact differences in every tile took 930
// us where the prompt takes 910.
constexpr float kTFar = 8192.0f;
constexpr uint32_t kTPolls = 400000u;

struct TileSmem {
  static constexpr int Q = 0, K = 65536, V = K + kKStages * 16384, Codes = V + kVStages * 16384, Bar = Codes + kAhead * kCodeBytes,
                       Rows = Bar + 320, Bad = Rows + 4 * kAhead, Total = Bad + 16;
};
static_assert(TileSmem::Bar % 16 == 0 && TileSmem::Total + 1024 <= 227 * 1024, "shared memory");

struct TileMerge { int q0, rows, h, qt, first, go, unused[2]; };

// A query tile and where in it a block's part begins
struct Item {
  int r, h, qt, n_qt, u, tiles;
  bool split;                                    // every other key tile to each half
  Request q;
  __device__ __forceinline__ int positions() const { return tiles * (split ? kSplitCost : kFullCost) + kItemCost; }
  __device__ __forceinline__ int tiles_to(int u) const {       // key tiles that begin before position u
    return min(tiles, split ? (u + kSplitCost - 1) / kSplitCost : (u + kFullCost - 1) / kFullCost);
  }
};
__device__ __forceinline__ int query_tiles(const AttnParams& p, const Request& q) { return (q.nq * p.G + kRows - 1) / kRows; }
__device__ __forceinline__ void size_item(const AttnParams& p, Item& x) {
  const int rows = x.q.nq * p.G, last = min(rows, (x.qt + 1) * kRows) - 1;
  const int keys = min(x.q.len, x.q.past + 1 + token_of(p, last));
  x.tiles = keys > 0 ? (keys + kKeys - 1) / kKeys : 0;
  x.split = rows - x.qt * kRows <= 128;
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
  size_item(p, x);
}
// A block's part as pieces of query tiles: key tiles [t0, t1) of `it`
struct Pieces {
  Item it;
  int left, t0, t1;
  bool began, ends;                              // earlier, in another block; here
  __device__ __forceinline__ bool take(const AttnParams& p) {
    while (left > 0) {
      t0 = it.tiles_to(it.u);
      t1 = it.tiles_to(it.u + left);
      began = it.u > 0;
      ends = t1 == it.tiles;
      if (t1 > t0 || (it.tiles == 0 && it.u == 0)) return true;
      done(p);
    }
    return false;
  }
  __device__ __forceinline__ void done(const AttnParams& p) {
    left -= it.positions() - it.u;
    if (left > 0) next_item(p, it);
  }
  __device__ __forceinline__ bool split() const { return it.split; }
};
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, tc::mbar_wait_abortable(bar, parity, abort_flag, 0, kTPolls));
}

struct SlowState { float m, l; bool ok; };

// A tile that needs masks or a new reference: the products are read again, the maximum taken, O rescaled where a row's reference
// moves (where the maximum passes it by `slack`), P formed.  `lim`: keys of the tile that the row sees; bad: blocks of sixteen keys that are
// not there.  A row's reference m is a product of the tensor core, its score m f.  Differences are taken before the factor here: equal scores
// have equal weights, whatever their size.
__device__ __noinline__ SlowState slow_tile(uint32_t tS, uint32_t tO, float f, int lim, uint32_t bad, float slack, float m, float l,
                                            uint64_t* pv_bar, uint32_t pv_parity, volatile int* abort_flag) {
  SlowState out{m, l, true};
  uint32_t see[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int n = lim - 32 * c;
    see[c] = n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
    if ((bad >> (2 * c)) & 1u) see[c] &= 0xFFFF0000u;
    if ((bad >> (2 * c + 1)) & 1u) see[c] &= 0x0000FFFFu;
  }
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    float x[32];
    tc::tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
    tc::tmem_wait_ld();
    const uint32_t mask = c ? see[1] : see[0];
#pragma unroll
    for (int e = 0; e < 32; ++e) mx = fmaxf(mx, (mask >> e) & 1u ? x[e] : -INFINITY);
  }
  const bool grow = m == -INFINITY ? mx > m : (mx - m) * f > slack;
  if (__any_sync(0xffffffffu, grow)) {
    const float alpha = !grow ? 1.f : m == -INFINITY ? 0.f : ex2f((m - mx) * f);
    if (pv_bar != nullptr) {                     // O must be quiescent
      if (!wait_warp(pv_bar, pv_parity, abort_flag)) { out.ok = false; return out; }
      tc::fence_after_sync();
#pragma unroll 1
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
  const float base = out.m == -INFINITY ? 0.f : out.m;
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {                  // P of columns 32 c .. lands in columns 16 c .., which have been read
    float x[32];
    tc::tmem_ld32(tS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
    tc::tmem_wait_ld();
    const uint32_t mask = c ? see[1] : see[0];
    uint32_t pk[16];
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      const float p0 = (mask >> e) & 1u ? ex2f(fmaf(x[e] - base, f, kTShift)) : 0.f, p1 = (mask >> (e + 1)) & 1u ? ex2f(fmaf(x[e + 1] - base, f, kTShift)) : 0.f;
      sum += p0 + p1;
      const __half2 hh = __floats2half2_rn(p0, p1);
      pk[e >> 1] = *reinterpret_cast<const uint32_t*>(&hh);
    }
    tc::tmem_st16(tS + 16 * c, pk);
  }
  tc::tmem_wait_st();
  out.l += sum;
  return out;
}

__device__ __forceinline__ void halves_meet() { asm volatile("bar.sync 1, 256;" ::: "memory"); }      // the eight softmax warps

template <bool kBf16>
__global__ void __launch_bounds__(kTileThreads, 1)
tile_kernel(const AttnParams p, int piece_rows) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + TileSmem::Bar);
  uint64_t* q_full = bars;                       // [half]
  uint64_t* k_full = bars + 2;                   // [stage]
  uint64_t* k_empty = k_full + kKStages;
  uint64_t* v_full = k_empty + kKStages;
  uint64_t* v_empty = v_full + kVStages;
  uint64_t* c_full = v_empty + kVStages;          // [kAhead]
  uint64_t* c_empty = c_full + kAhead;
  uint64_t* s_full = c_empty + kAhead;           // [half][2]
  uint64_t* p_ready = s_full + 4;
  uint64_t* pv_done = p_ready + 4;
  uint64_t* drained = pv_done + 4;               // [half]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int s_part[kTileThreads + 1], s_warp[kTileThreads / 32];
  __shared__ float2 s_state[2][128];             // (maximum, sum) of a half's rows, for the other
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

  if (warp == kIssue) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) { mbar_init(q_full + i, 128); mbar_init(drained + i, 1); }
      for (int i = 0; i < kKStages; ++i) { mbar_init(k_full + i, 4); mbar_init(k_empty + i, 2); }
      for (int i = 0; i < kVStages; ++i) { mbar_init(v_full + i, 4); mbar_init(v_empty + i, 2); }
      for (int i = 0; i < kAhead; ++i) { mbar_init(c_full + i, 1); mbar_init(c_empty + i, 4); }
      for (int i = 0; i < 4; ++i) { mbar_init(s_full + i, 1); mbar_init(p_ready + i, 128); mbar_init(pv_done + i, 1); }
      *abort_flag = 0;
      fence_mbar_init();
    }
    __syncwarp();
    tc::tmem_alloc(tmem_slot, 512);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- where this block's part lies
  auto weight = [&](const Request& q) {
    Item x;
    x.q = q;
    int w = 0;
    for (x.qt = 0, x.n_qt = query_tiles(p, q); x.qt < x.n_qt; ++x.qt) { size_item(p, x); w += x.positions(); }
    return w * p.H_KV;
  };
  const Prefix<kTileThreads, decltype(weight)> prefix(p, weight, s_part, s_warp);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const Cuts cuts(prefix.total, max(1, min((int)gridDim.x, prefix.total / (kItemCost + kFullCost))));
  const int block = blockIdx.x;
  const int b0 = cuts.begin(block);
  const int64_t piece_floats = (int64_t)piece_rows * 130;
  TileMerge* todo = reinterpret_cast<TileMerge*>(p.ws + 2 * piece_floats * gridDim.x) + block;
  if (tid == 0) todo->go = 0;
  Pieces pc;
  pc.left = block < cuts.blocks ? cuts.begin(block + 1) - b0 : 0;
  if (pc.left > 0) {
    Item it;
    int in;
    it.r = prefix.seek(b0, in);
    it.q = request_of(p, it.r);
    const int w = weight(it.q) / p.H_KV;
    it.h = in / w;
    in -= it.h * w;
    it.n_qt = query_tiles(p, it.q);
    for (it.qt = 0;; ++it.qt) {
      size_item(p, it);
      if (in < it.positions()) break;
      in -= it.positions();
    }
    it.u = in;
    pc.it = it;
  }
  int* key_rows = reinterpret_cast<int*>(smem + TileSmem::Rows);           // [kAhead] keys of a tile that are there, the last ones missing
  uint8_t* bads = smem + TileSmem::Bad;                                    // [16] blocks of a tile whose page is not there
  if (warp == kFetch) {
    // ------------------------------------------------------------ codes
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
        const bool in = tok < pc.it.q.len && lane < 4, there = in && (uint32_t)page < (uint32_t)p.num_pages;
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
                   p.pages + (int64_t)(page * p.H_KV + pc.it.h) * p.page_bytes + ((tok >> 4) & p.blocks_mask) * kBlockBytes, kBlockBytes, c_full + stage);
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
    uint32_t tile = 0, q_par = 0, ring = 0;      // tiles of this half and of the block so far
    bool ok = true;
    while (ok && pc.take(p)) {
      const int n_all = pc.t1 - pc.t0, first = pc.split() ? half : 0, step = pc.split() ? 2 : 1, n = (n_all - first + step - 1) / step;
      if (n > 0) {
        ok = wait_warp(q_full + half, q_par, abort_flag);
        q_par ^= 1u;
        int tq = 0;
        // a slot goes back when both halves have arrived; a half that has a tile to itself arrives twice
        auto hand_back = [&](uint64_t* bar) { tc::mma_commit(bar); if (step == 2) tc::mma_commit(bar); };
        auto qk = [&]() {
          const uint32_t at = ring + (uint32_t)(first + step * tq), ks = at % kKStages, slot = (tile + (uint32_t)tq) & 1u;
          ok = ok && wait_warp(k_full + ks, (at / kKStages) & 1u, abort_flag);
          if (!ok) return;
          tc::fence_after_sync();
          if (tc::elect_one()) {
            const uint32_t dS = tS + 64u * slot;
            const uint64_t bK = dK + (uint64_t)(ks * 1024);
#pragma unroll
            for (int k = 0; k < 8; ++k) tc::mma_bf16_ss(dS, dQ + (k >> 2) * 1024 + 2 * (k & 3), bK + (k >> 2) * 512 + 2 * (k & 3), idesc_qk, k > 0);
            hand_back(k_empty + ks);
            tc::mma_commit(s_full + 2 * half + slot);
          }
          __syncwarp();
          ++tq;
        };
        qk();
        if (n > 1) qk();
        for (int t = 0; ok && t < n; ++t) {
          const uint32_t at = ring + (uint32_t)(first + step * t), vs = at % kVStages, slot = (tile + (uint32_t)t) & 1u;
          ok = wait_warp(v_full + vs, (at / kVStages) & 1u, abort_flag) &&
               wait_warp(p_ready + 2 * half + slot, ((tile + (uint32_t)t) >> 1) & 1u, abort_flag);
          if (!ok) break;
          tc::fence_after_sync();
          if (tc::elect_one()) {
            const uint32_t aP = tS + 64u * slot;
            const uint64_t bV = dV + (uint64_t)(vs * 1024);
#pragma unroll
            for (int k = 0; k < 4; ++k) tc::mma_bf16_ts(tO, aP + 8 * k, bV + 128 * k, idesc_pv, (t > 0 || k > 0) ? 1u : 0u);
            hand_back(v_empty + vs);
            tc::mma_commit(pv_done + 2 * half + slot);
          }
          __syncwarp();
          if (t + 2 < n) qk();
        }
        tile += (uint32_t)n;
      }
      ring += (uint32_t)n_all;
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
    const Unpack uk = unpack_masks();
    int n_all = 0;
    while (pc.take(p)) { n_all += pc.t1 - pc.t0; pc.done(p); }
    int ks = 0, vs = 0;
    uint32_t kpar = 1u, vpar = 1u;               // empty barriers: the first round passes
    bool ok = true;
    uint32_t place[4];                           // of a row's four chunks under the 128-byte swizzle
#pragma unroll
    for (int k = 0; k < 4; ++k) place[k] = (quarter >> 1) * 8192 + (kTok * w + rowl) * 128 + (((((quarter & 1) << 2) + (k ^ turn)) ^ rowl) << 4);
    struct Codes { uint2 c[2][2]; __half2 s[2]; };
    auto read = [&](int stage, int kv) {
      const uint8_t* block = smem + TileSmem::Codes + stage * kCodeBytes + w * kBlockBytes;      // keys 16 w .. + 15
      const int info = key_rows[stage], rows = ((info >> (16 + w)) & 1) ? 0 : (info & 0xFFFF) - kTok * w;
      Codes x;
#pragma unroll
      for (int g = 0; g < 2; ++g) {              // keys 16 w + 8 g .. + 7
        const uint8_t* c = block + kv * kVOff + g * 512 + lane * 16;
        x.c[g][0] = *reinterpret_cast<const uint2*>(c + 4 * turn);
        x.c[g][1] = *reinterpret_cast<const uint2*>(c + 8 - 4 * turn);
        const uint16_t sb = *reinterpret_cast<const uint16_t*>(block + (kv ? kVsOff : kKsOff) + 2 * (8 * g + rowl));
        // keys that are not there: zeros, whatever lies here
        x.s[g] = __float2half2_rn(8 * g + rowl < rows ? __uint_as_float((uint32_t)sb << 16) : 0.f);
      }
      return x;
    };
    auto values = [&](const Codes& x, uint4 (&val)[2][4]) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        val[g][0] = values8(uk, x.c[g][0].x, x.s[g]); val[g][1] = values8(uk, x.c[g][0].y, x.s[g]);
        val[g][2] = values8(uk, x.c[g][1].x, x.s[g]); val[g][3] = values8(uk, x.c[g][1].y, x.s[g]);
      }
    };
    // K and V of a tile together: a question to a barrier costs some 100 clocks, a fence as much, and with K and V one after the other
    // they were 600 of a tile's 1500.  V has a slot more than K, so that K does not wait for a P V that is still to come.  The
    // values are in registers before their places are free.
#pragma unroll 1
    for (int tile = 0; tile < n_all; ++tile) {
      const int cs = tile % kAhead;
      ok = wait_warp(c_full + cs, (uint32_t)(tile / kAhead) & 1u, abort_flag);
      if (!ok) break;
      uint4 kval[2][4], vval[2][4];
      {
        const Codes kc = read(cs, 0), vc = read(cs, 1);
        values(kc, kval);
        values(vc, vval);
      }
      if (!__all_sync(0xffffffffu, mbar_test_wait(k_empty + ks, kpar) & mbar_test_wait(v_empty + vs, vpar))) {
        ok = wait_warp(k_empty + ks, kpar, abort_flag) && wait_warp(v_empty + vs, vpar, abort_flag);
        if (!ok) break;
      }
      uint8_t* k_to = smem + TileSmem::K + ks * 16384;
      uint8_t* v_to = smem + TileSmem::V + vs * 16384;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          *reinterpret_cast<uint4*>(k_to + place[k] + g * 1024) = kval[g][k];
          *reinterpret_cast<uint4*>(v_to + place[k] + g * 1024) = vval[g][k];
        }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) { tc::mbar_arrive(k_full + ks); tc::mbar_arrive(v_full + vs); tc::mbar_arrive(c_empty + cs); }
      if (++ks == kKStages) { ks = 0; kpar ^= 1u; }
      if (++vs == kVStages) { vs = 0; vpar ^= 1u; }
    }
  } else {
    // ------------------------------------------------------------ softmax: a thread per row
    const int half = warp >> 2, wq = warp & 3, r = wq * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(wq * 32) << 16), tO = lane_base + 256u + 128u * half;
    uint8_t* sQ = smem + TileSmem::Q + half * 32768;
    uint32_t tile = 0, all = 0;                  // tiles of this half and of the block so far
    bool ok = true;
    while (pc.take(p)) {
      const Request& q = pc.it.q;
      const bool split = pc.split();
      const int row0 = pc.it.qt * kRows + (split ? 0 : 128 * half), rows = min(128, q.nq * p.G - row0);
      const int n_all = pc.t1 - pc.t0, first = split ? half : 0, step = split ? 2 : 1, n = (n_all - first + step - 1) / step;
      const int row = row0 + r, i = token_of(p, row);
      const bool live = wq * 32 < rows;          // of the warp: one without rows only keeps the others' count
      float m = -INFINITY, l = 0.f;
      if (n > 0 && ok && !live) {
        tc::mbar_arrive(q_full + half);
#pragma unroll 1
        for (int t = 0; t < n && ok; ++t, ++tile) {
          ok = wait_warp(s_full + 2 * half + (tile & 1u), (tile >> 1) & 1u, abort_flag);
          tc::mbar_arrive(p_ready + 2 * half + (tile & 1u));
        }
      } else if (n > 0 && ok) {
        // queries: to their places in the operand tile, where each thread scales its row by a power of two so that fp16 holds it exactly
        const int chunk = lane & 15;
        const uint64_t from = r < rows ? (uint64_t)(reinterpret_cast<const uint16_t*>(p.q) + (int64_t)(q.q0 + i) * p.q_st +
                                                    (int64_t)(pc.it.h * p.G + row - i * p.G) * p.q_sh) : 0ull;
        const uint64_t any = __shfl_sync(0xffffffffu, from, 0);         // rows that are none are filled with zeros
        auto bring = [](uint32_t to, uint64_t at, bool there) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(at), "r"(there ? 16 : 0) : "memory");
        };
        auto place = [&](int row, int c) { return sQ + (c >> 3) * 16384 + row * 128 + (((c & 7) ^ (row & 7)) << 4); };
        // Sixteen lanes bring a row: a lane per row takes a line a lane, which eight warps wait for (64 new tokens of 32 heads over 8, 512 cached,
        // 25.7 us against 23.4; six chunks 144 and 136).  A single warp is quicker by itself (8 new tokens 17.4 us against 17.9).
        if (rows <= 32) {
#pragma unroll
          for (int c = 0; c < 16; ++c) bring(smem_u32(place(r, c)), (from ? from : any) + 16 * c, from != 0);
        } else {
#pragma unroll 4
          for (int k = 0; k < 16; ++k) {
            const int rr = 2 * k + (lane >> 4);
            const uint64_t at = __shfl_sync(0xffffffffu, from, rr);
            bring(smem_u32(place(wq * 32 + rr, chunk)), (at ? at : any) + 16 * chunk, at != 0);
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        uint32_t top2 = 0u;                      // magnitudes of 16-bit numbers order like integers
#pragma unroll 4
        for (int c = 0; c < 16; ++c) {
          const uint4 u = *reinterpret_cast<const uint4*>(place(r, c));
          top2 = __vmaxu2(__vmaxu2(__vmaxu2(top2, u.x & 0x7FFF7FFFu), u.y & 0x7FFF7FFFu), __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu));
        }
        auto value = [&](uint32_t u, int hi) {
          if (kBf16) return __uint_as_float(hi ? u & 0xFFFF0000u : u << 16);
          return __half2float(__ushort_as_half((unsigned short)(hi ? u >> 16 : u & 0xFFFFu)));
        };
        const float top = value(max(top2 & 0xFFFFu, top2 >> 16), 0);
        const int ex = (int)(__float_as_uint(top) >> 23), up = ex == 255 ? 0 : 140 - max(ex, 14);       // largest magnitude to [2^13, 2^14)
        const float scale = __uint_as_float((uint32_t)(127 + up) << 23), f = fminf(p.sml * __uint_as_float((uint32_t)(127 - up) << 23), 0x1.fffffep127f);
        const float2 scale2 = make_float2(scale, scale);
#pragma unroll 4
        for (int c = 0; c < 16; ++c) {
          const uint4 raw = *reinterpret_cast<const uint4*>(place(r, c));
          const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {          // channels k and k + 4 of the eight
            const float2 x = fmul2(make_float2(value(u[k >> 1], k & 1), value(u[2 + (k >> 1)], k & 1)), scale2);
            const __half2 hh = __floats2half2_rn(x.x, x.y);
            o[k] = *reinterpret_cast<const uint32_t*>(&hh);
          }
          *reinterpret_cast<uint4*>(place(r, c)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        fence_proxy_async_smem();
        tc::mbar_arrive(q_full + half);
        const int lim = r < rows ? min(q.len, q.past + 1 + i) : 0x7FFFFFFF;      // rows that are none see everything: finite, not written
        float shift = INFINITY;
        bool far = true;                         // no reference yet, or one whose rounding a weight would show: slow_tile
        const float2 f2 = make_float2(f, f);
#pragma unroll 1
        for (int t = 0; t < n; ++t, ++tile) {
          const uint32_t slot = tile & 1u;
          ok = wait_warp(s_full + 2 * half + slot, (tile >> 1) & 1u, abort_flag);
          if (!ok) break;
          tc::fence_after_sync();
          const uint32_t tS = lane_base + 128u * half + 64u * slot;
          const int at = first + step * t;
          const uint32_t bad = bads[(all + (uint32_t)at) & 15u];
          const int see = lim - (pc.t0 + at) * kKeys;
          const bool masks = __any_sync(0xffffffffu, see < kKeys || bad != 0u || far);
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
            far = m == -INFINITY || fabsf(m) * f > kTFar;
            shift = kTShift - m * f;
          } else {
            l += sum;
            tc::tmem_st32(tS, pk);
            tc::tmem_wait_st();
          }
          tc::fence_before_sync();
          tc::mbar_arrive(p_ready + 2 * half + slot);
        }
        if (ok) ok = wait_warp(pv_done + 2 * half + ((tile - 1u) & 1u), ((tile - 1u) >> 1) & 1u, abort_flag);
        if (m != -INFINITY) m *= f;              // the score, for the other half and other blocks
      }
      all += (uint32_t)n_all;
      if (!ok) { m = 0.f; l = __int_as_float(0x7FC00000); }            // gave up: the rows are NaN
      // weights of this half's O and of the other's, where both have some
      float wa = n > 0 && ok ? 1.f : 0.f, wb = 0.f;
      const bool other = split && n_all > 1;     // (a half without tiles has no O)
      if (split) {
        s_state[half][r] = make_float2(m, l);
        tc::fence_before_sync();
        halves_meet();
        const float2 o = s_state[half ^ 1][r];
        const float M = fmaxf(m, o.x), ref = M == -INFINITY ? 0.f : M;
        wa = ex2f(m - ref); wb = ex2f(o.x - ref);
        l = l * wa + o.y * wb;
        m = M;
        if (l != l) { wa = l; wb = l; }
      }
      tc::fence_after_sync();
      if (live) {
        // O leaves through the rows' own part of the query tile, 32 columns at a time, so that a store writes whole sectors.  Halves
        // that share their rows take two of the four parts each.
        const bool whole = !pc.began && pc.ends;
        const float inv = l == 0.f ? 0.f : 1.f / l, fa = whole ? wa * inv : wa, fb = whole ? wb * inv : wb;
        float* piece = p.ws + (int64_t)(2 * block + (pc.began ? 0 : 1)) * piece_floats;
        const int prow0 = row0 - pc.it.qt * kRows;
        uint8_t* stage = sQ + wq * 32 * 128;     // of the first half of the channels: 4 KB that only this warp touches
        const uint32_t tOther = lane_base + 256u + 128u * (half ^ 1);
#pragma unroll 1
        for (int ch = split ? 2 * half : 0; ch < (split ? 2 * half + 2 : 4); ++ch) {
          float o[32];
          if (split ? (half == 0 || other) : n > 0) {
            tc::tmem_ld32(tO + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
            tc::tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
          if (n_all == 0) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= fa;
          if (split && n_all > (half == 0 ? 1 : 0)) {
            float o2[32];
            tc::tmem_ld32(tOther + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(&o2[0]));
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fmaf(o2[e], fb, o[e]);
          }
          __syncwarp();
          // column 8 k + 2 j + b holds channel 8 k + 4 b + j
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = o[8 * k + 2 * j]; v[4 + j] = o[8 * k + 2 * j + 1]; }
            if (whole) {
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
#pragma unroll 4
            for (int rr = lane >> 2; rr < 32; rr += 8) {
              if (wq * 32 + rr >= rows) break;
              const int part = lane & 3, orow = row0 + wq * 32 + rr, gi = token_of(p, orow);
              *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + (int64_t)(q.q0 + gi) * p.o_st +
                                        (int64_t)(pc.it.h * p.G + orow - gi * p.G) * p.o_sh + ch * 32 + part * 8) =
                  *reinterpret_cast<const uint4*>(stage + rr * 128 + ((part ^ (rr & 7)) << 4));
            }
          } else {                               // eight lanes a row, 128 bytes
#pragma unroll 2
            for (int rr = lane >> 3; rr < 32 && wq * 32 + rr < rows; rr += 4) {
              const int part = lane & 7;
              *reinterpret_cast<float4*>(piece + (int64_t)(prow0 + wq * 32 + rr) * 128 + ch * 32 + part * 4) =
                  *reinterpret_cast<const float4*>(stage + rr * 128 + ((part ^ (rr & 7)) << 4));
            }
          }
          __syncwarp();
        }
        if (!whole && r < rows && !(split && half)) {
          piece[(int64_t)piece_rows * 128 + prow0 + r] = m;
          piece[(int64_t)piece_rows * 129 + prow0 + r] = l;
        }
      }
      if (split) { tc::fence_before_sync(); halves_meet(); }           // the other half has read this one's O and state
      if (pc.began && pc.ends && tid == 0) {
        const int start = b0 - pc.it.u;    // where the query tile begins: the block of that position has its first piece
        *todo = TileMerge{q.q0, min(kRows, q.nq * p.G - pc.it.qt * kRows), pc.it.h, pc.it.qt, cuts.block_of(start), 1, {0, 0}};
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
  const int grow = todo.qt * kRows + row, gi = token_of(p, grow);
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

// Rows of a piece: as many as a query tile of the call has, an even number: a row is 130 floats, and pieces, which are moved in
// 16-byte parts, lie one behind the other.
static int piece_rows_of(const AttnParams& p) { return (int)min((int64_t)kRows, ((int64_t)p.max_q_len * p.G + 1) & ~(int64_t)1); }

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
