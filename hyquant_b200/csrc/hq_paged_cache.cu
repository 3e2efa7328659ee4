// The paged 4-bit cache's bookkeeping (page_advance), its quantising write and the reading back of rows.
#include "hq_paged.cuh"

#include <type_traits>

namespace hq {
namespace paged {

// ---------------------------------------------------------------------------------------------- block tables and slot maps
// Latency-bound: a few KB in all, dependent steps.  One block (or, for many tokens, one cluster of eight whose blocks share
// the moves and the slots and each do the scans again): per request the tokens added and the pages taken and given back,
// three prefix sums, the verdict, then the moves and the slots spread evenly over the threads, an entry's request found by a
// search in shared memory.  Pages that are given back go onto the stack before pages are taken from it.
struct AdvanceParams {
  const int* kv_lens; const int* held; const int* add; const int* keep;
  int R;
  int* table; int64_t table_stride; int max_pages;
  int* free_pages; int free_cap; const int* free_count;
  int page_shift, T;
  int* kv_out; int* held_out; int* count_out; int* cu_q; int64_t* slots; int* positions; int* status;
};
constexpr int kAdvThreads = 1024;
constexpr int kAdvMostR = 8192;
// From 12288 rows of slots on, eight blocks: 8192 rows took 6.2 us with one and 6.7 with eight, 16384 8.9 and 7.5, 65536 21.0 and
// 8.7 (500 requests; four blocks 10.5).  Below, the cluster's launch and its barriers cost more than they save: 512 rows 4.2 and 5.7.
constexpr int kAdvBlocks = 8, kAdvMany = 12288;

__device__ __forceinline__ void adv_sync(bool cluster) {
  if (cluster) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  else __syncthreads();
}
// the largest r in [0, R) with a[r] <= x, for a[0] = 0 and x >= 0
__device__ __forceinline__ int adv_find(const int* a, int R, int x) {
  int lo = 0, hi = R;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kAdvThreads)
advance_kernel(const AdvanceParams p, int blocks) {
  extern __shared__ int sm[];
  int* s_cu = sm;                       // [R + 1] prefix sums: tokens added,
  int* s_more = s_cu + p.R + 1;         // pages taken,
  int* s_back = s_more + p.R + 1;       // pages given back
  int* s_keep = s_back + p.R + 1;       // [R]
  int* s_held = s_keep + p.R;           // [R]
  __shared__ long long w_add[33];
  __shared__ int w_more[33], w_back[33], s_bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = p.R;
  const int page = 1 << p.page_shift;
  const bool cluster = blocks > 1;
  if (tid == 0) s_bad = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __syncthreads();
  const int free_count = *p.free_count;
  const int per = (R + kAdvThreads - 1) / kAdvThreads, r0 = min(R, tid * per), r1 = min(R, r0 + per);
  long long add_sum = 0;
  int more_sum = 0, back_sum = 0, bad = 0;
  for (int r = r0; r < r1; ++r) {
    const int kv = p.kv_lens[r], held = p.held[r], add = p.add[r], keep = p.keep ? p.keep[r] : kv;
    const long long target = (long long)keep + add;
    if (kv < 0 || add < 0 || keep < 0 || keep > kv || held < 0 || held > p.max_pages || (((long long)kv + page - 1) >> p.page_shift) > held) bad |= 8;
    if (((target + page - 1) >> p.page_shift) > p.max_pages || target > 0x7FFFFFFF) bad |= 2;
    int more = 0, back = 0;
    if (!bad) {
      const int need = (int)((target + page - 1) >> p.page_shift);
      more = max(0, need - held); back = max(0, held - need);
    }
    s_keep[r] = keep; s_held[r] = held;
    s_cu[r] = add; s_more[r] = more; s_back[r] = back;      // turned into prefix sums below, by the same thread
    add_sum += bad ? 0 : add; more_sum += more; back_sum += back;
  }
  // block-wide exclusive scan of the three sums
  long long a = add_sum;
  int m = more_sum, b = back_sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long ta = __shfl_up_sync(0xffffffffu, a, o);
    const int tm = __shfl_up_sync(0xffffffffu, m, o), tb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) { a += ta; m += tm; b += tb; }
  }
  if (lane == 31) { w_add[warp] = a; w_more[warp] = m; w_back[warp] = b; }
  if (bad) atomicOr(&s_bad, bad);
  __syncthreads();
  if (warp == 0) {
    long long xa = w_add[lane];
    int xm = w_more[lane], xb = w_back[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long ta = __shfl_up_sync(0xffffffffu, xa, o);
      const int tm = __shfl_up_sync(0xffffffffu, xm, o), tb = __shfl_up_sync(0xffffffffu, xb, o);
      if (lane >= o) { xa += ta; xm += tm; xb += tb; }
    }
    const long long pa = __shfl_up_sync(0xffffffffu, xa, 1);
    const int pm = __shfl_up_sync(0xffffffffu, xm, 1), pb = __shfl_up_sync(0xffffffffu, xb, 1);
    w_add[lane] = lane ? pa : 0; w_more[lane] = lane ? pm : 0; w_back[lane] = lane ? pb : 0;
    if (lane == 31) { w_add[32] = xa; w_more[32] = xm; w_back[32] = xb; }
  }
  __syncthreads();
  const long long total_add = w_add[32];
  const int total_more = w_more[32], total_back = w_back[32];
  int why = s_bad;
  if (why == 0) {
    if (total_add > p.T) why |= 4;
    if (free_count < 0 || (long long)free_count + total_back > p.free_cap) why |= 8;
    else if (total_more > free_count + total_back) why |= 1;
  }
  const int stride = blocks * kAdvThreads, at = blockIdx.x * kAdvThreads + tid;
  if (why) {
    // every block has read the inputs before any writes an output that may be one of them
    adv_sync(cluster);
    for (int t = at; t < p.T; t += stride) { p.slots[t] = -1; p.positions[t] = 0; }
    if (blockIdx.x == 0) {
      for (int r = tid; r < R; r += kAdvThreads) {
        p.cu_q[r] = 0;
        const int kv = p.kv_lens[r], held = p.held[r];
        p.kv_out[r] = kv; p.held_out[r] = held;
      }
      if (tid == 0) { p.cu_q[R] = 0; *p.count_out = free_count; *p.status = why; }
    }
    return;
  }
  {
    int ea = (int)(w_add[warp] + (a - add_sum)), em = w_more[warp] + m - more_sum, eb = w_back[warp] + b - back_sum;
    for (int r = r0; r < r1; ++r) {
      const int x = s_cu[r], y = s_more[r], z = s_back[r];
      s_cu[r] = ea; s_more[r] = em; s_back[r] = eb;
      ea += x; em += y; eb += z;
    }
    if (tid == kAdvThreads - 1) { s_cu[R] = (int)total_add; s_more[R] = total_more; s_back[R] = total_back; }
  }
  adv_sync(cluster);
  if (blockIdx.x == 0) {
    for (int r = tid; r < R; r += kAdvThreads) {
      const int add = s_cu[r + 1] - s_cu[r];
      p.cu_q[r] = s_cu[r];
      p.kv_out[r] = s_keep[r] + add;
      p.held_out[r] = s_held[r] + (s_more[r + 1] - s_more[r]) - (s_back[r + 1] - s_back[r]);
    }
    if (tid == 0) {
      p.cu_q[R] = (int)total_add;
      *p.count_out = free_count + total_back - total_more;
      *p.status = 0;
    }
  }
  if (total_back > 0) {
    for (int i = at; i < total_back; i += stride) {
      const int r = adv_find(s_back, R, i), need = s_held[r] - (s_back[r + 1] - s_back[r]);
      p.free_pages[free_count + i] = p.table[r * p.table_stride + need + (i - s_back[r])];
    }
    adv_sync(cluster);
  }
  if (total_more > 0) {
    const int top = free_count + total_back - 1;
    for (int i = at; i < total_more; i += stride) {
      const int r = adv_find(s_more, R, i);
      p.table[r * p.table_stride + s_held[r] + (i - s_more[r])] = p.free_pages[top - i];
    }
    adv_sync(cluster);
  }
  for (int t = at; t < p.T; t += stride) {
    int64_t slot = -1;
    int pos = 0;
    if (t < (int)total_add) {
      const int r = adv_find(s_cu, R, t);
      pos = s_keep[r] + (t - s_cu[r]);
      slot = ((int64_t)p.table[r * p.table_stride + (pos >> p.page_shift)] << p.page_shift) + (pos & (page - 1));
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
  }
}

// ---------------------------------------------------------------------------------------------- rows in, rows out
// HBM-bound: 256 bytes a 16-bit row read, 66 written, or the other way round.  Eight lanes take the K row and the V row of one token
// and head, so that two rows' loads are in flight per lane; a lane has channels 8 sub .. + 7 and 64 + 8 sub .. + 7, so that an
// instruction moves whole lines (thirty-two bytes a lane in one piece: every line took two instructions, 17.1 and 19.9 us below).
// 12289 tokens of eight heads, in and out: bf16 and fp16 14.2 and 9.9 us, fp32 19.1 and 30.2; one behind the other in fp16 24.7, where
// their 127 MB at a copy's rate take 19.4.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* v) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}
__device__ __forceinline__ void load8(const __half* p, float* v) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float* v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
    v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
append_kernel(const T* __restrict__ k, const T* __restrict__ v, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, int n, int H,
              const int64_t* __restrict__ slots, uint8_t* __restrict__ pages, int64_t num_slots, int page_shift) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const int64_t rows = (int64_t)n * H, warps = (int64_t)gridDim.x * 8;
  for (int64_t r0 = 4 * ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)); r0 < rows; r0 += 4 * warps) {
    const int64_t mine = r0 + (lane >> 3), r = min(mine, rows - 1);       // groups past the end redo the last row and store nothing
    const int t = (int)((uint32_t)r / (uint32_t)H), h = (int)(r - (int64_t)t * H);
    const int64_t slot = __ldg(slots + t);
    float x[16], y[16];
    const T* kr = k + t * k_st + h * k_sh + 8 * sub;
    const T* vr = v + t * v_st + h * v_sh + 8 * sub;
    load8(kr, x); load8(kr + 64, x + 8);
    load8(vr, y); load8(vr + 64, y + 8);
    uint32_t ck[2], cv[2];
    const float ks = quant_row(x, ck), vs = quant_row(y, cv);
    if (mine < rows && slot >= 0 && slot < num_slots) {
      uint8_t* block = pages + block_offset(slot, h, H, page_shift);
      const int row = (int)(slot & (kTok - 1));
      uint32_t* to = reinterpret_cast<uint32_t*>(block + row * 64) + sub;
      to[0] = ck[0]; to[8] = ck[1];
      to += kVOff / 4;
      to[0] = cv[0]; to[8] = cv[1];
      if (sub < 2)
        *reinterpret_cast<uint16_t*>(block + (sub ? kVsOff : kKsOff) + 2 * row) = (uint16_t)(__float_as_uint(sub ? vs : ks) >> 16);
    }
  }
}

// eight values, in pairs (0 4) (1 5) (2 6) (3 7) as they are unpacked, to channels 0 .. 7
__device__ __forceinline__ void store8(__half* p, uint4 v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(prmt(v.x, v.y, 0x5410u), prmt(v.z, v.w, 0x5410u), prmt(v.x, v.y, 0x7632u), prmt(v.z, v.w, 0x7632u));
}
__device__ __forceinline__ void floats8(uint4 v, float2 (&f)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, uint4 v) {
  float2 f[4];
  floats8(v, f);
  const __nv_bfloat162 h[4] = {__floats2bfloat162_rn(f[0].x, f[1].x), __floats2bfloat162_rn(f[2].x, f[3].x), __floats2bfloat162_rn(f[0].y, f[1].y),
                               __floats2bfloat162_rn(f[2].y, f[3].y)};
  const uint32_t* w = reinterpret_cast<const uint32_t*>(h);
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(float* p, uint4 v) {
  float2 f[4];
  floats8(v, f);
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0].x, f[1].x, f[2].x, f[3].x);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[0].y, f[1].y, f[2].y, f[3].y);
}

template <typename T>
__global__ void __launch_bounds__(256)
read_kernel(const uint8_t* __restrict__ pages, int64_t num_slots, int page_shift, const int64_t* __restrict__ slots, int n, int H,
            T* __restrict__ k, T* __restrict__ v) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const int64_t rows = (int64_t)n * H, step = (int64_t)gridDim.x * 32;
  const Unpack u = unpack_masks();
  for (int64_t r = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3); r < rows; r += step) {
    const int t = (int)((uint32_t)r / (uint32_t)H), h = (int)(r - (int64_t)t * H);
    const int64_t slot = __ldg(slots + t);
    uint32_t c[4] = {0u, 0u, 0u, 0u};
    float ks = 0.f, vs = 0.f;
    if (slot >= 0 && slot < num_slots) {
      const uint8_t* block = pages + block_offset(slot, h, H, page_shift);
      const int row = (int)(slot & (kTok - 1));
      const uint32_t* from = reinterpret_cast<const uint32_t*>(block + row * 64) + sub;
      c[0] = __ldg(from); c[1] = __ldg(from + 8); c[2] = __ldg(from + kVOff / 4); c[3] = __ldg(from + kVOff / 4 + 8);
      ks = __uint_as_float((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(block + kKsOff) + row) << 16);
      vs = __uint_as_float((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(block + kVsOff) + row) << 16);
    }
    const __half2 k2 = __float2half2_rn(ks), v2 = __float2half2_rn(vs);
    T* kr = k + r * 128 + 8 * sub;
    T* vr = v + r * 128 + 8 * sub;
    store8(kr, values8(u, c[0], k2)); store8(kr + 64, values8(u, c[1], k2));
    store8(vr, values8(u, c[2], v2)); store8(vr + 64, values8(u, c[3], v2));
  }
}

static int shift_of(int page_size) { return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7; }

// A launch that the kernel before it in the stream lets begin early: the kernels wait for it (griddepcontrol.wait) before they touch
// memory, but their launch is over by then (rows of 16 tokens in and out 3.8 -> 3.4 us).  Of these only page_advance lets the next one
// begin early in turn, as attention does, and behind its own wait: what comes next may rely on every kernel but the one just before it
// (hq_decode_splitk does, which fetches older rows of its cache at once).  Blocks of read_kernel that wait beside append_kernel's took
// 29.3 us for a prompt's rows, not 24.8.
template <typename... P, typename... A>
static cudaError_t launch_early(void (*kernel)(P...), int grid, int cluster, int threads, int smem, cudaStream_t st, A... a) {
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, P(a)...);
}

static int row_grid(int64_t rows) {
  const int64_t want = (rows + 31) / 32, cap = (int64_t)sm_count() * 4;
  return (int)(want < cap ? want : cap);
}

}  // namespace paged
}  // namespace hq

extern "C" int hq_page_advance(const hq_page_advance_args* a, void* stream) {
  using namespace hq;
  using namespace hq::paged;
  HQ_REQUIRE(a != nullptr, HQ_ERR_INVALID, "hq_page_advance: null argument block");
  HQ_REQUIRE(a->struct_bytes == (int)sizeof(hq_page_advance_args), HQ_ERR_INVALID, "hq_page_advance: struct_bytes %d, expected %d", a->struct_bytes,
             (int)sizeof(hq_page_advance_args));
  HQ_REQUIRE(a->R >= 0 && a->T >= 0 && a->max_pages >= 0 && a->free_cap >= 0, HQ_ERR_INVALID, "hq_page_advance: negative size");
  HQ_REQUIRE(a->R <= kAdvMostR, HQ_ERR_UNSUPPORTED, "hq_page_advance: %d requests, at most %d", a->R, kAdvMostR);
  HQ_REQUIRE(page_size_ok(a->page_size), HQ_ERR_UNSUPPORTED, "hq_page_advance: page_size must be 16, 32, 64 or 128, got %d", a->page_size);
  HQ_REQUIRE(a->free_count && a->free_count_out && a->cu_q && a->status && (a->T == 0 || (a->slots && a->positions)), HQ_ERR_INVALID,
             "hq_page_advance: null pointer");
  HQ_REQUIRE(a->R == 0 || (a->kv_lens && a->held && a->add && a->kv_lens_out && a->held_out), HQ_ERR_INVALID, "hq_page_advance: null pointer");
  HQ_REQUIRE((a->R == 0 || a->max_pages == 0 || a->page_table) && (a->free_cap == 0 || a->free_pages), HQ_ERR_INVALID, "hq_page_advance: null pointer");
  HQ_REQUIRE((int64_t)a->R * a->max_pages <= 0x7FFFFFFF, HQ_ERR_UNSUPPORTED, "hq_page_advance: %d requests of %d pages", a->R, a->max_pages);
  HQ_REQUIRE(a->table_stride >= a->max_pages, HQ_ERR_INVALID, "hq_page_advance: table rows of %d pages overlap at stride %lld", a->max_pages,
             (long long)a->table_stride);
  const auto bits = [](auto*... p) { return (... | (uintptr_t)p); };
  HQ_REQUIRE(bits(a->kv_lens, a->held, a->add, a->keep, a->page_table, a->free_pages, a->free_count, a->kv_lens_out, a->held_out, a->free_count_out,
                  a->cu_q, a->positions, a->status) % 4 == 0 && (uintptr_t)a->slots % 8 == 0, HQ_ERR_ALIGNMENT,
             "hq_page_advance: slots must be 8-byte, the other arrays 4-byte aligned");
  const AdvanceParams p{a->kv_lens, a->held, a->add, a->keep, a->R, a->page_table, a->table_stride, a->max_pages, a->free_pages, a->free_cap,
                        a->free_count, shift_of(a->page_size), a->T, a->kv_lens_out, a->held_out, a->free_count_out, a->cu_q, a->slots,
                        a->positions, a->status};
  const int smem = (5 * a->R + 3) * (int)sizeof(int);
  static thread_local int attr_dev = -1;
  int dev = 0;
  HQ_CUDA(cudaGetDevice(&dev));
  if (attr_dev != dev) {
    HQ_CUDA(cudaFuncSetAttribute(advance_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (5 * kAdvMostR + 3) * (int)sizeof(int)));
    attr_dev = dev;
  }
  const int blocks = a->T >= kAdvMany ? kAdvBlocks : 1;
  HQ_CUDA(launch_early(advance_kernel, blocks, blocks, kAdvThreads, smem, (cudaStream_t)stream, p, blocks));
  return HQ_OK;
}

namespace hq {
namespace paged {
static int check_pool(const char* what, const void* pages, int64_t num_pages, int page_size, const int64_t* slots, int T, int H_KV) {
  HQ_REQUIRE(T >= 0 && H_KV >= 1 && num_pages >= 0, HQ_ERR_INVALID, "%s: bad size", what);
  HQ_REQUIRE(page_size_ok(page_size), HQ_ERR_UNSUPPORTED, "%s: page_size must be 16, 32, 64 or 128, got %d", what, page_size);
  HQ_REQUIRE((int64_t)T * H_KV <= 0x7FFFFFFF, HQ_ERR_UNSUPPORTED, "%s: %d tokens of %d heads are too many rows for one call", what, T, H_KV);
  HQ_REQUIRE(T == 0 || (slots && (pages || num_pages == 0)), HQ_ERR_INVALID, "%s: null pointer", what);
  HQ_REQUIRE(aligned16(pages) && (uintptr_t)slots % 8 == 0, HQ_ERR_ALIGNMENT, "%s: pages must be 16-byte, slots 8-byte aligned", what);
  return HQ_OK;
}
}  // namespace paged
}  // namespace hq

extern "C" int hq_paged_append(const void* k, const void* v, int dtype, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, int T,
                               int H_KV, const int64_t* slots, void* pages, int64_t num_pages, int page_size, void* stream) {
  using namespace hq;
  using namespace hq::paged;
  if (int rc = check_pool("hq_paged_append", pages, num_pages, page_size, slots, T, H_KV)) return rc;
  HQ_REQUIRE(dtype == HQ_BF16 || dtype == HQ_F16 || dtype == HQ_F32, HQ_ERR_UNSUPPORTED, "hq_paged_append: unknown dtype %d", dtype);
  if (T == 0 || num_pages == 0) return HQ_OK;
  HQ_REQUIRE(k && v, HQ_ERR_INVALID, "hq_paged_append: null pointer");
  HQ_REQUIRE(aligned16(k) && aligned16(v) && (k_st | k_sh | v_st | v_sh) % 8 == 0, HQ_ERR_ALIGNMENT,
             "hq_paged_append: rows must be 16-byte aligned (strides multiples of 8 elements)");
  auto go = [&](auto* rows) {
    using X = std::remove_pointer_t<decltype(rows)>;
    return launch_early(append_kernel<X>, row_grid((int64_t)T * H_KV), 1, 256, 0, (cudaStream_t)stream, (const X*)k, (const X*)v, k_st, k_sh, v_st,
                        v_sh, T, H_KV, slots, (uint8_t*)pages, num_pages * page_size, shift_of(page_size));
  };
  HQ_CUDA(dtype == HQ_BF16 ? go((__nv_bfloat16*)nullptr) : dtype == HQ_F16 ? go((__half*)nullptr) : go((float*)nullptr));
  return HQ_OK;
}

extern "C" int hq_paged_read(const void* pages, int64_t num_pages, int page_size, const int64_t* slots, int T, int H_KV, int dtype, void* k,
                             void* v, void* stream) {
  using namespace hq;
  using namespace hq::paged;
  if (int rc = check_pool("hq_paged_read", pages, num_pages, page_size, slots, T, H_KV)) return rc;
  HQ_REQUIRE(dtype == HQ_BF16 || dtype == HQ_F16 || dtype == HQ_F32, HQ_ERR_UNSUPPORTED, "hq_paged_read: unknown dtype %d", dtype);
  if (T == 0) return HQ_OK;
  HQ_REQUIRE(k && v, HQ_ERR_INVALID, "hq_paged_read: null pointer");
  HQ_REQUIRE(aligned16(k) && aligned16(v), HQ_ERR_ALIGNMENT, "hq_paged_read: k and v must be 16-byte aligned");
  auto go = [&](auto* rows) {
    using X = std::remove_pointer_t<decltype(rows)>;
    return launch_early(read_kernel<X>, row_grid((int64_t)T * H_KV), 1, 256, 0, (cudaStream_t)stream, (const uint8_t*)pages, num_pages * page_size,
                        shift_of(page_size), slots, T, H_KV, (X*)k, (X*)v);
  };
  HQ_CUDA(dtype == HQ_BF16 ? go((__nv_bfloat16*)nullptr) : dtype == HQ_F16 ? go((__half*)nullptr) : go((float*)nullptr));
  return HQ_OK;
}
