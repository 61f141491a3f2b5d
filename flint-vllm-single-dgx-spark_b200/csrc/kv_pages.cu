// Pages of the KV cache shared between streams: reserving, forking, freeing and compacting them on the device.
//
// The cache of all layers is one bf16 tensor [layers, blocks, kv_heads, 16, 256]; a page is block p of every layer.  The
// pool's state is whole numbers in device memory: ref[p], the number of streams that hold page p (0: free); block_tables
// [streams, max_blocks], -1 behind a stream's pages; num_pages[s] and seq_lens[s].  Pages are taken from the lowest free
// ids, in the order of the call's streams, so the result follows from the state alone.  Nothing is read back by the host:
// a request that does not fit is left out and recorded in the status word.
//
// A call that needs free pages is planned by one block: each thread counts the free ids of its own contiguous share of
// ref, one scan over the block turns the counts into ranks, and a second walk hands the ids out by rank.  The state is
// small (4 bytes a page); what costs is the copying, which a second launch spreads over all SMs: 16-byte loads and stores,
// a page of a layer (8 KB a KV head) to a block at a time.
//
// Measured: 386 pages of a pool of 1,536 moved in 48 layers (1.21 GB read and written) 219 us, 5.5 TB/s or 85% of the copy
// rate.  40 of 64 streams on a 6,057-token prompt freed and forked anew in 48 layers, 27 of them with a started page, and pages
// reserved for all: free 3.5, fork 17.1, reserve 5.8 us on the device (27 pages written and 5 read take 7.7).  A small call takes
// 2 to 4 us a launch on the device and 8 to 13 us of host time.
#include "common.cuh"
#include "runtime.cuh"
#include "tma.cuh"

namespace flint {

constexpr int kPgPage = 16;
constexpr int kPgT = 1024;                       // threads of the planning block
constexpr int kPgMaxRequests = 4096;             // streams of a call (and of a pool)
constexpr int kPgPer = kPgMaxRequests / kPgT;    // requests a planning thread holds
constexpr unsigned STATUS_BAD_STREAM = 4u;       // a stream id, length, page or table that does not fit
constexpr unsigned STATUS_NO_PAGES = 8u;

struct KvPagesWorkspace {
  unsigned status;
  int moves;                                     // compact: pages to move
  unsigned pad[30];
};
// behind it the plan: fork -- int4 (from row, to row, tokens, started page taken from) and int (its copy) per request;
// compact -- int2 (from, to) per move

struct KvPool {
  int* ref;
  int blocks;
  int* tables;
  int64_t bt_stride;
  int max_blocks;
  int* seq_lens;
  int* num_pages;
  int streams;
  KvPagesWorkspace* ws;
};

__device__ __forceinline__ int4* pg_fork_plan(const KvPool& p) { return reinterpret_cast<int4*>(p.ws + 1); }
__device__ __forceinline__ int* pg_fork_tail(const KvPool& p) { return reinterpret_cast<int*>(pg_fork_plan(p) + kPgMaxRequests); }
__device__ __forceinline__ int2* pg_moves(const KvPool& p) { return reinterpret_cast<int2*>(p.ws + 1); }

// Kernels that follow may look at tables, lengths and old pages before their wait on this grid (the decode attention does):
// they are started when its last block ends, so each block ends with its writes in place.
__device__ __forceinline__ void pg_publish() { __threadfence(); }

// The sum of v over the planning block and, in *before, over the threads ahead of this one.
__device__ __forceinline__ int pg_scan(int v, int* before, int* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                               // red of an earlier scan has been read
  if (lane == 31) red[warp] = x;
  __syncthreads();
  int t = red[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) t += y;
  }
  const int base = __shfl_sync(0xffffffffu, t, warp) - __shfl_sync(0xffffffffu, red[lane], warp);
  *before = base + x - v;
  return __shfl_sync(0xffffffffu, t, 31);
}
static_assert(kPgT == 32 * 32, "one lane per warp sum");

// The ids [lo, hi) of ref that this thread of the planning block walks.
struct PgShare {
  int lo, hi;
};
__device__ __forceinline__ PgShare pg_share(int blocks) {
  const int per = (blocks + kPgT - 1) / kPgT;
  const long long lo = (long long)threadIdx.x * per;
  return {(int)(lo < blocks ? lo : blocks), (int)(lo + per < blocks ? lo + per : blocks)};
}
__device__ __forceinline__ int pg_count_free(const KvPool& p, PgShare sh) {
  int n = 0;
  for (int id = sh.lo; id < sh.hi; ++id) n += p.ref[id] == 0;
  return n;
}

// First naming of each stream in `ids` (claim[] holds kPgMaxRequests ints of shared memory): claim[s] = its place.
__device__ __forceinline__ void pg_claim(const int* ids, int n, int streams, int* claim) {
  for (int i = threadIdx.x; i < kPgMaxRequests; i += kPgT) claim[i] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPgT)
    if (ids[i] >= 0 && ids[i] < streams) atomicMin(&claim[ids[i]], i);
  __syncthreads();
}

__global__ void __launch_bounds__(256) kv_free_kernel(const KvPool p, const int* streams) {
  __shared__ int s_n;
  pdl_wait();
  const int s = streams[blockIdx.x];
  if (s < 0 || s >= p.streams) {
    if (threadIdx.x == 0) atomicOr(&p.ws->status, STATUS_BAD_STREAM);
    return;
  }
  if (threadIdx.x == 0) {
    s_n = min(atomicExch(&p.num_pages[s], 0), p.max_blocks);      // a stream named twice is freed once
    p.seq_lens[s] = 0;
  }
  __syncthreads();
  int* row = p.tables + (int64_t)s * p.bt_stride;
  for (int i = threadIdx.x; i < s_n; i += 256) {
    const int page = row[i];
    row[i] = -1;
    if (page < 0 || page >= p.blocks) {
      atomicOr(&p.ws->status, STATUS_BAD_STREAM);
    } else if (atomicSub(&p.ref[page], 1) <= 0) {                 // it was free already
      atomicAdd(&p.ref[page], 1);
      atomicOr(&p.ws->status, STATUS_BAD_STREAM);
    }
  }
  pg_publish();
}

// One block.  Stream streams[i] gets pages up to lens[i] tokens; a demand beyond the free pages is refused whole.
__global__ void __launch_bounds__(kPgT) kv_reserve_kernel(const KvPool p, const int* streams, const int* lens, int n) {
  __shared__ int red[32], start[kPgMaxRequests], s_limit;
  extern __shared__ int claim[];                                  // reused for the requests' first new column
  pdl_wait();
  pg_claim(streams, n, p.streams, claim);
  int sid[kPgPer], need[kPgPer], have[kPgPer], mine = 0;
#pragma unroll
  for (int j = 0; j < kPgPer; ++j) {
    const int i = threadIdx.x * kPgPer + j;
    sid[j] = -1, need[j] = 0, have[j] = 0;
    if (i >= n) continue;
    const int s = streams[i], len = lens[i];
    const int want = len / kPgPage + (len % kPgPage != 0);
    if (s < 0 || s >= p.streams || claim[s] != i || len < 0 || want > p.max_blocks || p.num_pages[s] < 0) {
      atomicOr(&p.ws->status, STATUS_BAD_STREAM);
      continue;
    }
    sid[j] = s, have[j] = p.num_pages[s], need[j] = max(0, want - have[j]);
    mine += need[j];
  }
  int at;
  pg_scan(mine, &at, red);                                        // fits 32 bits: n * max_blocks is checked on the host
  if (threadIdx.x == 0) s_limit = 0;
  const PgShare sh = pg_share(p.blocks);
  int rank;
  const int n_free = pg_scan(pg_count_free(p, sh), &rank, red);
#pragma unroll
  for (int j = 0; j < kPgPer; ++j) {
    const int i = threadIdx.x * kPgPer + j;
    start[i] = at;                                                // ranks of the free pages that request i takes
    claim[i] = have[j];
    at += need[j];
    if (!need[j]) continue;
    if (at > n_free) {
      atomicOr(&p.ws->status, STATUS_NO_PAGES);
    } else {
      atomicMax(&s_limit, at);                                    // demands add up, so those met are the first ones
      p.num_pages[sid[j]] = have[j] + need[j];
    }
  }
  __syncthreads();
  const int limit = s_limit;
  for (int id = sh.lo; id < sh.hi && rank < limit; ++id) {
    if (p.ref[id] != 0) continue;
    int lo = 0, hi = kPgMaxRequests - 1;                          // the last request that starts at or before this rank
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= rank) lo = mid; else hi = mid - 1;
    }
    p.tables[(int64_t)streams[lo] * p.bt_stride + claim[lo] + (rank - start[lo])] = id;
    p.ref[id] = 1;
    ++rank;
  }
  pg_publish();
}

// One block.  Checks the forks, takes a page for each tail and writes the plan of the copies.  (The ids of the source's full
// pages are checked by the block that copies them, which is what makes the child: here they would cost a walk of every row.)
__global__ void __launch_bounds__(kPgT) kv_fork_plan_kernel(const KvPool p, const int* src, const int* dst, int n) {
  __shared__ int red[32], fresh[kPgMaxRequests];
  extern __shared__ int claim[];
  pdl_trigger();                                                  // the copying launch may line up
  pdl_wait();
  pg_claim(dst, n, p.streams, claim);
  int len[kPgPer], last[kPgPer], mine = 0;                        // len < 0: no fork; last: its source's started page
  bool tail[kPgPer];
#pragma unroll
  for (int j = 0; j < kPgPer; ++j) {
    const int i = threadIdx.x * kPgPer + j;
    len[j] = last[j] = -1, tail[j] = false;
    if (i >= n) continue;
    const int s = src[i], d = dst[i];
    bool ok = s >= 0 && s < p.streams && d >= 0 && d < p.streams && s != d && claim[d] == i && p.num_pages[d] == 0;
    if (ok) {
      const int L = p.seq_lens[s], pages = L / kPgPage + (L % kPgPage != 0);
      ok = L >= 0 && pages <= p.num_pages[s] && pages <= p.max_blocks;
      if (ok && L % kPgPage != 0) {
        last[j] = p.tables[(int64_t)s * p.bt_stride + L / kPgPage];
        ok = tail[j] = last[j] >= 0 && last[j] < p.blocks;
      }
      if (ok) len[j] = L;
    }
    if (!ok) atomicOr(&p.ws->status, STATUS_BAD_STREAM);
    mine += tail[j];
  }
  int at;
  const int wanted = pg_scan(mine, &at, red);
  const PgShare sh = pg_share(p.blocks);
  int rank;
  const int n_free = pg_scan(pg_count_free(p, sh), &rank, red);   // (the scan's barriers: every source has been read)
  const int limit = min(wanted, n_free);
  for (int id = sh.lo; id < sh.hi && rank < limit; ++id) {
    if (p.ref[id] != 0) continue;
    fresh[rank++] = id;
    p.ref[id] = 1;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPgPer; ++j) {
    const int i = threadIdx.x * kPgPer + j;
    if (i >= n) continue;
    int4 plan = make_int4(-1, -1, 0, -1);
    int to = -1;
    if (len[j] >= 0) {
      bool ok = true;
      if (tail[j]) {
        ok = at < limit;
        if (!ok) atomicOr(&p.ws->status, STATUS_NO_PAGES);
        else to = fresh[at];
        ++at;
      }
      if (ok) plan = make_int4(src[i], dst[i], len[j], last[j]);
    }
    pg_fork_plan(p)[i] = plan;
    pg_fork_tail(p)[i] = to;
  }
}

// 16-byte units of one page of one layer, from src to dst, by the whole block
__device__ __forceinline__ void pg_copy(uint4* dst, const uint4* src, int units) {
  for (int u = threadIdx.x; u < units; u += blockDim.x) dst[u] = src[u];
}

// grid (1 + layers, requests): the first block of a request makes the child, the others copy its source's started page (of no
// use, and to a page that is free again, where a full page's id is bad).
__global__ void __launch_bounds__(256) kv_fork_kernel(const KvPool p, uint4* kv, int64_t layer_units, int64_t block_units,
                                                      int units) {
  pdl_wait();
  const int4 f = pg_fork_plan(p)[blockIdx.y];
  const int to = pg_fork_tail(p)[blockIdx.y];
  if (f.x < 0) return;
  if (blockIdx.x == 0) {
    const int* from = p.tables + (int64_t)f.x * p.bt_stride;
    int* row = p.tables + (int64_t)f.y * p.bt_stride;
    const int whole = f.z / kPgPage;
    bool bad = false;
    for (int i = threadIdx.x; i < whole; i += 256) bad |= (unsigned)from[i] >= (unsigned)p.blocks;
    if (__syncthreads_or(bad)) {                                  // left out whole; its page goes back
      if (threadIdx.x == 0) {
        atomicOr(&p.ws->status, STATUS_BAD_STREAM);
        if (to >= 0) atomicSub(&p.ref[to], 1);
      }
    } else {
      for (int i = threadIdx.x; i < whole; i += 256) {
        row[i] = from[i];
        atomicAdd(&p.ref[from[i]], 1);
      }
      if (threadIdx.x == 0) {
        if (to >= 0) row[whole] = to;
        p.num_pages[f.y] = whole + (to >= 0);
        p.seq_lens[f.y] = f.z;
      }
    }
    pg_publish();
    return;
  }
  if (to < 0) return;
  uint4* layer = kv + (blockIdx.x - 1) * layer_units;
  pg_copy(layer + to * block_units, layer + f.w * block_units, units);
  pg_publish();
}

// One block.  remap[p]: where used page p lies afterwards (-1: free); the k-th used page behind the first `live` ids takes
// the k-th free id among them.
__global__ void __launch_bounds__(kPgT) kv_compact_plan_kernel(const KvPool p, int* remap, int* live_out) {
  __shared__ int red[32], s_below;
  pdl_trigger();
  pdl_wait();
  const PgShare sh = pg_share(p.blocks);
  int before;
  const int used = (sh.hi - sh.lo) - pg_count_free(p, sh);
  const int live = pg_scan(used, &before, red);
  if (threadIdx.x == 0) {
    s_below = live;                                               // used ids below `live` (live == blocks: all)
    live_out[0] = live;
  }
  __syncthreads();
  int2* moves = pg_moves(p);
  int u = before;                                                 // used ids below id
  for (int id = sh.lo; id < sh.hi; ++id) {
    const bool is_used = p.ref[id] != 0;
    if (id == live) s_below = u;
    if (id < live && !is_used) moves[id - u].y = id;
    remap[id] = is_used ? id : -1;
    u += is_used;
  }
  __syncthreads();
  const int below = s_below;
  u = before;
  for (int id = sh.lo; id < sh.hi; ++id) {
    if (p.ref[id] == 0) continue;
    if (id >= live) moves[u - below].x = id;
    ++u;
  }
  __syncthreads();
  const int n = live - below;
  for (int k = threadIdx.x; k < n; k += kPgT) {
    const int2 m = moves[k];
    remap[m.x] = m.y;
    p.ref[m.y] = p.ref[m.x];
    p.ref[m.x] = 0;
  }
  if (threadIdx.x == 0) p.ws->moves = n;
}

__global__ void __launch_bounds__(256) kv_compact_kernel(const KvPool p, const int* remap, uint4* kv, int layers,
                                                         int64_t layer_units, int64_t block_units, int units) {
  pdl_wait();
  const int64_t entries = (int64_t)p.streams * p.max_blocks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
    int* e = p.tables + i / p.max_blocks * p.bt_stride + i % p.max_blocks;
    const int page = *e;
    if (page >= 0 && page < p.blocks && remap[page] >= 0) *e = remap[page];
  }
  const int64_t copies = (int64_t)p.ws->moves * layers;
  for (int64_t i = blockIdx.x; i < copies; i += gridDim.x) {
    const int2 m = pg_moves(p)[i / layers];
    uint4* layer = kv + i % layers * layer_units;
    pg_copy(layer + m.y * block_units, layer + m.x * block_units, units);
  }
  pg_publish();
}

}  // namespace flint

using namespace flint;

int64_t flint::status_offset_kv_pages() { return (int64_t)offsetof(KvPagesWorkspace, status); }

extern "C" int64_t flint_kv_pages_workspace_bytes(int64_t blocks) {
  if (blocks < 1) return -1;
  const int64_t fork = kPgMaxRequests * (int64_t)(sizeof(int4) + sizeof(int)), compact = blocks * (int64_t)sizeof(int2);
  return (int64_t)sizeof(KvPagesWorkspace) + (fork > compact ? fork : compact);
}

static int kv_pool(KvPool* p, int32_t* ref, int64_t blocks, int32_t* tables, int64_t bt_stride, int64_t max_blocks,
                   int32_t* seq_lens, int32_t* num_pages, int64_t streams, void* workspace) {
  if (!ref || !tables || !num_pages || !workspace) return FLINT_ERR_ARGUMENT;
  if (blocks < 1 || blocks > (1 << 30) || streams < 1 || streams > kPgMaxRequests || max_blocks < 1 ||
      max_blocks > INT32_MAX / streams || bt_stride < max_blocks)
    return FLINT_ERR_SHAPE;
  if (!aligned(workspace, 16)) return FLINT_ERR_ALIGN;
  *p = KvPool{ref, (int)blocks, tables, bt_stride, (int)max_blocks, seq_lens, num_pages, (int)streams,
              static_cast<KvPagesWorkspace*>(workspace)};
  return num_sms() > 0 ? FLINT_OK : FLINT_ERR_DEVICE;
}

static int kv_cache_check(const void* kv, int64_t layers, int64_t num_kv_heads, int64_t stride_layer, int64_t stride_block) {
  if (!kv) return FLINT_ERR_ARGUMENT;
  if (layers < 1 || layers > 65535 || num_kv_heads < 1 || num_kv_heads > 1024 || stride_block < num_kv_heads * 16 * 256 ||
      (layers > 1 && stride_layer < 1))
    return FLINT_ERR_SHAPE;
  return aligned(kv, 16) && stride_layer % 8 == 0 && stride_block % 8 == 0 ? FLINT_OK : FLINT_ERR_ALIGN;
}

extern "C" int flint_kv_free(int32_t* ref, int64_t blocks, int32_t* block_tables, int64_t bt_stride, int64_t max_blocks,
                             int32_t* seq_lens, int32_t* num_pages, int64_t num_streams, const int32_t* streams, int64_t n,
                             void* workspace, int pdl, void* stream) {
  if (!streams || !seq_lens) return FLINT_ERR_ARGUMENT;
  KvPool p;
  const int rc = kv_pool(&p, ref, blocks, block_tables, bt_stride, max_blocks, seq_lens, num_pages, num_streams, workspace);
  if (rc) return rc;
  if (n < 1 || n > kPgMaxRequests) return FLINT_ERR_SHAPE;
  return launch(kv_free_kernel, dim3((unsigned)n), dim3(256), 0, stream, pdl, p, streams);
}

extern "C" int flint_kv_reserve(int32_t* ref, int64_t blocks, int32_t* block_tables, int64_t bt_stride, int64_t max_blocks,
                                int32_t* num_pages, int64_t num_streams, const int32_t* streams, const int32_t* lens,
                                int64_t n, void* workspace, int pdl, void* stream) {
  if (!streams || !lens) return FLINT_ERR_ARGUMENT;
  KvPool p;
  const int rc = kv_pool(&p, ref, blocks, block_tables, bt_stride, max_blocks, nullptr, num_pages, num_streams, workspace);
  if (rc) return rc;
  if (n < 1 || n > kPgMaxRequests) return FLINT_ERR_SHAPE;
  return launch(kv_reserve_kernel, dim3(1), dim3(kPgT), kPgMaxRequests * sizeof(int), stream, pdl, p, streams, lens, (int)n);
}

extern "C" int flint_kv_fork(void* kv, int64_t layers, int64_t num_kv_heads, int64_t stride_layer, int64_t stride_block,
                             int32_t* ref, int64_t blocks, int32_t* block_tables, int64_t bt_stride, int64_t max_blocks,
                             int32_t* seq_lens, int32_t* num_pages, int64_t num_streams, const int32_t* src,
                             const int32_t* dst, int64_t n, void* workspace, int pdl, void* stream) {
  if (!src || !dst || !seq_lens) return FLINT_ERR_ARGUMENT;
  KvPool p;
  int rc = kv_cache_check(kv, layers, num_kv_heads, stride_layer, stride_block);
  if (!rc) rc = kv_pool(&p, ref, blocks, block_tables, bt_stride, max_blocks, seq_lens, num_pages, num_streams, workspace);
  if (rc) return rc;
  if (n < 1 || n > kPgMaxRequests) return FLINT_ERR_SHAPE;
  rc = launch(kv_fork_plan_kernel, dim3(1), dim3(kPgT), kPgMaxRequests * sizeof(int), stream, pdl, p, src, dst, (int)n);
  if (rc) return rc;
  return launch(kv_fork_kernel, dim3((unsigned)layers + 1, (unsigned)n), dim3(256), 0, stream, pdl, p,
                static_cast<uint4*>(kv), stride_layer / 8, stride_block / 8, (int)num_kv_heads * 512);
}

extern "C" int flint_kv_compact(void* kv, int64_t layers, int64_t num_kv_heads, int64_t stride_layer, int64_t stride_block,
                                int32_t* ref, int64_t blocks, int32_t* block_tables, int64_t bt_stride, int64_t max_blocks,
                                int32_t* num_pages, int64_t num_streams, int32_t* remap, int32_t* live, void* workspace,
                                int pdl, void* stream) {
  if (!remap || !live) return FLINT_ERR_ARGUMENT;
  KvPool p;
  int rc = kv_cache_check(kv, layers, num_kv_heads, stride_layer, stride_block);
  if (!rc) rc = kv_pool(&p, ref, blocks, block_tables, bt_stride, max_blocks, nullptr, num_pages, num_streams, workspace);
  if (rc) return rc;
  rc = launch(kv_compact_plan_kernel, dim3(1), dim3(kPgT), 0, stream, pdl, p, remap, live);
  if (rc) return rc;
  return launch(kv_compact_kernel, dim3((unsigned)num_sms() * 8), dim3(256), 0, stream, pdl, p, (const int*)remap,
                static_cast<uint4*>(kv), (int)layers, stride_layer / 8, stride_block / 8, (int)num_kv_heads * 512);
}
