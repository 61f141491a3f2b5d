// Attention of many query rows over the paged KV cache: a prompt (or a chunk of one, or drafted tokens) read causally
// (flint_prefill_attention), and decode streams whose block tables begin with the same pages
// (flint_shared_prefix_attention).
//
// KV cache: HND bf16 [num_blocks, num_kv_heads, 16, 2 * 128], K in the first 128 columns of a token's row, V in the rest.
// A tile is up to 64 query rows of one KV head: consecutive tokens of one sequence, each with its G query heads (row =
// token * G + head), so that the group reads its keys once.  With c = scale * log2(e), a row at position p over the keys
// max(0, p - window + 1) .. p keeps the running maximum m and, in 32 bits, l = sum 2^(c (s - m)) and o = sum 2^(..) v;
// the probabilities are rounded to bf16 for the product with V only (l sums the unrounded ones, as the decode attention
// does).  A sink adds 2^(sink log2 e - c m) to l.  A row without keys gives zeros.  Cache slots that no row may see are
// never multiplied: their scores are replaced, their V rows read as zero.
#include "common.cuh"
#include "runtime.cuh"
#include "tma.cuh"

namespace flint {

constexpr int kPaD = 128;
constexpr int kPaPage = 16;
constexpr int kPaRows = 64;                    // query rows of a tile
constexpr int kPaKeys = 64;                    // keys of a step
constexpr int kPaLd = kPaD + 8;                // halves of a staged row: 16-byte units of 8 rows fall in 8 bank groups
constexpr float kPaLog2e = 1.4426950408889634f;
constexpr unsigned STATUS_BAD_SEQ = 4u;

struct PagedAttnWorkspace {
  unsigned status;
  unsigned pad[31];
};

struct PagedAttnArgs {
  const bf16* q;
  int64_t q_stride;                            // elements between tokens
  const bf16* kv;
  int64_t stride_block, stride_head;           // elements
  int64_t num_blocks;
  const int* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int* cu_seqlens;                       // [batch + 1], or null: sequence b is the one token b
  const int* seq_lens;
  const int *group_starts, *prefix_lens;       // shared prefixes only
  int groups;
  const float* sinks;
  int window, batch, tokens, Hkv, G;
  float c;
  bf16* out;
  int64_t out_stride;
  PagedAttnWorkspace* ws;
};

__device__ __forceinline__ void pa_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void pa_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttnArgs a) {
  __shared__ __align__(16) bf16 sk[kPaKeys][kPaLd], sv[kPaKeys][kPaLd];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g4 = lane >> 2, t4 = lane & 3;
  const int h = blockIdx.y, tile_tokens = kPaRows / a.G;
  if (blockIdx.x == 0 && h == 0)
    for (int i = tid; i < a.groups; i += 128) {
      const int s0 = a.group_starts[i], s1 = a.group_starts[i + 1], n = a.prefix_lens[i];
      if (s0 < 0 || s1 < s0 || s1 > a.batch || n < 0 || n > a.max_blocks * kPaPage) atomicOr(&a.ws->status, STATUS_BAD_SEQ);
    }
  // the tile's sequence and first token: sequences take ceil(n / tile_tokens) tiles each, in order
  int b = 0, first = 0, n = 0, t0 = 0;
  {
    int left = blockIdx.x;
    for (; b < a.batch; ++b) {
      first = a.cu_seqlens ? a.cu_seqlens[b] : b;
      n = (a.cu_seqlens ? a.cu_seqlens[b + 1] : b + 1) - first;
      if (first < 0 || n < 0 || first + n > a.tokens) {
        if (tid == 0) atomicOr(&a.ws->status, STATUS_BAD_SEQ);
        n = 0;
      }
      const int tiles = (n + tile_tokens - 1) / tile_tokens;
      if (left < tiles) break;
      left -= tiles;
    }
    if (b == a.batch) return;
    t0 = left * tile_tokens;
  }
  int len = a.seq_lens[b];
  if (len > a.max_blocks * kPaPage) {
    len = a.max_blocks * kPaPage;
    if (tid == 0) atomicOr(&a.ws->status, STATUS_BAD_SEQ);
  }
  const int rows = min(tile_tokens, n - t0) * a.G;
  const int pos0 = len - n + t0;                                  // position of the tile's first token
  const int pos_last = pos0 + min(tile_tokens, n - t0) - 1;
  const int end = max(0, pos_last + 1);
  const int begin = a.window > 0 ? max(0, pos0 - a.window + 1) & ~(kPaPage - 1) : 0;

  // this thread's rows of the warp's 16: r0 = 16 warp + g4 and r0 + 8
  int lo[2], hi[2];
  const bf16* qrow[2];
  bool valid[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * warp + g4 + 8 * i;
    valid[i] = r < rows;
    const int tok = r / a.G, p = pos0 + tok;
    hi[i] = valid[i] ? p + 1 : 0;
    lo[i] = a.window > 0 ? max(0, p - a.window + 1) : 0;
    qrow[i] = a.q + (int64_t)(first + t0 + tok) * a.q_stride + (h * a.G + r - tok * a.G) * kPaD;
  }
  uint32_t qa[8][4];
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qa[kk][i] = valid[i & 1] ? *reinterpret_cast<const uint32_t*>(qrow[i & 1] + 16 * kk + 8 * (i >> 1) + 2 * t4) : 0u;
  float o[16][4];
#pragma unroll
  for (int d = 0; d < 16; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  for (int k0 = begin; k0 < end; k0 += kPaKeys) {
    __syncthreads();
    for (int u = tid; u < kPaKeys * 32; u += 128) {
      const int key = u >> 5, unit = u & 31;                      // 16-byte units of a token's K | V row
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (k0 + key < end) {
        const int blk = a.block_tables[(int64_t)b * a.bt_stride + (k0 + key) / kPaPage];
        if (blk >= 0 && blk < a.num_blocks)
          v = *reinterpret_cast<const uint4*>(a.kv + blk * a.stride_block + h * a.stride_head +
                                              ((k0 + key) & (kPaPage - 1)) * 2 * kPaD + unit * 8);
      }
      *reinterpret_cast<uint4*>(unit < 16 ? &sk[key][unit * 8] : &sv[key][(unit - 16) * 8]) = v;
    }
    __syncthreads();
    float s[8][4];
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
    const int mat = lane >> 3, r8 = lane & 7;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
#pragma unroll
      for (int np = 0; np < 4; ++np) {
        uint32_t kf[4];
        pa_ldsm(smem_u32(&sk[16 * np + 8 * (mat >> 1) + r8][16 * kk + 8 * (mat & 1)]), kf);
        mma_bf16(s[2 * np], qa[kk], kf[0], kf[1]);
        mma_bf16(s[2 * np + 1], qa[kk], kf[2], kf[3]);
      }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = k0 + 8 * nt + 2 * t4 + (e & 1), i = e >> 1;
        if (key >= hi[i] || key < lo[i]) s[nt][e] = -INFINITY;
        top[i] = fmaxf(top[i], s[nt][e]);
      }
    float base[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      const float mn = fmaxf(m[i], top[i]);
      base[i] = mn == -INFINITY ? 0.f : mn * a.c;
      const float alpha = m[i] == -INFINITY ? 0.f : exp2f(m[i] * a.c - base[i]);
      m[i] = mn;
      l[i] *= alpha;
#pragma unroll
      for (int d = 0; d < 16; ++d) {
        o[d][2 * i] *= alpha;
        o[d][2 * i + 1] *= alpha;
      }
    }
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[nt][e] = exp2f(s[nt][e] * a.c - base[e >> 1]);
        l[e >> 1] += s[nt][e];
      }
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {                              // 16 keys at a time
      const uint32_t pa[4] = {pa_pack(s[2 * kt][0], s[2 * kt][1]), pa_pack(s[2 * kt][2], s[2 * kt][3]),
                              pa_pack(s[2 * kt + 1][0], s[2 * kt + 1][1]), pa_pack(s[2 * kt + 1][2], s[2 * kt + 1][3])};
#pragma unroll
      for (int dp = 0; dp < 8; ++dp) {
        uint32_t vf[4];
        pa_ldsm_t(smem_u32(&sv[16 * kt + 8 * (mat & 1) + r8][16 * dp + 8 * (mat >> 1)]), vf);
        mma_bf16(o[2 * dp], pa, vf[0], vf[1]);
        mma_bf16(o[2 * dp + 1], pa, vf[2], vf[3]);
      }
    }
  }
  pdl_trigger();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (!valid[i]) continue;
    const int r = 16 * warp + g4 + 8 * i, tok = r / a.G, qh = h * a.G + r - tok * a.G;
    float den = l[i];
    if (a.sinks && m[i] != -INFINITY) den += exp2f(a.sinks[qh] * kPaLog2e - m[i] * a.c);
    const float inv = m[i] == -INFINITY ? 0.f : 1.0f / den;
    bf16* dst = a.out + (int64_t)(first + t0 + tok) * a.out_stride + qh * kPaD;
#pragma unroll
    for (int d = 0; d < 16; ++d)
      *reinterpret_cast<uint32_t*>(dst + 8 * d + 2 * t4) = pa_pack(o[d][2 * i] * inv, o[d][2 * i + 1] * inv);
  }
}

}  // namespace flint

using namespace flint;

int64_t flint::status_offset_paged_attention() { return (int64_t)offsetof(PagedAttnWorkspace, status); }

static int paged_attn_check(const void* q, int64_t q_stride, const void* kv, int64_t num_blocks, int64_t Hkv,
                            int64_t stride_block, int64_t stride_head, const int32_t* bt, int64_t bt_stride,
                            int64_t max_blocks, const int32_t* seq_lens, int64_t window, int64_t batch, int64_t tokens,
                            int64_t Hq, const void* out, int64_t out_stride, const void* ws) {
  if (!q || !kv || !bt || !seq_lens || !out || !ws) return FLINT_ERR_ARGUMENT;
  if (window < 0 || window > INT32_MAX) return FLINT_ERR_ARGUMENT;
  if (batch < 1 || batch > 65535 || tokens < 1 || tokens > (1 << 24) || Hkv < 1 || Hkv > 128 || Hq < 1 || Hq % Hkv != 0 ||
      Hq / Hkv > 8 || num_blocks < 1 || num_blocks > INT32_MAX || max_blocks < 1 || max_blocks > (1 << 26) ||
      bt_stride < 0 || q_stride < Hq * kPaD || out_stride < Hq * kPaD || stride_head < kPaPage * 2 * kPaD ||
      stride_block < stride_head)
    return FLINT_ERR_SHAPE;
  if (!aligned(kv, 16) || stride_block % 8 != 0 || stride_head % 8 != 0 || !aligned(out, 16) || !aligned(q, 16) ||
      q_stride % 8 != 0 || out_stride % 8 != 0)
    return FLINT_ERR_ALIGN;
  if (num_sms() <= 0) return FLINT_ERR_DEVICE;
  return FLINT_OK;
}

static PagedAttnArgs paged_attn_args(const void* q, int64_t q_stride, const void* kv, int64_t num_blocks, int64_t Hkv,
                                     int64_t stride_block, int64_t stride_head, const int32_t* bt, int64_t bt_stride,
                                     int64_t max_blocks, const int32_t* seq_lens, const float* sinks, int64_t window,
                                     float scale, int64_t batch, int64_t tokens, int64_t Hq, void* out,
                                     int64_t out_stride, void* ws) {
  PagedAttnArgs a = {};
  a.q = (const bf16*)q; a.q_stride = q_stride; a.kv = (const bf16*)kv; a.stride_block = stride_block;
  a.stride_head = stride_head; a.num_blocks = num_blocks; a.block_tables = bt; a.bt_stride = bt_stride;
  a.max_blocks = (int)max_blocks; a.seq_lens = seq_lens; a.sinks = sinks; a.window = (int)window; a.batch = (int)batch;
  a.tokens = (int)tokens; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv); a.c = scale * kPaLog2e; a.out = (bf16*)out;
  a.out_stride = out_stride; a.ws = static_cast<PagedAttnWorkspace*>(ws);
  return a;
}

extern "C" int64_t flint_prefill_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t num_q_heads,
                                                           int64_t num_kv_heads) {
  if (batch < 1 || tokens < 1 || num_q_heads < 1 || num_kv_heads < 1) return -1;
  return (int64_t)sizeof(PagedAttnWorkspace);
}

extern "C" int flint_prefill_attention(const void* q, int64_t q_stride_t, const void* kv_cache, int64_t num_blocks,
                                       int64_t num_kv_heads, int64_t stride_block, int64_t stride_head,
                                       const int32_t* block_tables, int64_t bt_stride, int64_t max_blocks,
                                       const int32_t* cu_seqlens, const int32_t* seq_lens, const float* sinks,
                                       int64_t window, float scale, int64_t batch, int64_t tokens, int64_t num_q_heads,
                                       void* out, int64_t out_stride_t, void* workspace, int pdl, void* stream) {
  if (!cu_seqlens) return FLINT_ERR_ARGUMENT;
  int rc = paged_attn_check(q, q_stride_t, kv_cache, num_blocks, num_kv_heads, stride_block, stride_head, block_tables,
                            bt_stride, max_blocks, seq_lens, window, batch, tokens, num_q_heads, out, out_stride_t,
                            workspace);
  if (rc) return rc;
  PagedAttnArgs a = paged_attn_args(q, q_stride_t, kv_cache, num_blocks, num_kv_heads, stride_block, stride_head,
                                    block_tables, bt_stride, max_blocks, seq_lens, sinks, window, scale, batch, tokens,
                                    num_q_heads, out, out_stride_t, workspace);
  a.cu_seqlens = cu_seqlens;
  const int tile_tokens = kPaRows / a.G;
  const int64_t tiles = tokens / tile_tokens + batch;             // an upper bound of sum ceil(n_b / tile_tokens)
  return launch(paged_attn_kernel, dim3((unsigned)tiles, (unsigned)num_kv_heads), dim3(128), 0, stream, pdl, a);
}

extern "C" int64_t flint_shared_prefix_attention_workspace_bytes(int64_t batch, int64_t groups, int64_t num_q_heads,
                                                                 int64_t num_kv_heads) {
  if (batch < 1 || groups < 1 || num_q_heads < 1 || num_kv_heads < 1) return -1;
  return (int64_t)sizeof(PagedAttnWorkspace);
}

extern "C" int flint_shared_prefix_attention(const void* q, int64_t q_stride_b, const void* kv_cache, int64_t num_blocks,
                                             int64_t num_kv_heads, int64_t stride_block, int64_t stride_head,
                                             const int32_t* block_tables, int64_t bt_stride, int64_t max_blocks,
                                             const int32_t* seq_lens, const int32_t* group_starts,
                                             const int32_t* prefix_lens, int64_t groups, const float* sinks,
                                             int64_t window, float scale, int64_t batch, int64_t num_q_heads, void* out,
                                             int64_t out_stride_b, void* workspace, int pdl, void* stream) {
  if (!group_starts || !prefix_lens) return FLINT_ERR_ARGUMENT;
  if (groups < 1 || groups > batch) return FLINT_ERR_SHAPE;
  int rc = paged_attn_check(q, q_stride_b, kv_cache, num_blocks, num_kv_heads, stride_block, stride_head, block_tables,
                            bt_stride, max_blocks, seq_lens, window, batch, batch, num_q_heads, out, out_stride_b,
                            workspace);
  if (rc) return rc;
  PagedAttnArgs a = paged_attn_args(q, q_stride_b, kv_cache, num_blocks, num_kv_heads, stride_block, stride_head,
                                    block_tables, bt_stride, max_blocks, seq_lens, sinks, window, scale, batch, batch,
                                    num_q_heads, out, out_stride_b, workspace);
  a.group_starts = group_starts; a.prefix_lens = prefix_lens; a.groups = (int)groups;
  return launch(paged_attn_kernel, dim3((unsigned)batch, (unsigned)num_kv_heads), dim3(128), 0, stream, pdl, a);
}
