// Attention of many query rows over the paged KV cache: a prompt (or a chunk of one, or drafted tokens) read causally
// (flint_prefill_attention), and decode streams whose block tables begin with the same pages, which are read once for all
// of them (flint_shared_prefix_attention).
//
// KV cache: HND bf16 [num_blocks, num_kv_heads, 16, 2 * 128], K in the first 128 columns of a token's row, V in the rest.
// With c = scale * log2(e), a row over its visible keys keeps a reference m, l = sum 2^(c (s - m)) and o = sum 2^(..) v in
// 32 bits; the probabilities are rounded to bf16 for the product with V only (l sums the unrounded ones, as the decode
// attention does).  Results over disjoint keys join as m = max m_k, l = sum l_k 2^(c (m_k - m)), o likewise.  A sink adds
// 2^(sink log2 e - c m) to l.  A row without keys gives zeros: its l is 0.  m alone does not tell, since a maximum passes over
// NaN: a row whose scores are NaN has m = -inf and l = NaN, and gives NaN.
//
// Work.  An item is one KV head and up to two row tiles of 128 rows: floor(128 / G) consecutive query tokens (or streams)
// with their G heads each, so the group reads its keys once.  Items are laid on one line by what they cost (their keys and a
// constant) and the line is cut into equal shares, one per SM: a long prompt's items and a few rows on a long cache are both
// split evenly.  Where a cut falls into an item its parts leave (m, l, o) in the workspace, and a second launch joins them in
// the order of the keys, so results repeat bit for bit.
//   an item of two tiles: both tiles multiply the same keys; one's softmax runs under the other's products
//   an item of one tile:  its keys are dealt to the two halves of the block in turn, and joined at the end
//
// Block: two softmax groups of 4 warps (a thread per row), a warp each for TMA, for the MMAs and for cutting the items.
// Keys come 128 at a time: 8 pages, one TMA box of 16 tokens x 64 columns per half of K or V, 128-byte swizzle, into a ring
// of four 32 KB slots.  S = Q K^T (both from shared memory) and O += P V (P from tensor memory, where it overwrites its S;
// V as it lies, tokens as the K dimension) are tcgen05 products of 128 x 128 x 128, issued by one elected lane.  The MMAs of
// one thread run in order, so when S of a step has come, the O of the step before is complete: the softmax group may rescale
// it.  It does so only when a row's maximum rises by more than 2^8 over the reference, which the first steps do.
// Slots that no row may see are never multiplied: a page that an item does not reach is read out of bounds (zeros), its
// last page, if cut, is read with its first row shifted up, so that the rows behind the end are out of bounds too, and rows
// of V that a window has left behind in the first page are cleared in shared memory.
//
// Measured (32 heads on 4 KV heads): a prompt of 6,057 tokens 284 us (1.06 PFLOP/s), of 16,421 tokens 1.9 ms (1.16), in long
// runs at the card's power limit 327 us and 2.12 ms; 192 streams on three prefixes of up to 16,384 tokens 102 us.  A step of
// two tiles, 2,048 cycles of products, takes some 1.9 us: the tensor pipe is busy for 51 to 62% of it, the rest is the way
// S -> softmax (1.4 us) -> P -> S through four barriers.  Without the maximum or without the exponentials a prompt is only 6%
// faster; two threads a row (16 softmax warps) cost 20%, S in two buffers of 64 keys 5% (an MMA of N = 64 takes as long as
// one of N = 128), a share of the exponentials on the FMA pipes nothing.  What a call costs besides: 3 to 6 us to its first item
// and 2 to 3 us for the join's launch, which bound the small ones; an item, 2 to 4 us of filling and draining.
#include <limits.h>

#include <atomic>

#include "common.cuh"
#include "runtime.cuh"
#include "timeline.cuh"
#include "tma.cuh"

FLINT_TL_BUFFER

namespace flint {

constexpr int kPaD = 128;
constexpr int kPaPage = 16;
constexpr int kPaM = 128;                      // rows of a tile
constexpr int kPaKeys = 128;                   // keys of a step
constexpr int kPaSlots = 4;                    // ring slots of 128 keys x 128 columns (K or V)
constexpr int kPaSlotBytes = kPaKeys * kPaD * 2;
constexpr int kPaHalf = kPaSlotBytes / 2;      // 64 columns
constexpr int kPaPageHalf = kPaPage * 128;     // a page's 64 columns
constexpr int kPaRuns = 64;                    // runs of 32 segments that are kept
constexpr int kPaQueue = 4;                    // items cut ahead
constexpr int kPaThreads = 384;                // 2 x 4 softmax warps, TMA, MMA, items, one idle
constexpr int kPaTmem = 512;                   // columns: S0 (P0), S1 (P1), O0, O1, 128 each
constexpr float kPaLog2e = 1.4426950408889634f;
constexpr float kPaRise = 8.f;                 // log2 of how far p may exceed 1 before the reference moves
// Cost of an item of two tiles / of one beside its keys, in keys (a step of 128 takes some 2 us, an item 4 or 2 us more).
// At 130/60, 200/100, 260/120, 320/160, 400/200: 6,057 tokens 327, 298, 288, 303, 313 us; 192 streams 115, 104, 102, 106, 107;
// packed prompts under a window 76, 74, 67, 64, 64; 1,000 tokens 38, 35, 35, 34, 37; 2,048 behind 6,057 221 to 224.
constexpr int kPaFixed2 = 260, kPaFixed1 = 120;
// Least share of a block, in keys.  At 100, 200, 400, 800: 17 tokens 10.8, 10.6, 14.6, 23.1 us; a row on 1,000 keys 13.9, 15.9,
// 18.9, 26.7; four rows on 3,000 keys 22.0, 20.5, 21.8, 26.8; 2 streams 17.6, 20.1, 20.4, 28.7; 8 streams 24.0, 24.0, 24.5, 28.4.
constexpr int kPaLeast = 200;
constexpr unsigned STATUS_BAD_SEQ = 4u;
constexpr size_t kPaSmem = 1024 + 2 * kPaSlotBytes + (size_t)kPaSlots * kPaSlotBytes + kPaM * 32 * 4;

struct PagedAttnWorkspace {
  unsigned status;
  unsigned pad[31];
};

// Where the parts of an item are: with blocks first .. last, or one of the values below in `first`.
enum { PA_FINAL = -1, PA_HOME = -2, PA_NONE = -3 };
struct PaSplit {                               // a prompt's item that a block began and did not end
  int first, last, tok0, ntok, h;
};
struct PaRecord {                              // a stream's own keys, or its group's prefix, for one KV head
  int first, last;
  int tok0;                                    // the item's first stream
  int prefix;                                  // of a stream's own keys: its group's prefix has a record too
};

struct PagedAttnArgs {
  int64_t bt_stride;
  const int* block_tables;
  int max_blocks;
  const int* cu_seqlens;                       // prompts: [batch + 1]
  const int* seq_lens;
  const int *group_starts, *prefix_lens;       // shared prefixes
  int groups;
  const float* sinks;
  int window, batch, tokens, Hkv, G, num_blocks;
  int per, inv_g;                              // tokens of a row tile; 2^16 / G rounded up
  float c;
  bf16* out;
  int64_t out_stride;
  int wide;                                    // rows of out begin at 32 bytes
  PagedAttnWorkspace* ws;
  PaSplit* split;                              // prompts: one for each block (ntok 0: none)
  PaRecord* rec;                               // shared prefixes: [batch][Hkv] own keys, then [batch][Hkv] prefixes
  float2 *ml, *home_ml;                        // (m, l): slots [2 x blocks][256 rows], homes [2][batch][Hq]
  float4 *o, *home_o;                          // the same rows' o: slots [32 quads of columns][256 rows], homes [row][32]
};

struct PaItem {
  int tok0, ntok;                              // query tokens (streams)
  int h, table;                                // KV head, row of the block tables
  int begin, end;                              // keys; begin at a page
  int j0, j1;                                  // steps of this part
  int pos0;                                    // position of the first token; prefix: -1
  int dual;
  int dead;                                    // rows of the first page's slot whose keys no row of the item sees
  int out;                                     // slot, PA_HOME or PA_FINAL
  int home;                                    // 0: own keys, 1: prefix
};

// ---- tensor memory and MMA ----
__device__ __forceinline__ void pa_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pa_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void pa_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void pa_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// The loads so far have come; r (32 registers of the last one) is named so that nothing that reads it moves ahead.
__device__ __forceinline__ void pa_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
  asm volatile(""
               : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void pa_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pa_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pa_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The whole MMA warp runs these, so that addresses and descriptors stay in uniform registers; one elected lane (the same
// one every time) issues.  Inside a branch of one lane each MMA took some 125 cycles to issue, twice what it takes to run.
__device__ __forceinline__ void pa_commit(uint64_t* bar) {
  asm volatile(
      "{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_u32(bar))
      : "memory");
}
// Shared-memory operand, 128-byte swizzle (rows of 128 B, 8 rows to 1,024 B), as (low, high) words of its descriptor; the
// low word counts 16-byte units and takes offsets.  K along the row: 8-row groups 1,024 B apart.  K down the rows (V):
// 8 rows of K 1,024 B apart, the next 64 columns `lead` bytes on.
__device__ __forceinline__ uint32_t pa_desc_lo(uint32_t addr, uint32_t lead) {
  return ((addr >> 4) & 0x3FFFu) | ((lead >> 4) << 16);
}
constexpr uint32_t kPaDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// fp32 accumulator, bf16 operands, N = 128, M = 128
constexpr uint32_t kPaIdescQK = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kPaIdescPV = kPaIdescQK | (1u << 16);          // B with K down the rows
__device__ __forceinline__ void pa_mma_qk(uint32_t d, uint32_t q, uint32_t k) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {                                   // 16 columns of Q and K at a time
    const uint32_t off = ((i >> 2) * kPaHalf + (i & 3) * 32) >> 4;
    asm volatile(
        "{\n.reg .pred p, e;\n.reg .b64 qd, kd;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %5, 0;\n"
        "mov.b64 qd, {%1, %4};\nmov.b64 kd, {%2, %4};\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], qd, kd, %3, p;\n}" ::"r"(d), "r"(q + off), "r"(k + off),
        "r"(kPaIdescQK), "r"(kPaDescHi), "r"(i > 0 ? 1u : 0u)
        : "memory");
  }
}
// the last 112 keys, or the first 16; p: where P begins
__device__ __forceinline__ void pa_mma_pv(uint32_t d, uint32_t p, uint32_t v, int part, bool add) {
#pragma unroll
  for (int i = part ? 0 : 1; i < (part ? 1 : 8); ++i) {           // 16 keys at a time: 8 columns of P, 16 rows of V
    asm volatile(
        "{\n.reg .pred p, e;\n.reg .b64 vd;\nelect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %5, 0;\n"
        "mov.b64 vd, {%2, %4};\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], vd, %3, p;\n}" ::"r"(d), "r"(p + 8 * i),
        "r"(v + (uint32_t)((i * 2048) >> 4)), "r"(kPaIdescPV), "r"(kPaDescHi), "r"(add || part || i > 1 ? 1u : 0u)
        : "memory");
  }
}
// TMA boxes without an L2 hint: other blocks read the same keys
__device__ __forceinline__ void pa_tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void pa_tma_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// pairs of fp32 in a 64-bit register
__device__ __forceinline__ uint64_t pa_two(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 pa_split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t pa_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pa_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// bits lo .. hi - 1 of a word
__device__ __forceinline__ uint32_t pa_bits(int lo, int hi) {
  const uint32_t below_hi = hi >= 32 ? ~0u : hi > 0 ? (1u << hi) - 1 : 0u, below_lo = lo >= 32 ? ~0u : lo > 0 ? (1u << lo) - 1 : 0u;
  return below_hi & ~below_lo;
}
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 64 bytes of a row by one thread.  A row is a thread's: 32-byte stores fill a sector each; handing the columns round through
// shared memory, so that a store covers whole lines, took twice as long (2.2 us an item, a chain of short steps).
__device__ __forceinline__ void pa_store64(bf16* dst, const uint32_t* w, bool wide) {
  if (wide) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + 16 * i), "r"(w[8 * i]), "r"(w[8 * i + 1]),
                   "r"(w[8 * i + 2]), "r"(w[8 * i + 3]), "r"(w[8 * i + 4]), "r"(w[8 * i + 5]), "r"(w[8 * i + 6]), "r"(w[8 * i + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}
__device__ __forceinline__ float pa_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// A wait for the phase of the given parity that gives up after two seconds, or as soon as another warp of the block has.
// The lanes of a warp may not agree on that: what the whole warp has to do alike depends on a vote (pa_all).  The warps of
// the products and of the softmax vote once a step and go on until then (a vote behind each wait: 294 us against 281 for
// 6,057 tokens).
constexpr unsigned long long kPaWaitNs = 2000000000ull;
__device__ __forceinline__ unsigned long long pa_now() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __noinline__ bool pa_wait_long(uint64_t* bar, unsigned parity, volatile int* failed, unsigned* status) {
  const unsigned long long t0 = pa_now();
  while (!*failed) {
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (pa_now() - t0 > kPaWaitNs) {
      *failed = 1;
      atomicOr(status, STATUS_WAIT_TIMEOUT);
    }
  }
  return false;
}
__device__ __forceinline__ bool pa_wait(uint64_t* bar, unsigned parity, volatile int* failed, unsigned* status) {
#pragma unroll 1
  for (int i = 0; i < 32; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return pa_wait_long(bar, parity, failed, status);
}
__device__ __forceinline__ bool pa_all(bool ok) { return __all_sync(0xffffffffu, ok); }
// The same after a wait has run out, for copies and products that are still in flight.
__device__ __noinline__ void pa_drain(uint64_t* bar, unsigned parity) {
  const unsigned long long t0 = pa_now();
  while (!mbar_try_wait(bar, parity) && pa_now() - t0 < kPaWaitNs) {
  }
}

// row / G of a row below 256 (exact: the error of inv_g is below 1 / 256 of a quotient's step)
__device__ __forceinline__ int pa_token(const PagedAttnArgs& a, int row) { return (row * a.inv_g) >> 16; }

// ---- the items ----
// sum over i < k of max(0, a + i * t)
__device__ __forceinline__ long long pa_ramp(int a, int t, int k) {
  int i0 = a < 0 ? (int)(((unsigned)-a + t - 1) / (unsigned)t) : 0;
  if (i0 > k) i0 = k;
  return (long long)a * (k - i0) + t * (((k - 1ll) * k - (i0 - 1ll) * i0) / 2);
}
// a / b of non-negative numbers, in 32 bits where they fit (a 64-bit division takes some hundred cycles)
__device__ __forceinline__ long long pa_div(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// A run of row tiles on one line: a prompt's, a group's (its prefix) or a stream's own keys.  Every field is the same for
// all blocks, so that all of them cut the line at the same places.
struct PaSegment {
  int tok0, ntok;                              // its tokens (streams)
  int table;
  int pos0;                                    // position of the first token; prefix: -1
  int lo, hi;                                  // keys outside [lo, hi) are another segment's
  int home;
  long long cost;                              // of one KV head
};

struct PaLine {
  const PagedAttnArgs& a;
  const bool shared;
  const int per, tile;                         // tokens of a row tile, of an item

  __device__ PaLine(const PagedAttnArgs& args) : a(args), shared(args.group_starts != nullptr), per(args.per), tile(2 * args.per) {}
  __device__ int segments() const { return shared ? a.groups + a.batch : a.batch; }
  __device__ void complain(bool bad) const {
    if (bad && blockIdx.x == 0) atomicOr(&a.ws->status, STATUS_BAD_SEQ);
  }
  __device__ int length(int b) const { return length(b, a.seq_lens[b]); }
  __device__ int length(int b, int n) const {
    const int most = a.max_blocks * kPaPage;
    complain(n > most);
    return max(0, min(n, most));
  }
  // streams and shared tokens of group g; a group of one shares nothing
  __device__ int group(int g, int* first, int* prefix) const {
    const int s0 = a.group_starts[g], s1 = a.group_starts[g + 1], n = a.prefix_lens[g];
    const bool bad = s0 < 0 || s1 < s0 || s1 > a.batch || n < 0 || n > a.max_blocks * kPaPage;
    complain(bad);
    *first = s0;
    *prefix = bad || s1 - s0 < 2 ? 0 : n & ~(kPaPage - 1);
    return bad ? 0 : s1 - s0;
  }
  __device__ int prefix_of(int b) const {
    int lo = 0, hi = a.groups - 1;             // the last group that starts at or before b
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.group_starts[mid] <= b) lo = mid; else hi = mid - 1;
    }
    int first, prefix;
    const int n = group(lo, &first, &prefix);
    return b >= first && b < first + n ? prefix : 0;
  }
  __device__ PaSegment segment(int i) const {
    PaSegment s = {};
    if (i >= segments()) return s;
    if (!shared) {
      const int first = a.cu_seqlens[i], next = a.cu_seqlens[i + 1], len = a.seq_lens[i];
      const bool bad = first < 0 || next < first || next > a.tokens;
      complain(bad);
      s.tok0 = first, s.ntok = bad ? 0 : next - first, s.table = i;
      if (s.ntok) s.hi = length(i, len);
      s.pos0 = s.hi - s.ntok;
      complain(len < 0);
    } else if (i < a.groups) {
      int prefix;
      s.ntok = group(i, &s.tok0, &prefix);
      s.table = s.tok0, s.pos0 = -1, s.home = 1, s.hi = prefix;
      if (!prefix) s.ntok = 0;
    } else {
      const int b = i - a.groups;
      s.tok0 = b, s.ntok = 1, s.table = b;
      const int len = a.seq_lens[b];
      s.lo = prefix_of(b);
      s.hi = length(b, len);
      s.lo = min(s.lo, s.hi), s.pos0 = s.hi - 1;
    }
    s.cost = upto(s, (s.ntok + tile - 1) / tile);
    return s;
  }
  __device__ int tokens_of(const PaSegment& s, int i) const { return min(tile, s.ntok - i * tile); }
  // keys that item i is taken to cost; a segment of one item, as a stream's own keys are, in whole steps
  __device__ int keys(const PaSegment& s, int i) const {
    int n = a.window > 0 ? min(s.hi, a.window) : s.hi;
    if (!s.home) {
      const int p = s.pos0 + i * tile, e = p + tokens_of(s, i), b = a.window > 0 ? p - a.window + 1 : 0;
      n = max(0, max(0, e) - max(s.lo, b));
    }
    return s.ntok <= tile ? (n + kPaKeys - 1) & ~(kPaKeys - 1) : n;
  }
  __device__ int fixed(const PaSegment& s, int i) const { return tokens_of(s, i) > per ? kPaFixed2 : kPaFixed1; }
  // cost of the items before item k
  __device__ long long upto(const PaSegment& s, int k) const {
    const int m = (s.ntok + tile - 1) / tile;
    if (k <= 0 || m == 0) return 0;
    const int whole = min(k, m - 1);           // the last item may be shorter
    long long w;
    if (s.home) w = (long long)whole * keys(s, 0);
    else {
      w = pa_ramp(s.pos0 + tile, tile, whole);
      if (a.window > 0) w -= pa_ramp(s.pos0 - a.window + 1, tile, whole);
    }
    if (k >= m) w += keys(s, m - 1) + fixed(s, m - 1);
    return w + (long long)kPaFixed2 * whole;
  }
};
static_assert(kPaFixed1 > 0 && kPaFixed2 > 0, "every item has a place on the line");

__global__ void __launch_bounds__(kPaThreads, 1)
paged_attn_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mkv, const PagedAttnArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;                                             // two Q tiles, each two halves of 64 columns
  uint8_t* ring = sq + 2 * kPaSlotBytes;
  float4* sx = reinterpret_cast<float4*>(ring + kPaSlots * kPaSlotBytes);   // 32 columns of o between the halves
  __shared__ PaItem items[kPaQueue];
  __shared__ __align__(8) uint64_t b_item[kPaQueue], b_item_free[kPaQueue], b_full[kPaSlots], b_empty[kPaSlots], b_q, b_q_free,
      b_s[2], b_p[4], b_o[2], b_hand, b_take, b_end;
  __shared__ float2 s_ml[kPaM];
  __shared__ uint32_t s_taddr;
  __shared__ int s_failed;                                        // a wait ran out: every warp leaves
  __shared__ int s_sent[2];                                       // copies that were started: of keys, of Q
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned* status = &a.ws->status;
  if (tid == 0) {
    FLINT_TL(0);
    s_failed = 0;
    for (int i = 0; i < kPaQueue; ++i) {
      mbar_init(&b_item[i], 1);
      mbar_init(&b_item_free[i], 10);                             // 8 softmax warps, TMA, MMA
    }
    for (int i = 0; i < kPaSlots; ++i) {
      mbar_init(&b_full[i], 1);
      mbar_init(&b_empty[i], 1);
    }
    mbar_init(&b_q, 1);
    mbar_init(&b_q_free, 1);
    mbar_init(&b_hand, 4);
    mbar_init(&b_take, 4);
    mbar_init(&b_end, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&b_s[t], 1);
      mbar_init(&b_p[2 * t], 4);                                  // P of the last 112 and of the first 16 keys
      mbar_init(&b_p[2 * t + 1], 4);
      mbar_init(&b_o[t], 1);
    }
    fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_taddr)),
                 "r"((uint32_t)kPaTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pa_fence_before();
  __syncthreads();
  pa_fence_after();
  const uint32_t tmem = s_taddr;
  if (tid == 0) FLINT_TL(1);
  if (tid == 256) {
    tma_prefetch_desc(&mq);
    tma_prefetch_desc(&mkv);
  }
  pdl_wait();
  pdl_trigger();
  if (tid == 0) FLINT_TL(2);

  // what each run of 32 segments costs, by all warps; the ring is still empty
  const PaLine line(a);
  const int nseg = line.segments();
  long long* runs = reinterpret_cast<long long*>(ring);
  PaSegment* segs = reinterpret_cast<PaSegment*>(runs + kPaRuns);
  const int kept = nseg <= 32 * kPaRuns ? (nseg + 31) / 32 : 0;
  for (int i0 = 32 * ((warp + 2) % 12); i0 < 32 * kept; i0 += kPaThreads) {
    const PaSegment seg = line.segment(i0 + lane);
    segs[i0 + lane] = seg;
    long long c = seg.cost * a.Hkv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if (lane == 0) runs[i0 / 32] = c;
  }
  fence_proxy_async();                                            // (TMA writes these bytes later)
  __syncthreads();

  if (warp == 10) {
    // ---- items: this block's share of the line ----
    // (what the others left in the ring is read until the first item goes out: the TMA warp fills it after that)
    long long total = 0, my_run[2];
    for (int i = lane; i < kept; i += 32) total += runs[i];
    for (int i = 0; i < 2; ++i) my_run[i] = lane + 32 * i < kept ? runs[lane + 32 * i] : 0;
    if (!kept)
      for (int i0 = 0; i0 < nseg; i0 += 32) total += line.segment(i0 + lane).cost * a.Hkv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) FLINT_TL(3);
    // equal shares (of a sum over 32 bits' reach in 64): the first `rest` blocks have one unit more
    const long long shares = max(1ll, min((long long)gridDim.x, pa_div(total, kPaLeast)));
    const long long share = pa_div(total, shares), rest = total - share * shares;
    auto cut = [&](long long c) { return c >= shares ? total : share * c + min(c, rest); };
    const long long x0 = cut(blockIdx.x), x1 = blockIdx.x < shares ? cut(blockIdx.x + 1) : x0;
    long long at = 0;                                             // cost of the segments before the chunk's lane 0
    int n_items = 0;
    bool ok = true;
    PaSplit cut_item = {};
    for (int i0 = 0; i0 < nseg && at < x1 && ok; i0 += 32) {
      if (kept) {                                                 // a run before the share
        const long long c = __shfl_sync(0xffffffffu, my_run[i0 / 1024], i0 / 32 % 32);
        if (at + c <= x0) {
          at += c;
          continue;
        }
      }
      const PaSegment mine = kept && n_items == 0 ? segs[i0 + lane] : line.segment(i0 + lane);
      long long cum = mine.cost * a.Hkv;                          // inclusive scan over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, cum, o);
        if (lane >= o) cum += y;
      }
      const long long chunk = __shfl_sync(0xffffffffu, cum, 31);
      if (at + chunk <= x0) {
        at += chunk;
        continue;
      }
      // from the first segment that ends behind the share's start
      const unsigned live = __ballot_sync(0xffffffffu, mine.cost > 0 && at + cum > x0);
      for (int k = live ? __ffs(live) - 1 : 32; k < 32 && ok; ++k) {
        PaSegment s;
        s.tok0 = __shfl_sync(0xffffffffu, mine.tok0, k);
        s.ntok = __shfl_sync(0xffffffffu, mine.ntok, k);
        s.table = __shfl_sync(0xffffffffu, mine.table, k);
        s.pos0 = __shfl_sync(0xffffffffu, mine.pos0, k);
        s.lo = __shfl_sync(0xffffffffu, mine.lo, k);
        s.hi = __shfl_sync(0xffffffffu, mine.hi, k);
        s.home = __shfl_sync(0xffffffffu, mine.home, k);
        s.cost = __shfl_sync(0xffffffffu, mine.cost, k);
        const long long seg0 = at + __shfl_sync(0xffffffffu, cum, k) - s.cost * a.Hkv;
        if (s.cost == 0 || seg0 + s.cost * a.Hkv <= x0) continue;
        if (seg0 >= x1) break;
        const int m = (s.ntok + line.tile - 1) / line.tile;
        int h = 0, i = 0;
        if (x0 > seg0) {                                          // the first item that the share touches
          h = (int)pa_div(x0 - seg0, s.cost);
          const long long y = x0 - seg0 - h * s.cost;
          int hi = m;
          while (hi - i > 1) {                                    // 32 places at a time
            const int step = (hi - i + 31) / 32, k2 = i + lane * step;
            const int below = __popc(__ballot_sync(0xffffffffu, k2 < hi && line.upto(s, k2) <= y));
            i += (below - 1) * step;
            hi = min(hi, i + step);
          }
        }
        long long start = seg0 + h * s.cost + line.upto(s, i);
        int w = 0, fixed = 0;
        for (; h < a.Hkv && ok && start < x1; ++h, i = 0)
          for (; i < m && start < x1; ++i, start += fixed + w) {
            w = line.keys(s, i), fixed = line.fixed(s, i);
            const long long stop = start + fixed + w;
            PaItem it;
            it.tok0 = s.tok0 + i * line.tile, it.ntok = line.tokens_of(s, i), it.h = h, it.table = s.table;
            it.dual = it.ntok > line.per;
            it.home = s.home;
            if (s.home) {                                         // the keys that the tile's streams see of the prefix
              int lo = INT_MAX, hi = 0, by = 0;
              for (int r = lane; r < it.ntok; r += 32) {
                const int len = line.length(it.tok0 + r);
                if (len > hi) hi = len, by = it.tok0 + r;
                if (len > 0) lo = min(lo, a.window > 0 ? max(0, len - a.window) : 0);
              }
              const int most = __reduce_max_sync(0xffffffffu, hi);  // that stream's table has every page that one of them sees
              it.table = __reduce_min_sync(0xffffffffu, hi == most ? by : INT_MAX);
              hi = most;
              lo = __reduce_min_sync(0xffffffffu, lo);
              it.pos0 = -1;
              it.end = min(s.hi, hi);
              it.begin = lo < it.end ? lo & ~(kPaPage - 1) : it.end;
              it.dead = lo < it.end ? lo - it.begin : 0;
            } else {
              it.pos0 = s.pos0 + i * line.tile;
              it.end = max(0, it.pos0 + it.ntok);
              const int lo = a.window > 0 ? max(0, it.pos0 - a.window + 1) : 0;
              it.begin = min(max(s.lo, lo & ~(kPaPage - 1)), it.end);
              it.dead = max(0, lo - it.begin);
            }
            if (it.dead > 0 && it.end < it.begin + kPaPage) it.dead += it.begin + kPaPage - it.end;   // the last page too
            const int steps = (it.end - it.begin + kPaKeys - 1) / kPaKeys;
            // how many steps lie before place x of the line
            const unsigned unit = steps ? max(1u, ((unsigned)w + steps - 1) / (unsigned)steps) : 1u;
            auto before = [&](long long x) -> int {
              if (x >= stop) return steps;
              return x <= start + fixed ? 0 : min(steps, (int)((unsigned)(x - start - fixed) / unit));
            };
            it.j0 = before(x0), it.j1 = before(x1);
            PaRecord rec = {PA_NONE, PA_NONE, it.tok0, !s.home && s.lo > 0};
            bool first = false;                                   // this part writes the record
            if (steps == 0) {
              if (start < x0) continue;
              first = true;
              it.out = PA_FINAL;
              if (s.home || rec.prefix) it.out = PA_HOME, rec.first = PA_NONE;
              else rec.first = PA_FINAL;
            } else {
              if (it.j0 == it.j1 && (it.j0 == 0 || it.j0 == steps)) continue;
              first = it.j0 == 0;
              if (it.j0 == 0 && it.j1 == steps) {
                it.out = s.home || rec.prefix ? PA_HOME : PA_FINAL;
                rec.first = it.out;
              } else {
                it.out = 2 * blockIdx.x + (it.j0 == 0);
                rec.first = blockIdx.x;
                if (first) {
                  int c = blockIdx.x + 1;                         // the first block that begins behind it, 32 at a time
                  for (unsigned in = ~0u; in == ~0u; c += in == ~0u ? 32 : __ffs(~in) - 1)
                    in = __ballot_sync(0xffffffffu, before(cut(c + lane)) < steps);
                  rec.last = c - 1;
                }
              }
            }
            if (first && line.shared) {
              PaRecord* to = a.rec + (s.home ? (int64_t)a.batch * a.Hkv : 0);
              for (int r = lane; r < it.ntok; r += 32) to[(int64_t)(it.tok0 + r) * a.Hkv + h] = rec;
            } else if (first && rec.first >= 0) {
              cut_item = {rec.first, rec.last, it.tok0, it.ntok, h};
            }
            const int q = n_items % kPaQueue;
            if (n_items >= kPaQueue && !pa_all(pa_wait(&b_item_free[q], (unsigned)((n_items / kPaQueue - 1) & 1), &s_failed, status))) {
              ok = false;
              break;
            }
            if (n_items == 0) fence_proxy_async();                // the ring's bytes have been read
            if (lane == 0) {
              items[q] = it;
              mbar_arrive(&b_item[q]);
              if (n_items == 0) FLINT_TL(4);
            }
            __syncwarp();
            ++n_items;
          }
      }
      at += chunk;
    }
    if (lane == 0 && !line.shared) a.split[blockIdx.x] = cut_item;
    // an item without tokens ends the block
    const int q = n_items % kPaQueue;
    if (n_items >= kPaQueue && ok) ok = pa_all(pa_wait(&b_item_free[q], (unsigned)((n_items / kPaQueue - 1) & 1), &s_failed, status));
    if (ok && lane == 0) {
      items[q].ntok = 0;
      mbar_arrive(&b_item[q]);
    }
    __syncwarp();
  } else if (warp == 8) {
    // ---- TMA ----
    int slot = 0, parity = 1, nq = 0, sent = 0, q_sent = 0;       // an empty ring's slots count as released
    int none = 0;                                                 // negative: a page that the table does not have
    bool ok = true;
    for (int n = 0; pa_all(ok); ++n) {
      if (!pa_all(pa_wait(&b_item[n % kPaQueue], (unsigned)((n / kPaQueue) & 1), &s_failed, status))) break;
      const PaItem it = items[n % kPaQueue];
      __syncwarp();
      if (lane == 0) mbar_arrive(&b_item_free[n % kPaQueue]);
      if (it.ntok == 0) break;
      const int steps = it.j1 - it.j0;
      if (steps == 0) continue;
      const int* row = a.block_tables + (int64_t)it.table * a.bt_stride;
      const int pages_end = (it.end + kPaPage - 1) / kPaPage;
      // (of a prefix under a window, pages between two streams' keys may be gone by right: no row sees them)
      const int heed = it.home && a.window > 0 ? 0 : -1;
      // table entries of four steps, one per lane; the first ones are on their way while Q is sent for
      int held = it.j0 >> 2, ids = it.begin / kPaPage + held * 32 + lane;
      ids = ids < pages_end ? row[ids] : a.num_blocks;
      auto load = [&](int j, int column) {                        // step j's K (column 0) or V (column 128)
        const int p0 = it.begin / kPaPage + j * 8;
        if (held != j >> 2) {
          held = j >> 2;
          none |= ids & heed;
          const int p = it.begin / kPaPage + held * 32 + lane;
          ids = p < pages_end ? row[p] : a.num_blocks;
        }
        const int blk = __shfl_sync(0xffffffffu, ids, (j & 3) * 8 + (lane & 7));
        if (ok && !pa_wait(&b_empty[slot], (unsigned)parity, &s_failed, status)) ok = false;
        if (ok && lane == 0) mbar_arrive_expect_tx(&b_full[slot], kPaSlotBytes);
        sent += ok;
        __syncwarp();
        if (ok && lane < 8) {
          const int left = it.end - (p0 + lane) * kPaPage;        // tokens from this page on
          const int shift = left > 0 && left < kPaPage ? kPaPage - left : 0;
          const uint32_t dst = smem_u32(ring + slot * kPaSlotBytes) + lane * kPaPageHalf;
          pa_tma_4d(dst, &mkv, column, -shift, it.h, blk, &b_full[slot]);
          pa_tma_4d(dst + kPaHalf, &mkv, column + 64, -shift, it.h, blk, &b_full[slot]);
        }
        __syncwarp();
        if (++slot == kPaSlots) slot = 0, parity ^= 1;
      };
      // Q as soon as its buffer is free; the first keys need not wait for that.  One copy of this code: a call of one step
      // takes as long as its instructions take to come.
      const int q_at = __all_sync(0xffffffffu, mbar_try_wait(&b_q_free, (unsigned)((nq & 1) ^ 1))) ? 0 : 1;
      int kj = it.j0, vj = it.j0;                                 // the next step of K, of V
#pragma unroll 1
      for (int i = 0; vj < it.j1; ++i) {
        if (i == q_at) {
          if (ok && !pa_wait(&b_q_free, (unsigned)((nq & 1) ^ 1), &s_failed, status)) ok = false;
          if (ok && lane == 0) {
            const int tiles = it.dual ? 2 : 1, per = a.per;
            mbar_arrive_expect_tx(&b_q, (unsigned)(tiles * 2 * per * a.G * 128));
#pragma unroll 1
            for (int t = 0; t < 2 * tiles; ++t)
              pa_tma_3d(smem_u32(sq) + t * kPaHalf, &mq, (t & 1) * 64, it.h * a.G, it.tok0 + (t >> 1) * per, &b_q);
          }
          q_sent += ok;
          ++nq;
          __syncwarp();
        }
        // two tiles: K0 V0 K1 V1 ..; one: K0 K1 V0 K2 V1 ..
        const bool k = kj < it.j1 && kj - vj < (it.dual ? 1 : 2);
        load(k ? kj : vj, k ? 0 : 128);
        if (k) ++kj;
        else ++vj;
        if (n == 0 && i == 0 && lane == 0) FLINT_TL(5);
      }
      none |= ids & heed;
    }
    if (__any_sync(0xffffffffu, none < 0) && lane == 0) atomicOr(status, STATUS_BAD_SEQ);
    if (lane == 0) s_sent[0] = sent, s_sent[1] = q_sent;
  } else if (warp == 9) {
    // ---- MMA ----
    int slot = 0, parity = 0, p_par[2] = {0, 0}, nq = 0;
    bool ok = true;
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t q_desc = pa_desc_lo(smem_u32(sq), 16), k_desc = pa_desc_lo(smem_u32(ring), 16),
                   v_desc = pa_desc_lo(smem_u32(ring), kPaHalf);
    constexpr uint32_t kTile = kPaSlotBytes >> 4;
    auto next = [&]() {                                           // the next slot of the ring, filled
      const int at = slot;
      ok &= pa_wait(&b_full[at], (unsigned)parity, &s_failed, status);
      if (++slot == kPaSlots) slot = 0, parity ^= 1;
      return at;
    };
    auto qk = [&](int t, int q, int k) {                          // S of half t of the block
      pa_mma_qk(base + 128 * t, q_desc + q * kTile, k_desc + k * kTile);
      pa_commit(&b_s[t]);
    };
    auto pv = [&](int t, int v, bool add) {                       // O += P V, in two parts as P comes
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        ok &= pa_wait(&b_p[2 * t + part], (unsigned)p_par[t], &s_failed, status);
        pa_fence_after();
        pa_mma_pv(base + 256 + 128 * t, base + 128 * t + 64, v_desc + v * kTile, part, add);
      }
      p_par[t] ^= 1;
    };
    // what a window has left behind may be anything, and 0 times NaN is NaN
    auto clear = [&](int v, int rows) {
      for (int i = lane; i < rows * 16; i += 32)
        *reinterpret_cast<uint4*>(ring + v * kPaSlotBytes + (i & 1) * kPaHalf + (i >> 1) * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
    };
    for (int n = 0;; ++n) {
      if (!pa_all(ok && pa_wait(&b_item[n % kPaQueue], (unsigned)((n / kPaQueue) & 1), &s_failed, status))) break;
      const PaItem& it = items[n % kPaQueue];
      const int ntok = __shfl_sync(0xffffffffu, it.ntok, 0), dual = __shfl_sync(0xffffffffu, it.dual, 0),
                steps = __shfl_sync(0xffffffffu, it.j1 - it.j0, 0), dead = __shfl_sync(0xffffffffu, it.j0 ? 0 : it.dead, 0);
      if (lane == 0) mbar_arrive(&b_item_free[n % kPaQueue]);
      __syncwarp();
      if (ntok == 0) break;
      if (steps == 0) continue;
      ok &= pa_wait(&b_q, (unsigned)(nq++ & 1), &s_failed, status);
      if (n == 0 && lane == 0) FLINT_TL(6);
      pa_fence_after();
      if (dual) {
        int k = next();
        qk(0, 0, k);
        qk(1, 1, k);
        pa_commit(&b_empty[k]);
        if (steps == 1) pa_commit(&b_q_free);
        for (int j = 0; j < steps && pa_all(ok); ++j) {
          const int v = next();
          if (j + 1 < steps) k = next();
          if (j == 0 && dead > 0) clear(v, dead);
          pv(0, v, j > 0);
          if (j + 1 < steps) {
            qk(0, 0, k);
          } else {
            pa_commit(&b_o[0]);
          }
          pv(1, v, j > 0);
          pa_commit(&b_empty[v]);
          if (j + 1 < steps) {
            qk(1, 1, k);
            pa_commit(&b_empty[k]);
            if (j + 2 == steps) pa_commit(&b_q_free);
          } else {
            pa_commit(&b_o[1]);
          }
        }
      } else {
        for (int t = 0; t < 2 && t < steps; ++t) {
          const int k = next();
          qk(t, 0, k);
          pa_commit(&b_empty[k]);
          if (t + 1 == steps) pa_commit(&b_q_free);
        }
        for (int j = 0; j < steps && pa_all(ok); ++j) {
          const int t = j & 1, v = next();
          if (j == 0 && dead > 0) clear(v, dead);
          if (t) pv(1, v, j > 1);
          else pv(0, v, j > 1);
          pa_commit(&b_empty[v]);
          if (j + 2 < steps) {
            const int k = next();
            qk(t, 0, k);
            pa_commit(&b_empty[k]);
            if (j + 3 == steps) pa_commit(&b_q_free);
          } else {
            pa_commit(&b_o[t]);
          }
        }
      }
    }
  } else if (warp < 8) {
    // ---- softmax: group t of 128 threads, one row each ----
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_col = tmem + lanes + 128 * t, o_col = tmem + lanes + 256 + 128 * t;
    int s_par = 0, o_par = 0, handed = 0;                         // handed: quarters of o from group 1 to group 0 so far
    bool ok = true;
    for (int n = 0;; ++n) {
      if (!pa_all(pa_wait(&b_item[n % kPaQueue], (unsigned)((n / kPaQueue) & 1), &s_failed, status))) break;
      const PaItem it = items[n % kPaQueue];
      __syncwarp();
      if (lane == 0) mbar_arrive(&b_item_free[n % kPaQueue]);
      if (it.ntok == 0) break;
      const int per = a.per, steps = it.j1 - it.j0, row_tok = pa_token(a, row);
      const int tok = row_tok + (it.dual ? t * per : 0);
      const int qh = it.h * a.G + row - row_tok * a.G;
      const bool valid = row_tok < per && tok < it.ntok;
      int lo = 0, hi = 0;                                         // this row's keys
      if (valid) {
        if (!it.home) hi = it.pos0 + tok + 1;
        else hi = max(0, min(a.seq_lens[it.tok0 + tok], a.max_blocks * kPaPage));
        if (a.window > 0) lo = max(0, hi - a.window);
        hi = max(0, min(hi, it.end));
      }
      const bool idle = !__any_sync(0xffffffffu, valid);
      float m = -INFINITY, l = 0.f;
      const int stride = it.dual ? 1 : 2, mine0 = it.dual ? 0 : t;
      const int last_page = it.end & ~(kPaPage - 1);              // a cut last page: its tokens lie at its slot's end
      const int shift = it.end > last_page ? kPaPage - (it.end - last_page) : 0;
      for (int j = mine0; j < steps && pa_all(ok); j += stride) {
        ok &= pa_wait(&b_s[t], (unsigned)s_par, &s_failed, status);
        s_par ^= 1;
        pa_fence_after();
        if (n == 0 && j == 0 && tid == 0) FLINT_TL(7);
        if (idle) {                                               // no row of this warp is one: P may be anything
          pa_fence_before();
          if (lane == 0) {
            mbar_arrive(&b_p[2 * t]);
            mbar_arrive(&b_p[2 * t + 1]);
          }
          continue;
        }
        const int k0 = it.begin + (it.j0 + j) * kPaKeys;
        const bool hidden = __any_sync(0xffffffffu, lo > k0 || hi < k0 + kPaKeys);
        // a bit for each column whose key this row sees: up to the cut page as they are, in it behind the shift
        uint32_t see[4];
        if (hidden) {
          const int lp = min(kPaKeys, last_page - k0);
          const int a0 = lo - k0, a1 = min(hi - k0, shift ? lp : kPaKeys);
          const int c0 = shift ? max(lp, lo - k0) + shift : kPaKeys, c1 = hi - k0 + shift;
#pragma unroll
          for (int q = 0; q < 4; ++q) see[q] = pa_bits(a0 - 32 * q, a1 - 32 * q) | pa_bits(c0 - 32 * q, c1 - 32 * q);
        }
        auto hide = [&](uint32_t* r, int q) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(see[q] & (1u << i))) r[i] = 0xFF800000u;        // -inf
        };
        // First pass: the maximum.  The first 64 columns are read again below: all 128 held for both passes leave too few
        // registers for the exponentials to overlap.
        uint32_t r[4][32];
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < 4; ++q) pa_ld32(s_col + 32 * q, r[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          pa_wait_ld(r[q]);
          if (hidden) hide(r[q], q);
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            top[(i >> 1) & 3] = pa_max3(top[(i >> 1) & 3], __uint_as_float(r[q][i]), __uint_as_float(r[q][i + 1]));
        }
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const bool rise = (mx - m) * a.c > kPaRise || (m == -INFINITY && mx > -INFINITY);
        if (__any_sync(0xffffffffu, rise)) {
          const float alpha = rise ? pa_ex2((m - mx) * a.c) : 1.f;
          if (rise) m = mx;
          l *= alpha;
          if (j > mine0) {                                        // o of the steps so far
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              uint32_t o[32];
              pa_ld32(o_col + 32 * q, o);
              pa_wait_ld(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              pa_st32(o_col + 32 * q, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m * a.c;
        const uint64_t c2 = pa_two(a.c, a.c), nb2 = pa_two(-base, -base);
        uint64_t sum[2] = {0, 0};
        // Second pass, from the last columns, which are still here, to the first: 32 keys' P take the 16 columns from
        // 64 + 16 q on, whose scores have been read.
#pragma unroll
        for (int q = 3; q >= 0; --q) {
          uint32_t* x = r[q];
          if (q == 1) {
            pa_wait_ld(r[1]);
            pa_wait_ld(r[0]);
            if (hidden) hide(r[1], 1), hide(r[0], 0);
          }
          if (q == 2) pa_ld32(s_col + 32, r[1]), pa_ld32(s_col, r[0]);
          uint32_t p[16];
#pragma unroll
          for (int i = 15; i >= 0; --i) {
            const float2 y = pa_split(pa_fma2(pa_two(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), c2, nb2));
            const float p0 = pa_ex2(y.x), p1 = pa_ex2(y.y);
            sum[i & 1] = pa_add2(sum[i & 1], pa_two(p0, p1));
            p[i] = pa_pack(p0, p1);
            if (q == 0 && i == 8) {                               // all but the first 16 keys: the MMA warp starts on them
              pa_st8(s_col + 64 + 8, p + 8);
              pa_wait_st();
              pa_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&b_p[2 * t]);
            }
          }
          if (q > 0) pa_st16(s_col + 64 + 16 * q, p);
          else {
            pa_st8(s_col + 64, p);
            pa_wait_st();
            pa_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b_p[2 * t + 1]);
          }
        }
        const float2 part = pa_split(pa_add2(sum[0], sum[1]));
        l += part.x + part.y;
        if (n == 0 && j == 0 && tid == 0) FLINT_TL(8);
      }
      const bool any = mine0 < steps;
      if (any) {
        ok &= pa_wait(&b_o[t], (unsigned)o_par, &s_failed, status);
        o_par ^= 1;
        pa_fence_after();
        if (n == 0 && tid == 0) FLINT_TL(9);
      }
      if (!pa_all(ok)) break;
      // two halves of one tile: group 1 hands its (m, l, o) over, 64 columns at a time
      const bool join = !it.dual && steps > 1;
      float f0 = 1.f, f1 = 0.f;
      auto hand = [&](const uint32_t* o, int quarter) {           // group 1: 32 columns (and m, l beside the first ones)
        if (handed > 0) ok &= pa_wait(&b_take, (unsigned)((handed - 1) & 1), &s_failed, status);
        if (quarter == 0) s_ml[row] = make_float2(m, l);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          sx[row * 8 + ((i + row) & 7)] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                      __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
        __syncwarp();
        if (lane == 0) mbar_arrive(&b_hand);
        ++handed;
      };
      auto take = [&](uint32_t* o, int quarter) {                 // group 0
        ok &= pa_wait(&b_hand, (unsigned)(handed & 1), &s_failed, status);
        if (quarter == 0) {
          const float2 other = s_ml[row];
          const float mm = fmaxf(m, other.x);
          f0 = m == -INFINITY ? 0.f : pa_ex2((m - mm) * a.c);
          f1 = other.x == -INFINITY ? 0.f : pa_ex2((other.x - mm) * a.c);
          l = l * f0 + other.y * f1;
          m = mm;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 x = sx[row * 8 + ((i + row) & 7)];
          o[4 * i] = __float_as_uint(__uint_as_float(o[4 * i]) * f0 + x.x * f1);
          o[4 * i + 1] = __float_as_uint(__uint_as_float(o[4 * i + 1]) * f0 + x.y * f1);
          o[4 * i + 2] = __float_as_uint(__uint_as_float(o[4 * i + 2]) * f0 + x.z * f1);
          o[4 * i + 3] = __float_as_uint(__uint_as_float(o[4 * i + 3]) * f0 + x.w * f1);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&b_take);
        ++handed;
      };
      if (it.dual || t == 0 || join) {
        const bool writes = valid && (it.dual || t == 0);
        const int64_t slot_row = it.out >= 0 ? (int64_t)it.out * 256 + (it.dual ? t * 128 : 0) + row : 0;
        const int64_t home_row = (int64_t)(it.home * a.batch + it.tok0 + tok) * a.Hkv * a.G + qh;
        bf16* dst = a.out + (int64_t)(it.tok0 + tok) * a.out_stride + qh * kPaD;
        float inv = 1.f;
#pragma unroll 1
        for (int quarter = 0; quarter < 4; ++quarter) {
          uint32_t o[32];
          if (any) {
            pa_ld32(o_col + 32 * quarter, o);
            pa_wait_ld(o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
          if (join) {
            if (t == 1) hand(o, quarter);
            else take(o, quarter);
          }
          if (!it.dual && t == 1) continue;
          if (quarter == 0) {
            if (it.out != PA_FINAL) {
              if (writes) *(it.out >= 0 ? a.ml + slot_row : a.home_ml + home_row) = make_float2(m, l);
            } else {
              float den = l;
              if (a.sinks && valid && m != -INFINITY) den += pa_ex2(a.sinks[qh] * kPaLog2e - m * a.c);
              inv = 1.0f / den;
            }
          }
          if (it.out == PA_FINAL) {
            if (writes) {
              uint32_t w[16];
#pragma unroll
              for (int i = 0; i < 16; ++i)
                w[i] = l == 0.f ? 0u : pa_pack(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
              pa_store64(dst + 32 * quarter, w, a.wide);
            }
          } else if (writes && l != 0.f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 x = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                           __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
              if (it.out >= 0) a.o[((int64_t)it.out * 32 + 8 * quarter + i) * 256 + (it.dual ? t * 128 : 0) + row] = x;
              else a.home_o[home_row * 32 + 8 * quarter + i] = x;
            }
          }
        }
      }
      if (n == 0 && tid == 0) FLINT_TL(10);
      pa_fence_before();                                          // o has been read: the next item's products may follow p
    }
  }
  pa_fence_before();
  __syncthreads();
  if (s_failed) {                                                 // nothing may be in flight when the block's memory goes
    if (warp == 8) {
      for (int k = max(0, s_sent[0] - kPaSlots); k < s_sent[0]; ++k) pa_drain(&b_full[k % kPaSlots], (unsigned)(k / kPaSlots & 1));
      if (s_sent[1]) pa_drain(&b_q, (unsigned)(s_sent[1] - 1 & 1));
    } else if (warp == 9) {
      pa_commit(&b_end);
      pa_drain(&b_end, 0);
    }
    __syncthreads();
  }
  if (tid == 0) FLINT_TL(11);
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)kPaTmem) : "memory");
}

// Joins the parts of the rows that were cut, the prefix's first, in the order of their keys: 8 / Groups rows at a time, a
// thread per row, quad of columns and group of parts (every Groups-th); the groups' sums are joined in their order.  Prompts:
// kPaJoin blocks for each item that was cut; streams: a block for 8 / Groups of their rows.  Parts' (m, l), then their o, are
// loaded four at a time, since what this costs is the latency of L2.
constexpr int kPaJoin = 8;
template <int Groups>
__global__ void __launch_bounds__(256, 4) paged_join_kernel(const PagedAttnArgs a, int blocks) {
  constexpr int kRows = 8 / Groups;
  __shared__ float4 s_o[Groups > 1 ? 256 : 1];
  __shared__ float2 s_ml[Groups > 1 ? 8 : 1];
  pdl_wait();
  const int sub = threadIdx.x & 7, quad = threadIdx.x >> 3, row_in = sub % kRows, group = sub / kRows, per = a.per;
  float m, l;
  float4 o;
  auto add = [&](float2 ml, float4 x) {
    if (ml.y == 0.f) return;
    const float mm = fmaxf(m, ml.x), f0 = m == -INFINITY ? 0.f : pa_ex2((m - mm) * a.c),
                f1 = ml.x == -INFINITY ? 0.f : pa_ex2((ml.x - mm) * a.c);    // (of NaN: 0 times it stays NaN)
    l = l * f0 + ml.y * f1;
    o.x = o.x * f0 + x.x * f1, o.y = o.y * f0 + x.y * f1, o.z = o.z * f0 + x.z * f1, o.w = o.w * f0 + x.w * f1;
    m = mm;
  };
  auto parts = [&](int first, int last, int at, int g) {          // at: the token's place in its item
    const int row = at / per * kPaM + at % per * a.G + g;
    if (first < 0 || last >= blocks || at < 0 || at >= 2 * per) return;
    for (int c0 = first + group; c0 <= last; c0 += 4 * Groups) {
      float2 ml[4];
      float4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + i * Groups;
        ml[i] = c <= last ? __ldcg(a.ml + (2 * c + (c == first)) * 256 + row) : make_float2(-INFINITY, 0.f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + i * Groups;
        if (ml[i].y != 0.f) x[i] = __ldcg(a.o + ((2 * c + (c == first)) * 32 + quad) * 256 + row);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) add(ml[i], x[i]);
    }
  };
  auto begin = [&]() { m = -INFINITY, l = 0.f, o = make_float4(0.f, 0.f, 0.f, 0.f); };
  auto finish = [&](bool valid, int64_t tok, int qh) {            // every thread of the block
    if (Groups > 1) {
      if (quad == 0) s_ml[sub] = make_float2(m, l);
      s_o[quad * 8 + sub] = o;
      __syncthreads();
      if (group == 0)
#pragma unroll
        for (int k = 1; k < Groups; ++k) add(s_ml[k * kRows + row_in], s_o[quad * 8 + k * kRows + row_in]);
      __syncthreads();
    }
    if (!valid || group != 0) return;
    float den = l;
    if (a.sinks && m != -INFINITY) den += pa_ex2(a.sinks[qh] * kPaLog2e - m * a.c);
    const float inv = l == 0.f ? 0.f : 1.0f / den;
    const uint2 w = make_uint2(pa_pack(o.x * inv, o.y * inv), pa_pack(o.z * inv, o.w * inv));
    reinterpret_cast<uint2*>(a.out + tok * a.out_stride + qh * kPaD)[quad] = w;
  };
  if (!a.group_starts) {
    const PaSplit e = a.split[blockIdx.x / kPaJoin];
    const int rows = e.ntok * a.G;
    for (int r0 = (int)(blockIdx.x % kPaJoin) * kRows; r0 < rows; r0 += kRows * kPaJoin) {
      const int r = r0 + row_in, at = pa_token(a, r), g = r - at * a.G;
      begin();
      if (r < rows) parts(e.first, e.last, at, g);
      finish(r < rows, e.tok0 + at, e.h * a.G + g);
    }
    return;
  }
  const int64_t r = (int64_t)blockIdx.x * kRows + row_in;
  const int Hq = a.Hkv * a.G;
  const bool valid = r < (int64_t)a.batch * Hq;
  const int tok = valid ? (int)(r / Hq) : 0, qh = valid ? (int)(r - (int64_t)tok * Hq) : 0, h = qh / a.G;
  const PaRecord own = a.rec[(int64_t)tok * a.Hkv + h];
  const bool todo = valid && own.first != PA_FINAL;
  auto from = [&](const PaRecord& rec, int home) {
    if (rec.first != PA_HOME) {
      parts(rec.first, rec.last, tok - rec.tok0, qh - h * a.G);
    } else if (group == 0) {
      const int64_t row = (int64_t)(home * a.batch + tok) * Hq + qh;
      const float2 ml = a.home_ml[row];
      if (ml.y != 0.f) add(ml, a.home_o[row * 32 + quad]);
    }
  };
  begin();
  if (todo) {
    if (own.prefix) from(a.rec[((int64_t)a.batch + tok) * a.Hkv + h], 1);
    from(own, 0);
  }
  finish(todo, tok, qh);
}

}  // namespace flint

using namespace flint;

int64_t flint::status_offset_paged_attention() { return (int64_t)offsetof(PagedAttnWorkspace, status); }

// The workspace: status, the blocks' cut items, (m, l) and o of their slots (two per block); with shared prefixes also the
// homes and the records.  Every call writes what it reads.
struct PaLayout {
  int64_t split, ml, o, rec, home_ml, home_o, bytes;
};
static PaLayout pa_layout(int64_t blocks, int64_t records, int64_t homes) {
  PaLayout w;
  w.split = sizeof(PagedAttnWorkspace);
  w.ml = w.split + (blocks * (int64_t)sizeof(PaSplit) + 127) / 128 * 128;
  w.o = w.ml + blocks * 512 * (int64_t)sizeof(float2);
  w.rec = w.o + blocks * 512 * 32 * (int64_t)sizeof(float4);
  w.home_o = w.rec + (records * (int64_t)sizeof(PaRecord) + 127) / 128 * 128;
  w.home_ml = w.home_o + homes * 32 * (int64_t)sizeof(float4);
  w.bytes = w.home_ml + homes * (int64_t)sizeof(float2);
  return w;
}
static int pa_blocks() {
  const int n = num_sms();
  return n > 0 ? n : 148;
}

static int paged_attn(const void* q, int64_t q_stride, const void* kv, int64_t num_blocks, int64_t Hkv, int64_t stride_block,
                      int64_t stride_head, const int32_t* bt, int64_t bt_stride, int64_t max_blocks, const int32_t* cu_seqlens,
                      const int32_t* seq_lens, const int32_t* group_starts, const int32_t* prefix_lens, int64_t groups,
                      const float* sinks, int64_t window, float scale, int64_t batch, int64_t tokens, int64_t Hq, void* out,
                      int64_t out_stride, void* ws, int pdl, void* stream) {
  if (!q || !kv || !bt || !seq_lens || !out || !ws) return FLINT_ERR_ARGUMENT;
  if (window < 0 || out == q || !(scale > 0.f) || !(scale < 1e30f)) return FLINT_ERR_ARGUMENT;
  if (batch < 1 || batch > (1 << 20) || tokens < 1 || tokens > (1 << 24) || Hkv < 1 || Hkv > 128 || Hq < 1 || Hq % Hkv != 0 ||
      Hq / Hkv > 8 || num_blocks < 1 || num_blocks >= INT32_MAX || max_blocks < 1 || max_blocks > (1 << 25) || bt_stride < 0 ||
      q_stride < Hq * kPaD || out_stride < Hq * kPaD || stride_head < kPaPage * 2 * kPaD || stride_block < kPaPage * 2 * kPaD)
    return FLINT_ERR_SHAPE;
  if (!aligned(kv, 16) || stride_block % 8 != 0 || stride_head % 8 != 0 || !aligned(out, 16) || !aligned(q, 16) ||
      q_stride % 8 != 0 || out_stride % 8 != 0 || !aligned(ws, 16))
    return FLINT_ERR_ALIGN;
  const int blocks = num_sms();
  if (blocks <= 0) return FLINT_ERR_DEVICE;
  const int G = (int)(Hq / Hkv), per = kPaM / G;
  CUtensorMap mq, mkv;
  const uint64_t qd[3] = {kPaD, (uint64_t)Hq, (uint64_t)tokens}, qs[2] = {kPaD * 2, (uint64_t)q_stride * 2};
  const uint32_t qb[3] = {64, (uint32_t)G, (uint32_t)per};
  int rc = encode_bf16_3d(&mq, q, qd, qs, qb);
  if (rc) return rc;
  const uint64_t kd[4] = {2 * kPaD, kPaPage, (uint64_t)Hkv, (uint64_t)num_blocks};
  const uint64_t ks[3] = {2 * kPaD * 2, (uint64_t)stride_head * 2, (uint64_t)stride_block * 2};
  const uint32_t kb[4] = {64, kPaPage, 1, 1};
  rc = encode_bf16_4d(&mkv, kv, kd, ks, kb);
  if (rc) return rc;
  PagedAttnArgs a = {};
  a.block_tables = bt; a.bt_stride = bt_stride; a.max_blocks = (int)max_blocks; a.cu_seqlens = cu_seqlens;
  a.seq_lens = seq_lens; a.group_starts = group_starts; a.prefix_lens = prefix_lens; a.groups = (int)groups; a.sinks = sinks;
  a.window = window >= max_blocks * kPaPage ? 0 : (int)window;    // (a window over every length hides nothing)
  a.batch = (int)batch; a.tokens = (int)tokens; a.Hkv = (int)Hkv; a.G = G;
  a.num_blocks = (int)num_blocks; a.per = per; a.inv_g = (65536 + G - 1) / G; a.c = scale * kPaLog2e; a.out = (bf16*)out; a.out_stride = out_stride;
  a.wide = aligned(out, 32) && out_stride % 16 == 0;
  a.ws = static_cast<PagedAttnWorkspace*>(ws);
  const PaLayout w = pa_layout(blocks, group_starts ? 2 * batch * Hkv : 0, group_starts ? 2 * batch * Hq : 0);
  uint8_t* base = static_cast<uint8_t*>(ws);
  a.split = reinterpret_cast<PaSplit*>(base + w.split);
  a.rec = reinterpret_cast<PaRecord*>(base + w.rec);
  a.ml = reinterpret_cast<float2*>(base + w.ml);
  a.o = reinterpret_cast<float4*>(base + w.o);
  a.home_ml = reinterpret_cast<float2*>(base + w.home_ml);
  a.home_o = reinterpret_cast<float4*>(base + w.home_o);
  static std::atomic<uint64_t> ready{0};                          // devices whose shared-memory limit is raised
  int dev = 0;
  num_sms(&dev);
  if (!(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    rc = record_cuda(cudaFuncSetAttribute(paged_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPaSmem),
                     FLINT_ERR_LAUNCH);
    if (rc) return rc;
    ready.fetch_or(uint64_t(1) << dev);
  }
  rc = launch(paged_attn_kernel, dim3((unsigned)blocks), dim3(kPaThreads), kPaSmem, stream, pdl, mq, mkv, a);
  if (rc) return rc;
  // A prompt's item is cut between its steps, and tables of eight pages hold one step (17 tokens: 10.9 us on the device
  // without the join, 12.9 with it).
  if (!group_starts && max_blocks * kPaPage <= kPaKeys) return FLINT_OK;
  // Four groups share a row's parts where one pass of blocks then takes all rows, since each pass costs a chain of loads.
  // Streams: their blocks of two rows are resident at once (four an SM).  32 heads on 4 KV heads and a 6,048-token prefix, four
  // groups / one: 256 rows 22.7 / 26.2 us a call, 1,024 rows 26.7 / 28.2, 2,048 rows 35.0 / 32.4, 4,096 rows 53 / 45.
  // Prompts: an item's eight blocks of two rows hold all that a KV head has.  Behind 6,057 tokens, 8 rows 19.4 / 22.5 us,
  // 32 rows 25.6 / 23.0, 64 rows 37.7 / 24.2.
  const int64_t rows = (group_starts ? batch : tokens) * Hq;
  const int per_block = (group_starts ? rows <= 2 * 4 * blocks : tokens * G <= 2 * kPaJoin) ? 2 : 8;
  const dim3 grid((unsigned)(group_starts ? (rows + per_block - 1) / per_block : (int64_t)blocks * kPaJoin));
  return per_block == 2 ? launch(paged_join_kernel<4>, grid, dim3(256), 0, stream, pdl, a, blocks)
                        : launch(paged_join_kernel<1>, grid, dim3(256), 0, stream, pdl, a, blocks);
}

extern "C" int64_t flint_prefill_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t num_q_heads,
                                                           int64_t num_kv_heads) {
  if (batch < 1 || tokens < 1 || num_q_heads < 1 || num_kv_heads < 1) return -1;
  return pa_layout(pa_blocks(), 0, 0).bytes;
}

extern "C" int flint_prefill_attention(const void* q, int64_t q_stride_t, const void* kv_cache, int64_t num_blocks,
                                       int64_t num_kv_heads, int64_t stride_block, int64_t stride_head,
                                       const int32_t* block_tables, int64_t bt_stride, int64_t max_blocks,
                                       const int32_t* cu_seqlens, const int32_t* seq_lens, const float* sinks,
                                       int64_t window, float scale, int64_t batch, int64_t tokens, int64_t num_q_heads,
                                       void* out, int64_t out_stride_t, void* workspace, int pdl, void* stream) {
  if (!cu_seqlens) return FLINT_ERR_ARGUMENT;
  return paged_attn(q, q_stride_t, kv_cache, num_blocks, num_kv_heads, stride_block, stride_head, block_tables, bt_stride,
                    max_blocks, cu_seqlens, seq_lens, nullptr, nullptr, 0, sinks, window, scale, batch, tokens, num_q_heads,
                    out, out_stride_t, workspace, pdl, stream);
}

extern "C" int64_t flint_shared_prefix_attention_workspace_bytes(int64_t batch, int64_t groups, int64_t num_q_heads,
                                                                 int64_t num_kv_heads) {
  if (batch < 1 || groups < 1 || num_q_heads < 1 || num_kv_heads < 1) return -1;
  return pa_layout(pa_blocks(), 2 * batch * num_kv_heads, 2 * batch * num_q_heads).bytes;
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
  return paged_attn(q, q_stride_b, kv_cache, num_blocks, num_kv_heads, stride_block, stride_head, block_tables, bt_stride,
                    max_blocks, nullptr, seq_lens, group_starts, prefix_lens, groups, sinks, window, scale, batch, batch,
                    num_q_heads, out, out_stride_b, workspace, pdl, stream);
}

FLINT_TL_READER(flint_timeline_paged_attention)
