// packed_attn.cuh -- exact attention of a packed batch: whole prompts, chunks
// of prompts and single tokens of many sequences in one launch, K/V packed or
// in slots, optionally behind a prefix that all sequences share.
//
// For sequence b with nq query tokens and n keys, query i of head h:
//   out = sum_j w_j V_j / sum_j w_j,  w_j = exp(scale q . K_j),
// over the keys j it may see (causal: j <= n - nq + i; else all n), and, with
// a shared prefix, over all prefix keys too.  A query that sees no key gives 0.
//
// Rows.  A tile has 128 rows = TMEM lanes: TT = 128 / G tokens times the G
// query heads of one KV head (row = token * G + head in group), so K and V are
// read once for the group and a single token still fills G rows.  An item is
// (up to 2 TT query tokens, one KV head) against its key tiles of 128 tokens.
//
// Work split.  Lengths live on the device only; every CTA derives the same
// schedule from them (packed_schedule.cuh): the work of all items forms one
// line that the CTAs, one per SM, cut into equal shares.  An item cut by a
// share's border leaves pieces (reference point, sum and unnormalised output,
// fp32) in the workspace.  A CTA takes the item that earlier CTAs began last,
// and the one that holds an item's last piece joins all of them in CTA order:
// no atomics on results, the same result each run.  It waits for marks of
// lower CTAs only, which never wait for it.  With a shared prefix, rows have
// two items and k_packed_combine_rows joins all their parts.
//
// One CTA, 384 threads: warps 0-3 and 4-7 are the softmax of tile slots 0 and
// 1 (a thread owns a row), warps 8 and 11 load (TMA; K and V, and Q), warp 9
// issues the MMAs, warp 10 walks the schedule into a ring of item descriptors.
// All items of a CTA form one stream of tasks u, task u on slot u % 2: a
// two-tile item is (tile 0, key tile j), (tile 1, key tile j) for each j, the
// two sharing K and V; a one-tile item is its key tiles in turn, joined over
// the slots in registers at its end, and an item of one key tile takes one
// slot and leaves the other to the next item.  The MMA warp issues S of task u + 2 behind P V of task u,
// across item borders, so one slot's products run under the other's softmax
// and an item's epilogue under the next one's scores.  Per task:
//   S = Q K^T    tcgen05.mma kind::f16 into 128 fp32 TMEM columns
//   P = 2^(S scale log2 e - m)   one thread per row, rounded to the input
//                type, in tensor memory (64 columns)
//   O += P V     tcgen05.mma with P as the tensor-memory A operand
// The reference point m is raised only when a score passes it by more than a
// step (log2 units), and normalising by the same m is exact.  P is rounded to
// the input type because the tensor cores multiply in it: half a step of that
// type relative to each weight.  bf16 has the range of fp32: m is the running
// maximum, raised by steps above 8.  f16 is subnormal below 2^-14, and a row with
// one dominant key may have most of its mass in thousands of weights that small:
// m lies 11 below the running maximum and is raised by steps above 4 (P up to
// 2^15), so a weight keeps its half step down to 2^-25 of the largest, and one
// below that is off by 2^-36 of the largest at most.  Sums, maxima and O are fp32.
//
// Rows behind a sequence's end: their scores are masked by selection (any bit
// pattern, NaN included, drops out), and the V rows of the last, partial
// 16-token step are zeroed in shared memory before the product, steps past it
// are not issued.  Rows of the sequence itself that the causal mask hides take
// part in an item's products, with weight 0, up to the end of its last key tile:
// only a value that is not finite shows, at queries up to 2 TT + 126 tokens ahead.
//
// What bounds it (B200, 32 query / 8 KV heads of 128 dims, bf16): prompts by a
// slot's chain of scores, softmax and products, 3,500 cycles a two-tile step
// (fitted over 1 to 4 items of 8 to 64 key tiles a CTA) against 2,048 of
// products, and at 16K tokens by the board's power (1.83 ms = 1,200 TFLOP/s in a
// graph, 2.02 = 1,091 called in turn); single tokens by memory (8 at 16K keys: 94
// us, 5.7 TB/s of K and V); short calls by latency, 12 us besides the steps.
// Rolled loops and one copy of each role's code are deliberate: with unrolled
// roles (20 KB more) the instruction cache missed 20 % of its requests and ragged
// prompts took 240 us, against 184 when the roles were made compact (160 now).
#pragma once
#include "packed_schedule.cuh"
#include "prefill.cuh"

namespace hokv {

constexpr int PA_THREADS = 384;
constexpr int PA_ROWS = 128;        // rows of a tile
// Registers of a thread: 168 at launch, then 200 for the 8 softmax warps, which hold a row of 128 scores, and 104 for
// the other 4.  The sum may not pass what the block was launched with, or the raise would wait for good: the launch
// checks the build's count.  (208 and 88: 1 to 3 % slower, 192 and 120: 0.5 %.)
constexpr int PA_REGS = 168, PA_REGS_ROW = 200, PA_REGS_ISSUE = 104;
static_assert(256 * PA_REGS_ROW + 128 * PA_REGS_ISSUE <= PA_THREADS * PA_REGS, "register split");
constexpr int PA_QUEUE = 8;         // item descriptors in flight
constexpr float PA_LOG2E = 1.4426950408889634f;

template <int D>
struct PaGeo {
  static constexpr int NB = D / 64;                       // 64-dim column blocks
  // Tensor memory: S of the slots in columns 0 and 128, O in 256 and 384; P in 64 columns of its own behind a 64-dim
  // O, over S otherwise.
  static constexpr int P0 = D == 64 ? 256 + 64 : 0;
  static constexpr int Q_BYTES = PA_ROWS * D * 2;         // one query tile
  static constexpr int KV_BYTES = PA_BN * D * 2;          // one K or V tile
  static constexpr int STAGES = D == 64 ? 8 : 4;          // ring of K and V tiles
  static constexpr int OUT_BYTES = 8 * 4096;              // 32 rows x 64 dims of O per softmax warp, on their way out
  static constexpr int SMEM = 2 * Q_BYTES + STAGES * KV_BYTES + OUT_BYTES + 2048;
};

struct alignas(64) PaMaps {
  CUtensorMap q, k, v, out, pk, pv;
};

struct PaP : PaSched {
  void* out;
  int64_t ost, osh;              // output element strides (token, head)
  int Hq, G, D, zero_tail, tma_out;   // tma_out: tokens of a warp's 32 rows, 0 when they are not whole tokens
  float sl2;                     // scale * log2(e)
  float raw_step;                // f16: the step above which m is raised, as a score stands in S
  int k_t, k_h, k_b, v_t, v_h, v_b, pk_t, pk_h, pk_b, pv_t, pv_h, pv_b;   // coordinate slots of the maps
  float2* ml;                    // [n_ctas][2][256] (m, sum)
  float4* o;                     // [n_ctas][2][D / 4][256]
  unsigned long long* ready;     // [n_ctas][2][8] the call's token when 32 rows of a piece are written, then 0 again
  unsigned long long token;      // this call's; a replayed call's marks also carry g_pa_failures
  int2* tok_info;                // prefix only: [2][T][Hkv] (first | last CTA << 8 or -1: row-wise, token in item)
  float2* row_ml;                // prefix only: [2][T][Hq]
  float4* row_o;                 // prefix only: [2][T][Hq][D / 4]
};

// The item that this CTA joins at its end: the one whose last piece it holds.
struct PaJoinItem {
  int n, first, tok0, n_tok, hk;   // pieces (0: none to join) from CTA `first` on, rows
  int left;                        // softmax warps that have joined their part
  unsigned long long token;        // what this launch's marks hold
};
// CTAs that gave up, since the library was loaded on the device.  One that did may leave marks behind, and a graph
// replays its call's token: the marks of a launch carry both, so that later replays do not take old marks for theirs.
// Every CTA reads the count at its start.  It only changes while a call fails; a call on another stream that starts at
// that moment may see both values, and then its own waits run out.
__device__ unsigned long long g_pa_failures = 0;
// Workspace slot of piece i of an item whose first one is CTA `first`'s.
__device__ __forceinline__ int pa_slot(int first, int i) { return (first + i) * 2 + (i == 0 ? 1 : 0); }

// A reader's place in the CTA's task stream: item fields, its task j of `tasks`.
struct PaCursor {
  int it = 0, n = 0, two = 0, tasks = 0, j = 0, left = 0, src = 0, hk = 0, tok0 = 0, slot = 0, row0 = 0;
  bool done = false;
};

// ---- signals kept back (instrumented build only) --------------------------------
// Built with -DHOKV_HOLD, hokv_hold() makes CTAs 3, 11, 19, ... keep back signals that other roles or CTAs wait for,
// and shortens the packed attention's waits, so that a test sees them run out.  The product build compiles none of it.
enum { PA_HOLD_MARK = 1, PA_HOLD_P = 2, PA_HOLD_STOP = 4 };   // a piece's marks; the first warp's weights; the stream's end
#ifdef HOKV_HOLD
__device__ int g_hold = 0;
__device__ __forceinline__ int pa_hold() { return *reinterpret_cast<volatile int*>(&g_hold); }
__device__ __forceinline__ bool pa_held(int what) { return (pa_hold() & what) && blockIdx.x % 8 == 3; }
__device__ __forceinline__ unsigned long long pa_limit(unsigned long long ns) { return pa_hold() ? ns / 50 : ns; }
#else
__device__ __forceinline__ constexpr bool pa_held(int) { return false; }
__device__ __forceinline__ constexpr unsigned long long pa_limit(unsigned long long ns) { return ns; }
#endif

// ---- barriers ----------------------------------------------------------------

__device__ __forceinline__ bool pa_try_wait(uint32_t bar, unsigned parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// Bounded wait of every calling thread; the first that gives up marks the CTA
// aborted, and every other wait of the CTA then ends too.
__device__ __forceinline__ bool pa_wait_more(uint32_t bar, unsigned parity, volatile uint32_t* abort_flag) {
  const unsigned long long t0 = global_ns();
  while (!pa_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (global_ns() - t0 > pa_limit(TC_WAIT_NS)) {
      if (atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0u) dev_flag(HOKV_ERR_TIMEOUT);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool pa_wait(uint64_t* bar, unsigned parity, volatile uint32_t* abort_flag) {
  return pa_try_wait(smem_u32(bar), parity) || pa_wait_more(smem_u32(bar), parity, abort_flag);
}
// The whole warp's wait: near the limit its lanes may see different ends, and all of them go on or none does.
__device__ __forceinline__ bool pa_wait_warp(uint64_t* bar, unsigned parity, volatile uint32_t* abort_flag) {
  return __all_sync(0xffffffffu, pa_wait(bar, parity, abort_flag));
}

// The same for a mark in global memory, which another CTA sets: shares are
// equal but a long call's CTAs may end some way apart.
constexpr unsigned long long PA_MARK_NS = 10 * TC_WAIT_NS;
__device__ __forceinline__ bool pa_wait_ready(const unsigned long long* mark, unsigned long long token,
                                              volatile uint32_t* abort_flag) {
  const unsigned long long t0 = global_ns();
  while (true) {
    if (*abort_flag) return false;
    unsigned long long v;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(mark) : "memory");
    if (v == token) return true;
    if (global_ns() - t0 > pa_limit(PA_MARK_NS)) {
      if (atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0u) dev_flag(HOKV_ERR_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ void store_release(unsigned long long* p, unsigned long long v) {
  asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

__device__ __forceinline__ void pa_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The MMA warp runs as a whole with warp-uniform values and one elected lane
// issues: operands that the compiler cannot prove uniform cost a loop of votes
// per instruction (130 cycles for each MMA, twice the 128 x 128 x 16 product
// itself).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
  return e;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Halves of umma_desc_sw (128-byte swizzle): the low one holds address and
// leading byte offset, the high one the stride byte offset and constants.
__device__ __forceinline__ uint32_t pa_desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4) << 16; }
constexpr uint32_t PA_DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;

// kind::f16 MMA, A and B in shared memory.
__device__ __forceinline__ void pa_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "n"(PA_DESC_HI)
      : "memory");
}
// The same with A in tensor memory (16-bit pairs per column).
__device__ __forceinline__ void pa_mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc), "n"(PA_DESC_HI)
      : "memory");
}

// 16 packed columns of this thread's lane into tensor memory, without waiting.
__device__ __forceinline__ void tmem_st16_nw(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// Waits for the thread's tensor-memory loads; v is not used before.
__device__ __forceinline__ void tmem_wait_ld32(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
// Columns from `left` on do not count.
__device__ __forceinline__ void mask32(float (&v)[32], int left) {
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : -INFINITY;
}
// x f + a for 8 fp32 columns of this thread's lane.
__device__ __forceinline__ void tmem_fma8(uint32_t taddr, float f, float a) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
  tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = __float_as_uint(fmaf(__uint_as_float(r[j]), f, a));
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));   // NaN wins
  return d;
}

// Where a row's reference point m lies below its largest score, and how far a score may pass m before m is raised.
template <typename T>
struct PaRange {
  static constexpr bool NARROW = std::is_same<T, __half>::value;   // weights may leave the type's range
  static constexpr float LIFT = NARROW ? 11.f : 0.f, MOST = NARROW ? 15.f : 8.f;
  // From here on fp32 holds m too coarsely for f16 weights (off by a quarter at 2^22): scores are taken relative to the
  // one that set m before they are scaled.
  static constexpr float FAR = 0x1p22f;
};

// One 32-byte store (a whole sector): a thread's row of O.
__device__ __forceinline__ void st_global_32(void* p, const uint32_t* u) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]),
               "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}

// ---- the kernel ----------------------------------------------------------------

template <int D, typename T>
__global__ void __launch_bounds__(PA_THREADS, 1) k_packed_attn(const __grid_constant__ PaMaps maps, const PaP p) {
  using PG = PaGeo<D>;
  using PR = PaRange<T>;
  constexpr int ST = PG::STAGES;
  constexpr int BF = std::is_same<T, __half>::value ? 0 : 1;
  extern __shared__ __align__(1024) unsigned char pa_smem[];
  unsigned char* sQ = pa_smem;
  unsigned char* sKV = sQ + 2 * PG::Q_BYTES;
  unsigned char* sOut = sKV + ST * PG::KV_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sOut + PG::OUT_BYTES);
  uint64_t* q_full = bars;                 // [2] query buffers: TMA bytes
  uint64_t* q_empty = bars + 2;            // [2] MMA commit after the last S that reads the buffer
  uint64_t* s_full = bars + 4;             // [2] MMA commit
  uint64_t* p_full = bars + 6;             // [2] 4 softmax warps
  uint64_t* o_full = bars + 8;             // [2] MMA commit after the slot's last P V of an item
  uint64_t* o_empty = bars + 10;           // [2] 4 softmax warps: O read
  uint64_t* ml_full = bars + 12;           // 4 warps of slot 1: (m, l) in shared memory
  uint64_t* it_full = bars + 13;           // [PA_QUEUE] scheduler
  uint64_t* it_empty = it_full + PA_QUEUE; // [PA_QUEUE] 2 load + MMA + 8 softmax warps
  uint64_t* kv_full = it_empty + PA_QUEUE; // [ST] TMA bytes
  uint64_t* kv_empty = kv_full + ST;       // [ST] MMA commit
  uint64_t* mma_done = kv_empty + ST;      // MMA commit at the end of a CTA that gave up
  static_assert(14 + 2 * PA_QUEUE + 2 * ST <= 48, "barriers");
  uint32_t* ctl = reinterpret_cast<uint32_t*>(bars + 48);                   // [0] tmem base, [1] abort
  PaItem* queue = reinterpret_cast<PaItem*>(bars + 49);                     // [PA_QUEUE]
  float2* s_ml = reinterpret_cast<float2*>(bars + 49 + PA_QUEUE * sizeof(PaItem) / 8);   // [128] slot 1's (m, l)
  PaJoinItem* s_join = reinterpret_cast<PaJoinItem*>(s_ml + 128);
  static_assert((49 + 128) * 8 + PA_QUEUE * sizeof(PaItem) + sizeof(PaJoinItem) <= 2048, "control block");
  volatile uint32_t* abort_flag = &ctl[1];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(ctl)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 0) {
    mbar_init(ml_full, 4);
    mbar_init(mma_done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < PA_QUEUE; ++i) {
      mbar_init(&it_full[i], 1);
      mbar_init(&it_empty[i], 11);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    ctl[1] = 0u;
    s_join->n = s_join->left = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tmem = 0;   // all 512 columns are this CTA's: the base is column 0
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int TT = p.TT, G = p.G;

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PA_REGS_ROW));
    // ---- softmax of tile slot sl, one row per thread ----------------------------
    const int sl = warp >> 2, row = tid & 127;
    const int row_tok = row / G, row_g = row - row_tok * G;
    const int first_tok = ((warp & 3) * 32) / G;   // lowest token of this warp's rows
    const uint32_t lane_sel = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lane_sel + (uint32_t)(sl * 128);
    const uint32_t o_addr = tmem + lane_sel + (uint32_t)(256 + sl * 128);
    const uint32_t p_addr = tmem + lane_sel + (uint32_t)(PG::P0 + sl * 128);
    // rows of out on 32-byte boundaries and in whole 16-element steps: 32-byte stores
    const bool wide = p.D % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) % 32 | (uint64_t)(p.ost % 16) | (uint64_t)(p.osh % 16)) == 0;
    unsigned s_ph = 0, o_ph = 0, o1_ph = 0, ml_ph = 0;   // phases of s_full[sl], o_full[sl]; slot 0: o_full[1], ml_full
    int u = 0;   // tasks of the items so far
    bool ok = true;
    for (int it = 0; ok; ++it) {
      const int qi = it % PA_QUEUE;
      ok = pa_wait_warp(&it_full[qi], (unsigned)((it / PA_QUEUE) & 1), abort_flag);
      if (!ok) break;
      const volatile PaItem& w = queue[qi];   // read again where needed: registers are short in the loop
      if (w.out_mode == PA_STOP) break;
      const bool two = w.n_tok > TT;
      const int n = w.j1 - w.j0;
      if (two) u = (u + 1) & ~1;                           // a two-tile item begins on slot 0
      const int skip = two ? 0 : (sl - u) & 1;             // this slot's first key tile
      const int mine = two ? n : (n - skip + 1) >> 1;      // its number of key tiles
      const bool join = !two && n > 1;                     // both slots hold parts of the same rows
      const bool other = two || join || ((u & 1) != sl);   // the other slot has a part of this item
      u += two ? 2 * n : n;
      const bool warp_ok = first_tok < TT && (two ? sl * TT : 0) + first_tok < w.n_tok;   // any row of the warp in use
      // keys this row sees, and the least such limit of the warp, counted from the slot's key tile
      int lim = min(w.kv_len, w.pos0 + (two ? sl * TT : 0) + row_tok + 1) - (w.j0 + skip) * PA_BN;
      int wlim = __shfl_sync(0xffffffffu, lim, 0);
      const int step = two ? PA_BN : 2 * PA_BN;
      auto item_done = [&]() {
        __syncwarp();
        if (lane == 0) pa_arrive(&it_empty[qi]);
      };
      float m_run = -INFINITY, l_run = 0.f, nm = 0.f;        // nm: what is added to a scaled score
      float raw_most = -INFINITY, m_raw = 0.f;               // f16: scores above this raise m; what is taken from scores
      bool any_far = false;                                  // in the warp
      for (int i = 0; i < mine; ++i, lim -= step, wlim -= step) {
        // no vote here (1 % of a prompt): a CTA that gave up runs through the item on what is there, and drops it at its end
        (void)pa_wait(&s_full[sl], s_ph, abort_flag);
        __syncwarp();
        s_ph ^= 1;
        tc_fence_after();
        if (warp_ok) {
          // The row stays in registers between its maximum and its weights (a pass from tensor memory for each: 16K
          // prompt 1,862 us against 1,772, 4 x 4,096 tokens of 64 dims 797 against 726).
          const bool masked = wlim < PA_BN;
          float v[4][32];
#pragma unroll 1
          for (bool moved = false;; moved = true) {   // once, but for scores that fp32 holds too coarsely
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32_nw(s_addr + c * 32, v[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_wait_ld32(v[c]);
            if (masked) {
#pragma unroll
              for (int c = 0; c < 4; ++c) mask32(v[c], lim - c * 32);
            }
            if (PR::NARROW && moved) break;
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
#pragma unroll
              for (int j = 0; j < 32; j += 2) mx[j >> 1 & 3] = max3(mx[j >> 1 & 3], v[c][j], v[c][j + 1]);
            }
            const float raw = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]), mt = raw * p.sl2;
            // also for NaN, and for the first key a row sees
            const bool grow = PR::NARROW ? !(raw <= raw_most) : !(mt <= m_run + PR::MOST);
            if (i == 0 || __any_sync(0xffffffffu, grow)) {
              const float m_new = PR::NARROW ? fmaf(raw, p.sl2, -PR::LIFT) : mt;
              if (i > 0) {
                // O was last written by this slot's previous P V, complete before this S
                const float f = grow ? pf_ex2(m_run - m_new) : 1.f;
                l_run *= f;
#pragma unroll 1
                for (int c = 0; c < D; c += 8) tmem_fma8(o_addr + c, f, 0.f);   // rare: few registers
                tmem_wait_st();
              }
              if (grow) {
                m_run = m_new + (mt - mt);            // an infinite maximum gives NaN, as inf - inf does
                if constexpr (PR::NARROW) {
                  m_raw = raw;
                  raw_most = __fadd_rd(raw, p.raw_step);
                }
              }
              nm = m_run == -INFINITY ? 0.f : -m_run;
              if constexpr (PR::NARROW) {
                const bool far = m_run != -INFINITY && fabsf(m_run) >= PR::FAR;
                if (far) nm = PR::LIFT;
                else m_raw = 0.f;
                any_far = __any_sync(0xffffffffu, far);
              }
            }
            if (!PR::NARROW || !any_far) break;
#pragma unroll 1
            for (int c = 0; c < PA_BN; c += 8) tmem_fma8(s_addr + c, 1.f, -m_raw);   // P is not written yet
            tmem_wait_st();
          }
          const float2 s2 = make_float2(p.sl2, p.sl2), n2 = make_float2(nm, nm);
          float2 acc[2];
          acc[0] = acc[1] = make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 a = __ffma2_rn(make_float2(v[c][2 * j], v[c][2 * j + 1]), s2, n2);
              const float2 e = make_float2(pf_ex2(a.x), pf_ex2(a.y));
              acc[j & 1] = __fadd2_rn(acc[j & 1], e);
              pk[j] = pack2<T>(e.x, e.y);
            }
            tmem_st16_nw(p_addr + c * 16, pk);   // columns of their own, or of S that were read before
          }
          acc[0] = __fadd2_rn(acc[0], acc[1]);
          l_run += acc[0].x + acc[0].y;
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && !(warp == 0 && pa_held(PA_HOLD_P))) pa_arrive(&p_full[sl]);
      }
      // ---- epilogue: O of this slot (slot 0 joins both parts of a one-tile item) ------
      if (sl == 0 && other) o1_ph ^= 1;   // slot 1 completes a phase too
      if (mine == 0) {
        item_done();
        continue;
      }
      ok = __all_sync(0xffffffffu, pa_wait(&o_full[sl], o_ph, abort_flag) && !*abort_flag);
      if (!ok) break;
      o_ph ^= 1;
      tc_fence_after();
      if (join && sl == 1) {
        s_ml[row] = make_float2(m_run, l_run);
        __syncwarp();
        if (lane == 0) pa_arrive(ml_full);
        item_done();
        continue;   // slot 0 reads O_1 and frees it
      }
      float f0 = 1.f, f1 = 0.f;
      if (join) {
        ok = pa_wait_warp(&o_full[1], o1_ph ^ 1, abort_flag) && pa_wait_warp(ml_full, ml_ph, abort_flag);
        if (!ok) break;
        ml_ph ^= 1;
        tc_fence_after();
        const float2 b = s_ml[row];
        const float mm = fmaxf(m_run, b.x);
        f0 = m_run == -INFINITY ? 0.f : pf_ex2(m_run - mm);
        f1 = b.x == -INFINITY ? 0.f : pf_ex2(b.x - mm);
        m_run = mm;
        l_run = l_run * f0 + b.y * f1;
      }
      const bool nothing = l_run == 0.f;
      const float inv = nothing ? 0.f : 1.f / l_run;
      const int tok = (two ? sl * TT : 0) + row_tok;                  // this row's token in the item
      const bool row_ok = row_tok < TT && tok < w.n_tok;
      const int out_mode = w.out_mode, src = w.src, out_at = w.out_at;
      const int64_t t = w.tok0 + tok;
      const int hq = w.hk * G + row_g;
      const int prow = (two ? sl * 128 : 0) + row;      // row in a piece
      if (out_mode != PA_DIRECT && row_ok) {
        if (out_mode == PA_PIECE) p.ml[(int64_t)out_at * 256 + prow] = make_float2(m_run, l_run);
        else p.row_ml[((int64_t)src * p.T + t) * p.Hq + hq] = make_float2(m_run, l_run);
      }
      if (warp_ok) {
        // whole rows of whole tokens leave through shared memory (128-byte swizzled) and TMA; a warp with rows of
        // no token (a sequence's end, groups that do not divide 32) stores its own rows, 32 bytes at a time
        const bool bulk = out_mode == PA_DIRECT && p.tma_out > 0 && __all_sync(0xffffffffu, row_ok);
        unsigned char* stage = sOut + warp * 4096 + lane * 128;
#pragma unroll 1   // short code: an item's end is often its first use
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          tmem_ld32(o_addr + c * 32, o);
          if (join) {
            float o1[32];
            tmem_ld32(o_addr + 128 + c * 32, o1);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = o[j] * f0 + o1[j] * f1;
          }
          if (nothing) {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = 0.f;
          }
          if (out_mode == PA_DIRECT) {
            uint32_t u[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) u[j] = pack2<T>(o[2 * j] * inv, o[2 * j + 1] * inv);
            if (bulk) {
              if ((c & 1) == 0) {   // the last copy has read the stage
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint4*>(stage + ((((c & 1) * 4 + j) ^ (lane & 7)) << 4)) =
                    make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
              if (c & 1) {
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                  asm volatile(
                      "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(&maps.out),
                      "r"((c >> 1) * 64), "r"(0), "r"(w.hk), "r"((int)t), "r"(smem_u32(stage))
                      : "memory");
                  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
              }
            } else if (row_ok) {
              T* og = reinterpret_cast<T*>(p.out) + t * p.ost + hq * p.osh + c * 32;
              if (wide) {
#pragma unroll
                for (int j = 0; j < 16; j += 8)
                  if (c * 32 + 2 * j < p.D) st_global_32(og + 2 * j, &u[j]);
              } else {
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                  if (c * 32 + 2 * j < p.D)
                    *reinterpret_cast<uint4*>(og + 2 * j) = make_uint4(u[j], u[j + 1], u[j + 2], u[j + 3]);
              }
            }
          } else if (row_ok) {
            const bool piece = out_mode == PA_PIECE;
            float4* base = piece ? p.o + ((int64_t)out_at * (D / 4)) * 256 + prow
                                 : p.row_o + (((int64_t)src * p.T + t) * p.Hq + hq) * (D / 4);
            const int step = piece ? 256 : 1;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              base[(c * 8 + j / 4) * step] = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        pa_arrive(&o_empty[sl]);
        if (join) pa_arrive(&o_empty[1]);
        if (out_mode == PA_PIECE && p.prefix == 0) {   // these rows of the piece are written
          __threadfence();
          if (!pa_held(PA_HOLD_MARK)) store_release(&p.ready[(int64_t)out_at * 8 + (prow >> 5)], s_join->token);
        }
      }
      item_done();
    }
    // ---- the item whose last piece this CTA holds: join its pieces, in CTA order --------
    if (ok && s_join->n > 0) {
      const int n = s_join->n, first = s_join->first, words = s_join->n_tok > TT ? 8 : 4;
      // the other pieces belong to CTAs before this one, and were the last of their whole items
      bool got = true;
#pragma unroll 1
      for (int e = lane; got && e < n * words; e += 32)
        got = pa_wait_ready(&p.ready[pa_slot(first, e / words) * 8 + e % words], s_join->token, abort_flag);
      __syncwarp();
      __threadfence();
      if (__all_sync(0xffffffffu, got)) {
        // a thread owns a row (of the next power of two) and every so many 16-dim units of it
        const int rows = s_join->n_tok * G, shift = 32 - __clz(rows - 1 | 1);
        const int r = tid & ((1 << shift) - 1), tok = r / G, g = r - tok * G, tile = tok >= TT ? 1 : 0;
        const int prow = tile * PA_ROWS + (tok - tile * TT) * G + g;
        float m = -INFINITY, l = 0.f;
        if (r < rows) {
#pragma unroll 4
          for (int i = 0; i < n; ++i) {
            const float2 ml = p.ml[pa_slot(first, i) * 256 + prow];
            const float mn = fmaxf(m, ml.x);
            l = l * (m == -INFINITY ? 0.f : pf_ex2(m - mn)) + ml.y * (ml.x == -INFINITY ? 0.f : pf_ex2(ml.x - mn));
            m = mn;
          }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* og = reinterpret_cast<T*>(p.out) + (int64_t)(s_join->tok0 + tok) * p.ost + (int64_t)(s_join->hk * G + g) * p.osh;
#pragma unroll 1
        for (int u = tid >> shift; r < rows && u * 16 < p.D; u += 256 >> shift) {
          float4 a[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) a[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
          for (int i = 0; i < n; ++i) {
            const int at = pa_slot(first, i);
            const float4* src = p.o + ((int64_t)at * (D / 4) + u * 4) * 256 + prow;
            const float x = p.ml[at * 256 + prow].x;
            float4 o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = __ldcg(src + j * 256);
            const float f = x == -INFINITY ? 0.f : pf_ex2(x - m);
            if (f != 0.f) {   // a piece that saw nothing holds no values
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                a[j].x += o[j].x * f; a[j].y += o[j].y * f; a[j].z += o[j].z * f; a[j].w += o[j].w * f;
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 4; j += 2)
            if (u * 16 + j * 4 < p.D)
              *reinterpret_cast<uint4*>(og + u * 16 + j * 4) =
                  make_uint4(pack2<T>(a[j].x * inv, a[j].y * inv), pack2<T>(a[j].z * inv, a[j].w * inv),
                             pack2<T>(a[j + 1].x * inv, a[j + 1].y * inv), pack2<T>(a[j + 1].z * inv, a[j + 1].w * inv));
        }
        __syncwarp();
        // the last warp takes the marks back: a replayed call starts without them
        if (__shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(&s_join->left, 1) : 0, 0) == 7)
          for (int e = lane; e < n * words; e += 32) p.ready[pa_slot(first, e / words) * 8 + e % words] = 0;
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // the last rows are written
    if (p.zero_tail) {   // rows ahead of the first sequence and behind the last, of an output this call allocated
      // no 64-bit division: it is a call, for which registers of the whole kernel were spilled (prompts 1 to 2 % slower)
      const int first = pa_first(p), owned = pa_used(p) - first;
#pragma unroll 1
      for (int i = (int)blockIdx.x; i < p.T - owned; i += (int)gridDim.x) {
        const int64_t t = i < first ? i : i + owned;
#pragma unroll 1
        for (int e = tid; e < p.Hq * (p.D / 8); e += 256) {
          const int h = e / (p.D / 8);
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + t * p.ost + h * p.osh + (e - h * (p.D / 8)) * 8) = make_uint4(0, 0, 0, 0);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_REGS_ISSUE));
    auto all = [&](bool x) { return (bool)__all_sync(0xffffffffu, x); };
    // Positions c at the next task on slot sl; false when there is none: at the end of the stream (c.done), or when
    // the next item begins on slot 0 and this is slot 1.  `release`: this cursor is its warp's last reader.
    auto next_task = [&](PaCursor& c, int sl, bool& ok, bool release, bool loads) __attribute__((always_inline)) {
      if (c.done) return false;
      if (c.j == c.tasks) {
        const int qi = c.it % PA_QUEUE;
        ok = pa_wait_warp(&it_full[qi], (unsigned)((c.it / PA_QUEUE) & 1), abort_flag);
        if (!ok) return false;
        ++c.it;
        const PaItem& w = queue[qi];
        c.done = uniform(w.out_mode) == PA_STOP;
        c.n = uniform(w.j1 - w.j0);
        c.two = uniform(w.n_tok > TT);
        if (loads) {
          c.src = uniform(w.src);
          c.hk = uniform(w.hk);
          c.tok0 = uniform(w.tok0);
          c.slot = uniform(w.slot);
          c.row0 = uniform(w.row0 + w.j0 * PA_BN);
        } else {
          c.left = uniform(w.kv_len - w.j0 * PA_BN);
        }
        c.tasks = c.two ? 2 * c.n : c.n;
        c.j = 0;
        __syncwarp();
        if (release && lane == 0) pa_arrive(&it_empty[qi]);
        if (c.done) return false;
      }
      return !(c.two && c.j == 0 && sl == 1);
    };
    if (warp == 8) {
      // ---- loads of K and V, in the order of use -------------------------------------
      const int used = p.prefix > 0 ? 6 : 4;
      if (lane < used) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps) + lane * sizeof(CUtensorMap)) : "memory");
      unsigned stage = 0, stage_ph = 1, loads = 0;
      PaCursor ck, cv;
      bool ok = true;
      // the K (or V) tile that S (or P V) of the next task on slot sl reads first
      auto step = [&](PaCursor& c, int sl, bool is_v) __attribute__((always_inline)) {
        if (!next_task(c, sl, ok, is_v, true)) return;
        const int j = c.j++;
        if (c.two && (j & 1)) return;
        ok = pa_wait_warp(&kv_empty[stage], stage_ph, abort_flag);
        if (!ok) return;
        const CUtensorMap* m = c.src ? (is_v ? &maps.pv : &maps.pk) : (is_v ? &maps.v : &maps.k);
        const int at_t = c.src ? (is_v ? p.pv_t : p.pk_t) : (is_v ? p.v_t : p.k_t);
        const int at_h = c.src ? (is_v ? p.pv_h : p.pk_h) : (is_v ? p.v_h : p.k_h);
        const int row = c.row0 + (c.two ? j >> 1 : j) * PA_BN;
        const int c1 = at_t == 1 ? row : at_h == 1 ? c.hk : c.slot, c2 = at_t == 2 ? row : at_h == 2 ? c.hk : c.slot,
                  c3 = at_t == 3 ? row : at_h == 3 ? c.hk : c.slot;
        if (elect_one()) {
          pf_expect_tx(&kv_full[stage], PG::KV_BYTES);
#pragma unroll
          for (int a = 0; a < PG::NB; ++a)
            pf_tma4(sKV + stage * PG::KV_BYTES + a * PA_BN * 128, m, a * 64, c1, c2, c3, &kv_full[stage]);
        }
        __syncwarp();
        ++loads;
        if (++stage == ST) stage = 0, stage_ph ^= 1;
      };
      // K runs two tasks ahead
#pragma unroll 1
      for (int i = -2; ok && !cv.done; ++i) {
        if (i >= 0) step(cv, i & 1, true);
        if (ok) step(ck, i & 1, false);
      }
      // the copies in flight land before the CTA ends, whoever gave up on them
#pragma unroll 1
      for (unsigned k = loads > ST ? loads - ST : 0; k < loads; ++k) (void)mbar_wait(&kv_full[k % ST], (k / ST) & 1);
    } else if (warp == 9) {
      // ---- MMA issue --------------------------------------------------------------
      const int kd = (p.D + 15) / 16;
      const uint32_t idesc_s = umma_idesc_f16(PA_BN, BF, 0), idesc_o = umma_idesc_f16(kd * 16, BF, 1);
      const uint32_t q_lo = pa_desc_lo(smem_u32(sQ), 16), k_lo = pa_desc_lo(smem_u32(sKV), 16),
                     v_lo = pa_desc_lo(smem_u32(sKV), PA_BN * 128);
      unsigned stage = 0, stage_ph = 0, q_ph = 0, p_ph = 0, oe_ph = 3;   // a phase bit per buffer or slot
      unsigned k_stage = 0, v_stage = 0;
      int ks = 0, qb = 0;
      PaCursor cs, cp;
      bool ok = true;
      // the next tile of the ring, once its bytes have landed
      auto next_tile = [&]() __attribute__((always_inline)) {
        const unsigned st = stage;
        ok = pa_wait_warp(&kv_full[st], stage_ph, abort_flag);
        if (++stage == ST) stage = 0, stage_ph ^= 1;
        return st;
      };
      // S of the next task on slot sl
      auto issue_s = [&](int sl) __attribute__((always_inline)) {
        if (!next_task(cs, sl, ok, false, false)) return;
        const int j = cs.j++;
        if (!cs.two && j == 0) qb ^= 1;
        const int buf = cs.two ? sl : qb ^ 1;
        if (!cs.two || sl == 0) k_stage = next_tile();
        if (cs.two ? j < 2 : j == 0) {
          ok = all(ok && pa_wait(&q_full[buf], q_ph >> buf & 1, abort_flag));
          q_ph ^= 1u << buf;
        }
        if (!ok) return;
        tc_fence_after();
        const uint32_t a = q_lo + buf * (PG::Q_BYTES >> 4), b = k_lo + k_stage * (PG::KV_BYTES >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kc = 0; kc < D / 16; ++kc) {   // 16 dims = 32 bytes inside a 64-dim column block
            const uint32_t off = (uint32_t)(((kc >> 2) * PA_ROWS * 128 + (kc & 3) * 32) >> 4);
            if (kc < kd) pa_mma_ss(sl * 128, a + off, b + off, idesc_s, kc > 0);
          }
          umma_commit(&s_full[sl]);
          if (!cs.two || sl == 1) umma_commit(&kv_empty[k_stage]);
          if (j >= cs.tasks - 1 - cs.two) umma_commit(&q_empty[buf]);
        }
        __syncwarp();
      };
      // P V of the next task on slot sl
      auto issue_pv = [&](int sl) __attribute__((always_inline)) {
        if (!next_task(cp, sl, ok, true, false)) return;
        const int j = cp.j++;
        const bool first = j < 2, last = j >= cp.tasks - 2;   // of the item on this slot
        if (!cp.two || sl == 0) {
          v_stage = next_tile();
          // 16-token steps of the tile; rows behind the sequence inside the last one are zeroed
          const int valid = min(PA_BN, cp.left - (cp.two ? j >> 1 : j) * PA_BN);
          ks = (valid + 15) >> 4;
          if (ok && (valid & 15)) {
            unsigned char* tile = sKV + v_stage * PG::KV_BYTES;
            const int rows = ks * 16 - valid;
#pragma unroll 1
            for (int e = lane; e < rows * PG::NB * 8; e += 32) {
              const int r = valid + e / (PG::NB * 8), c = e % (PG::NB * 8);
              *reinterpret_cast<uint4*>(tile + (c >> 3) * PA_BN * 128 + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();
            __syncwarp();
          }
        }
        bool got = ok && pa_wait(&p_full[sl], p_ph >> sl & 1, abort_flag);
        p_ph ^= 1u << sl;
        if (first) {   // the epilogue of the slot's last item has read O (passes at once the first time)
          got = got && pa_wait(&o_empty[sl], oe_ph >> sl & 1, abort_flag);
          oe_ph ^= 1u << sl;
        }
        ok = all(got);
        if (!ok) return;
        tc_fence_after();
        const uint32_t b = v_lo + v_stage * (PG::KV_BYTES >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kc = 0; kc < PA_BN / 16; ++kc)
            if (kc < ks) pa_mma_ts(256 + sl * 128, PG::P0 + sl * 128 + kc * 8, b + kc * (2048 >> 4), idesc_o, !first || kc > 0);
          if (last) umma_commit(&o_full[sl]);
          if (!cp.two || sl == 1) umma_commit(&kv_empty[v_stage]);
        }
        __syncwarp();
      };
      // Tasks well inside one item, from slot 0 on: P V and the S behind it are issued together, with nothing to look
      // up in between.  The tensor pipe takes a few instructions ahead, so it idles for all that this warp does
      // between two of them.
      auto steady = [&]() __attribute__((always_inline)) {
        const int m = cs.it == cp.it && cp.j >= 2 ? (cs.tasks - cs.j - 2) & ~1 : 0;
        if (m <= 0) return;
        const uint32_t q_at = q_lo + (cs.two ? 0 : (qb ^ 1) * (PG::Q_BYTES >> 4)), q_step = cs.two ? PG::Q_BYTES >> 4 : 0;
#pragma unroll 1
        for (int i = 0; i < m; ++i) {
          const int sl = i & 1;
          bool got = true;
          if (!cs.two || sl == 0) {
            v_stage = stage;
            got = pa_wait(&kv_full[stage], stage_ph, abort_flag);
            if (++stage == ST) stage = 0, stage_ph ^= 1;
            k_stage = stage;
            got = pa_wait(&kv_full[stage], stage_ph, abort_flag) && got;
            if (++stage == ST) stage = 0, stage_ph ^= 1;
          }
          got = pa_wait(&p_full[sl], p_ph >> sl & 1, abort_flag) && got;
          p_ph ^= 1u << sl;
          ok = all(got);
          if (!ok) return;
          tc_fence_after();
          const uint32_t bv = v_lo + v_stage * (PG::KV_BYTES >> 4), bk = k_lo + k_stage * (PG::KV_BYTES >> 4);
          const uint32_t a = q_at + sl * q_step, d = sl * 128;
          if (elect_one()) {
#pragma unroll
            for (int kc = 0; kc < PA_BN / 16; ++kc) pa_mma_ts(256 + d, PG::P0 + d + kc * 8, bv + kc * (2048 >> 4), idesc_o, 1);
#pragma unroll
            for (int kc = 0; kc < D / 16; ++kc) {
              const uint32_t off = (uint32_t)(((kc >> 2) * PA_ROWS * 128 + (kc & 3) * 32) >> 4);
              if (kc < kd) pa_mma_ss(d, a + off, bk + off, idesc_s, kc > 0);
            }
            umma_commit(&s_full[sl]);
            if (!cs.two || sl == 1) {
              umma_commit(&kv_empty[v_stage]);
              umma_commit(&kv_empty[k_stage]);
            }
          }
          __syncwarp();
        }
        cs.j += m;
        cp.j += m;
      };
      // S runs two tasks ahead.  One copy of this code for all cases: it competes for the instruction cache.
#pragma unroll 1
      for (int i = -2; ok && !cp.done; ++i) {
        const int sl = i & 1;
        if (sl == 0) steady();
        if (i >= 0 && ok) issue_pv(sl);
        if (ok) issue_s(sl);
      }
    } else if (warp == 11) {
      // ---- loads of the query tiles: both buffers for a two-tile item, else one, in turn --------
      unsigned q_ph = 3, q_uses = 0;   // a phase bit per buffer
      int qb = 0;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const int qi = it % PA_QUEUE;
        ok = pa_wait_warp(&it_full[qi], (unsigned)((it / PA_QUEUE) & 1), abort_flag);
        if (!ok) break;
        const int mode = uniform(queue[qi].out_mode), two = uniform(queue[qi].n_tok > TT), hk = uniform(queue[qi].hk),
                  tok0 = uniform(queue[qi].tok0);
        __syncwarp();
        if (lane == 0) pa_arrive(&it_empty[qi]);
        if (mode == PA_STOP) break;
#pragma unroll 1
        for (int t = 0; t < (two ? 2 : 1); ++t) {
          const int buf = two ? t : qb;
          ok = pa_wait_warp(&q_empty[buf], q_ph >> buf & 1, abort_flag);   // passes at once the first time
          if (!ok) break;
          q_ph ^= 1u << buf;
          q_uses |= 1u << buf;
          if (elect_one()) {
            pf_expect_tx(&q_full[buf], (uint32_t)(PG::NB * TT * G * 128));
#pragma unroll
            for (int a = 0; a < PG::NB; ++a)
              pf_tma4(sQ + buf * PG::Q_BYTES + a * PA_ROWS * 128, &maps.q, a * 64, 0, hk, tok0 + t * TT, &q_full[buf]);
          }
          __syncwarp();
        }
        if (!two) qb ^= 1;
      }
      for (int i = 0; i < 2; ++i)   // as for K and V
        if (q_uses >> i & 1) (void)mbar_wait(&q_full[i], q_ph >> i & 1);
    } else if (warp == 10) {
      // ---- schedule: this CTA's share of the unit line ------------------------------
      unsigned long long failures = 0;   // on its way during the scan
      if (lane == 0) failures = *reinterpret_cast<volatile unsigned long long*>(&g_pa_failures);
      bool bad = false;
      const int64_t mine = pa_lane_units(p, lane, bad);
      if (bad) dev_flag(HOKV_ERR_DEVICE_INPUT);
      if (lane == 0) s_join->token = p.token ^ (failures * 0xd1342543de82ef95ull);
      int64_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const int64_t total = __shfl_sync(0xffffffffu, incl, 31);
      const int64_t share = pa_share(p, total);
      const int64_t begin = min((int64_t)blockIdx.x * share, total), end = min(begin + share, total);
      int n_items = 0;
      auto push = [&](const PaItem& w) {
        const int qi = n_items % PA_QUEUE, use = n_items / PA_QUEUE;
        if (use > 0 && !pa_wait_warp(&it_empty[qi], (unsigned)((use - 1) & 1), abort_flag)) return false;
        if (lane == 0) {
          queue[qi] = w;
          pa_arrive(&it_full[qi]);
        }
        __syncwarp();
        ++n_items;
        return true;
      };
      bool ok = true;
      PaItem tail = {};
      if (begin < end) {
        const PaStart at = pa_find_start(p, begin, [&](int) { return mine; }, [&](int) { return incl; });
        ok = pa_walk(p, (int)blockIdx.x, begin, end, at.s, at.at, at.pr, [&](const PaItem& w, bool begins, bool ends,
                                                                    int64_t item_at, int sh, int tiles) {
          if (w.out_mode == PA_PIECE && p.prefix == 0 && !begins) {
            // an item that earlier CTAs began comes last: its other pieces are done by then, and whoever holds its
            // last piece joins them (waiting for lower CTAs only)
            tail = w;
            if (ends && lane == 0) {
              s_join->first = pa_first_cta(share, item_at);
              s_join->tok0 = w.tok0;
              s_join->n_tok = w.n_tok;
              s_join->hk = w.hk;
              s_join->n = (int)blockIdx.x - s_join->first + 1;
            }
            return true;
          }
          if (p.prefix > 0 && begins) {   // where k_packed_combine_rows finds this item's rows
            const int info = ends ? -1 : (int)blockIdx.x | pa_last_cta(share, item_at, sh, tiles) << 8;
#pragma unroll 1
            for (int i = lane; i < w.n_tok; i += 32)
              p.tok_info[((int64_t)w.src * p.T + w.tok0 + i) * p.Hkv + w.hk] = make_int2(info, i);
          }
          if (w.j0 == w.j1) {   // nothing to see: zeros, or an empty part of a row
#pragma unroll 1
            for (int e = lane; e < w.n_tok * G * (p.D / 8); e += 32) {
              const int r = e / (p.D / 8), tok = r / G;
              const int64_t t = w.tok0 + tok;
              const int h = w.hk * G + r - tok * G;
              if (w.out_mode == PA_ROWWISE) p.row_ml[((int64_t)w.src * p.T + t) * p.Hq + h] = make_float2(-INFINITY, 0.f);
              else *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + t * p.ost + h * p.osh + e % (p.D / 8) * 8) = make_uint4(0, 0, 0, 0);
            }
            return true;
          }
          return push(w);
        });
      }
      if (ok && tail.out_mode == PA_PIECE) ok = push(tail);
      if (ok && !pa_held(PA_HOLD_STOP)) {
        tail.out_mode = PA_STOP;
        push(tail);
      }
    }
  }
  // every role is done: each item's last products were awaited by its
  // epilogue, or the CTA gave up, and the products in flight are awaited here
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    if (*abort_flag) {
      if (lane == 0) atomicAdd(&g_pa_failures, 1ull);
      if (elect_one()) umma_commit(mma_done);
      __syncwarp();
      (void)mbar_wait(mma_done, 0);
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

// ---- joining the parts of a row ----------------------------------------------------
// With a shared prefix every row joins its prefix part and its own part, each
// one row-wise result or the pieces of a cut item.  Grid (tokens, KV heads,
// heads of a group in steps of PA_JOIN).  Bound by latency, not bytes: a long
// prefix cut over every SM leaves dozens of pieces of a few rows.  The warps
// take pieces in turn, each with running statistics of its own, and meet once
// in shared memory; both orders are fixed: the same result each run.
constexpr int PA_JOIN = 8;

template <int D, typename T>
__global__ void __launch_bounds__(256) k_packed_combine_rows(const PaP p) {
  constexpr int K = D / 16;   // 4-dim groups of a lane
  __shared__ float2 s_ml[8][PA_JOIN];
  __shared__ __align__(16) float4 s_o[8][K][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int t = blockIdx.x, hk = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane % PA_JOIN, g = blockIdx.z * PA_JOIN + r, hq = hk * p.G + min(g, p.G - 1);
  if (t < pa_first(p) || t >= pa_used(p)) return;
  int first[2], n[2], prow[2];   // own keys, prefix
#pragma unroll
  for (int src = 0; src < 2; ++src) {
    const int2 info = p.tok_info[((int64_t)src * p.T + t) * p.Hkv + hk];
    // a token that no valid sequence covers has no entry: any value stays inside the workspace
    const int tok = min(max(info.y, 0), 2 * p.TT - 1), tile = tok >= p.TT ? 1 : 0;
    prow[src] = tile * PA_ROWS + (tok - tile * p.TT) * p.G + hq - hk * p.G;
    first[src] = info.x < 0 ? -1 : min(info.x & 255, p.n_ctas - 1);
    n[src] = info.x < 0 ? 1 : max(min(info.x >> 8, p.n_ctas - 1) - first[src] + 1, 1);
  }
  float m = -INFINITY, l = 0.f;
  float4 a[K];
#pragma unroll
  for (int k = 0; k < K; ++k) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (int i = warp; i < n[0] + n[1]; i += 8) {
    const int src = i < n[0] ? 0 : 1, piece = src ? i - n[0] : i;
    const int64_t rw = ((int64_t)src * p.T + t) * p.Hq + hq;
    const int64_t at = pa_slot(first[src], piece);
    const bool rowwise = first[src] < 0;
    const float2 ml = rowwise ? p.row_ml[rw] : p.ml[at * 256 + prow[src]];
    const float4* base = rowwise ? p.row_o + rw * (D / 4) : p.o + at * (D / 4) * 256 + prow[src];
    const int step = rowwise ? 1 : 256;
    float4 o[K];
#pragma unroll
    for (int k = 0; k < K; ++k) o[k] = base[(int64_t)((lane >> 3) + 4 * k) * step];
    if (ml.x != -INFINITY) {   // a part that saw nothing holds no values
      const float mn = fmaxf(m, ml.x);
      const float fa = m == -INFINITY ? 0.f : pf_ex2(m - mn), fb = pf_ex2(ml.x - mn);
      l = l * fa + ml.y * fb;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        a[k].x = a[k].x * fa + o[k].x * fb; a[k].y = a[k].y * fa + o[k].y * fb;
        a[k].z = a[k].z * fa + o[k].z * fb; a[k].w = a[k].w * fa + o[k].w * fb;
      }
      m = mn;
    }
  }
  if (lane < PA_JOIN) s_ml[warp][r] = make_float2(m, l);
#pragma unroll
  for (int k = 0; k < K; ++k) s_o[warp][k][lane] = a[k];
  __syncthreads();
  const int d = ((lane >> 3) + 4 * warp) * 4;   // warp k takes the lanes' group k
  if (warp >= K || g >= p.G || d >= p.D) return;
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, s_ml[w][r].x);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float2 ml = s_ml[w][r];
    const float f = ml.x == -INFINITY ? 0.f : pf_ex2(ml.x - m);
    const float4 x = s_o[w][warp][lane];
    l += ml.y * f;
    o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* og = reinterpret_cast<T*>(p.out) + (int64_t)t * p.ost + (int64_t)hq * p.osh + d;
  *reinterpret_cast<uint2*>(og) = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
}

}  // namespace hokv
