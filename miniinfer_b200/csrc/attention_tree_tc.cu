// Attention of a tree of new tokens over the paged cache in bf16 on the fifth-generation tensor cores (tcgen05), head sizes 64 to 256.
// attention_tree.cuh says which keys a row sees.
//
// The rows of one (item, key/value head) - all heads of its group for up to 128 / G tokens, or twice that - are the M of the products, so a key is
// fetched once for all of them: a tree of 32 over groups of 4 fills the 128 rows, and reading keys and values is what the
// operator costs.  The tiles of 128 keys (64 for heads beyond 128) of all (item, head, rows) units lie on one line, item after item, and every SM gets an equal stretch of
// it: contexts of any mixture of lengths keep all SMs busy to the end.  A unit that lies in one stretch is written out; the
// pieces of one that several share are left as sums that are not normalised, two at most a block, and tree_join_kernel adds them up.
//
// Roles of a block: a producer warp (queries of a unit, keys and values tile by tile into a ring of boxes, by TMA in the 128-byte swizzle;
// a lane a box, the next tile's pages looked up ahead), a thread that issues all products, eight softmax warps.  Weights stay in tensor memory,
// over the scores they come from.  With 128 rows (QT = 1) two score buffers take turns, scores run two tiles ahead, and two threads share a row;
// with 256 (QT = 2, heads up to 128) two sets of rows take turns on one tile of keys, a thread a row, and keys and values are
// fetched once for both.
//
// Weights of invisible keys are zeros in P V, so whatever is not finite among the values of a tile that the mask touches is taken out in
// shared memory first; a row that does see such a value gets it added at the end.  Only those tiles pay for it.
//
// The weight of the running maximum is exactly 1; weights are rounded to bf16, and the sum that divides the row is that of the rounded ones.
#include <cuda.h>
#include <string.h>

#include "attention_tree.cuh"

namespace {

using namespace mi_tree;

constexpr int BM = 128, BOX = 64, BUFFERS = 2;
constexpr int SOFTMAX_WARPS = 8, PRODUCER_WARP = 8, MMA_WARP = 9, THREADS = 320;
constexpr int TMEM_COLS = 512, S_COL = 256;
constexpr int MAX_UNITS = 12;                 // boxes of the ring: a tile's keys or its values each
constexpr int WAIT_LIMIT = 1 << 22;
constexpr int SMEM_BYTES = 227 << 10, SMEM_TAIL = 4096;      // behind queries and ring: barriers, maxima, sums

struct Tc {
  Args a;
  int* status;
  int2* units;                   // [items * nkv * max_parts]: first block, pieces
  int boxes, steps, n_out;       // boxes and 16s of columns of a row, columns of P V
  int ring, box_rows;            // units of the ring; rows of a TMA box of keys
  int tokens, max_parts;         // tokens of a set of 128 rows; parts of the largest item
  float scale_log2;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Bounded wait.  `abort` is a flag in shared memory: once any wait has run out, all waits return.
__device__ __forceinline__ void mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  const uint32_t addr = smem_u32(bar);
  for (int i = 0; i < WAIT_LIMIT; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    if (done) return;
    if ((i & 63) == 63 && *abort) return;
  }
  *abort = 1;
  atomicExch(status, 2);
}
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The barrier gets an arrival when all products issued so far by this thread are done.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D[tmem] (+)= A[smem] * B[smem], and with A in tensor memory (lane = row, two bf16 of consecutive k to a column).
__device__ __forceinline__ void tc_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 consecutive columns of this thread's lane, written.
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// N consecutive columns of this thread's lane (lane = 32 * (warp % 4) + lane of the warp), read.
__device__ __forceinline__ void tmem_ld(float (&v)[32], uint32_t taddr) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld(float (&v)[64], uint32_t taddr) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
// Shared-memory operand descriptor, 128-byte swizzle: start address, leading and stride byte offsets in 16-byte units,
// descriptor version 1 (bits 46..47), layout type 2 = 128-byte swizzle (bits 61..63).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lbo_bytes >> 4) & 0x3FFF) << 16) |
         ((uint64_t)((sbo_bytes >> 4) & 0x3FFF) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor of kind::f16: float32 accumulator (bits 4..5 = 1), bf16 A and B (bits 7..9 and 10..12 = 1), B K-major or
// MN-major (bit 16), N / 8 at bits 17..22, M / 16 at bits 24..28.
__host__ __device__ constexpr uint32_t instr_desc(int M, int N, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The line of tiles: item after item, in an item head after head, in a head part after part (QT * tokens tokens each).
struct Line {
  int t_begin, tiles, parts;     // of an item: first tile that some row sees, tiles, parts
};
template <int QT, int BN>
__device__ __forceinline__ Line line_of(const Tc& k, const Item& it) {
  Line l;
  l.t_begin = (k.a.window > 0 ? max(0, it.start - k.a.window + 1) : 0) / BN;
  l.tiles = it.n > 0 ? (it.ctx + BN - 1) / BN - l.t_begin : 0;
  l.parts = (it.n + QT * k.tokens - 1) / (QT * k.tokens);
  return l;
}
__device__ __forceinline__ long long stretch_begin(long long total, int b, int blocks) { return total * b / blocks; }

// Where a block's stretch begins, and how long it is.
struct Start {
  int item, left;
  long long offset, total;       // tiles of the item before the stretch; of the whole line
  int blocks;                    // that have a stretch
};

// A stretch's next piece of a unit.
struct Piece {
  Item it;
  Line l;
  int b, head, part, j0, n;      // item, key/value head, part; first tile of the unit's, tiles
  bool whole;
  int slot;                      // of the sums, where the unit goes on in other blocks
};
template <int QT, int BN>
struct Walk {
  const Tc& k;
  int item, left;
  long long offset;
  Item it;
  Line l;
  bool first = true;
  __device__ Walk(const Tc& k_, const Start& s) : k(k_), item(s.item), left(s.left), offset(s.offset) {
    if (left > 0) load();
  }
  __device__ void load() {
    it = item_of(k.a, item);
    l = line_of<QT, BN>(k, it);
  }
  __device__ bool next(Piece& p) {
    if (left <= 0) return false;
    long long all = (long long)l.tiles * k.a.nkv * l.parts;
    while (offset >= all) {      // (also items without tokens)
      offset -= all;
      if (++item >= k.a.items) return false;
      load();
      all = (long long)l.tiles * k.a.nkv * l.parts;
    }
    const int unit = (int)(offset / l.tiles);
    p.it = it;
    p.l = l;
    p.b = item;
    p.head = unit / l.parts;
    p.part = unit - p.head * l.parts;
    p.j0 = (int)(offset - (long long)unit * l.tiles);
    p.n = min(left, l.tiles - p.j0);
    p.whole = p.n == l.tiles;
    p.slot = 2 * (int)blockIdx.x + (p.j0 == 0 ? 1 : 0);
    offset += p.n;
    left -= p.n;
    return true;
  }
};

// Bits of the keys key0 .. key0 + 31 that a row sees: of the context from `begin` on, of the new ones by the token's mask (and the window).
__device__ __forceinline__ uint32_t seen_bits(const Args& a, const Item& it, int key0, int begin, const int* mask) {
  auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
  uint32_t bits = below(it.start - key0) & ~below(begin - key0);
  const int j0 = key0 - it.start;
  if (j0 > -32 && j0 < it.n) {
    uint32_t nodes;
    if (j0 < 0) {
      nodes = (uint32_t)mask[0] << -j0;
    } else {
      const uint32_t lo = (uint32_t)mask[j0 >> 5], hi = (j0 >> 5) + 1 < a.words ? (uint32_t)mask[(j0 >> 5) + 1] : 0u;
      nodes = __funnelshift_r(lo, hi, j0 & 31);
    }
    nodes &= below(it.n - j0);
    if (a.window > 0) {
      for (uint32_t todo = nodes; todo; todo &= todo - 1) {
        const int e = __ffs(todo) - 1;
        if (a.positions[it.row0 + j0 + e] < begin) nodes &= ~(1u << e);
      }
    }
    bits |= nodes;
  }
  return bits;
}

// What the P V products have left out of a row's sums: values that are not finite, of keys that the row sees (a rare call).
__device__ __noinline__ void add_not_finite(const Args& a, const Item& it, int head, int key_begin, int key_end, int begin, const int* mask, int col, float (&o)[32]) {
  const __nv_bfloat16* kv = reinterpret_cast<const __nv_bfloat16*>(a.kv);
  for (int key0 = key_begin; key0 < key_end; key0 += 32) {
    for (uint32_t bits = seen_bits(a, it, key0, begin, mask); bits; bits &= bits - 1) {
      const int key = key0 + __ffs(bits) - 1;
      if (key >= key_end) break;
      const __nv_bfloat16* v = kv + ((((size_t)page_of(a, it, key) * 2 + 1) * a.nkv + head) * a.page_size + key % a.page_size) * a.hd;
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (col + e < a.hd) {
          const float x = __bfloat162float(v[col + e]);
          if (!(fabsf(x) < INFINITY)) o[e] += x;
        }
    }
  }
}

template <int QT, int BN>
__global__ void __launch_bounds__(THREADS, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map, const Tc k) {
  constexpr int HALVES = 2 / QT, W = BN / HALVES;      // threads that share a row, their columns
  constexpr int COL_BYTES = BN * 128, Q_COL_BYTES = BM * 128;
  constexpr int P_COUNT = SOFTMAX_WARPS / QT;
  constexpr int LAG = QT == 1 ? 2 : 1;                  // tiles between two uses of a score buffer
  constexpr int P_AT = QT == 1 ? 0 : 64;                // where in it the weights begin
  const Args& a = k.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int q_bytes = k.boxes * Q_COL_BYTES, unit_bytes = k.boxes * COL_BYTES;      // of a set of rows; of a tile's keys or values
  unsigned char *q_s = smem, *ring_s = smem + QT * q_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring_s + k.ring * unit_bytes);
  uint64_t *q_full = bars, *q_empty = bars + 1, *o_free = bars + 2;
  uint64_t *u_full = bars + 3, *u_empty = u_full + MAX_UNITS;
  uint64_t *s_full = u_empty + MAX_UNITS, *p_full = s_full + BUFFERS, *o_full = p_full + BUFFERS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + BUFFERS);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* spoiled = abort + 1;      // [2]: the last piece, by parity, in which a value was not finite
  Start* start = reinterpret_cast<Start*>(bars + 40);
  float* row_max = reinterpret_cast<float*>(bars + 48);      // QT = 1: [2 tiles][2 halves][BM]; then the halves' sums [2][BM]
  float* row_sum = row_max + 4 * BM;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_free, SOFTMAX_WARPS);
    for (int u = 0; u < k.ring; ++u) {
      mbar_init(&u_full[u], 1);
      mbar_init(&u_empty[u], 1);
    }
    for (int b = 0; b < BUFFERS; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], P_COUNT);
      mbar_init(&o_full[b], 1);
    }
    *abort = 0;
    spoiled[0] = spoiled[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  mi::grid_dependency_sync();
  if (warp == PRODUCER_WARP) {      // where this block's stretch of the line begins
    auto tiles_of = [&](int b) {
      if (b >= a.items) return 0ll;
      const Line l = line_of<QT, BN>(k, item_of(a, b));
      return (long long)l.tiles * a.nkv * l.parts;
    };
    auto scan = [&](long long x) {      // sums up to and with this lane
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      return x;
    };
    const long long mine0 = tiles_of(lane);      // the first 32 items stay in registers
    long long total = __shfl_sync(0xffffffffu, scan(mine0), 31);
    for (int b0 = 32; b0 < a.items; b0 += 32) total += __shfl_sync(0xffffffffu, scan(tiles_of(b0 + lane)), 31);
    const int blocks = (int)min(total, (long long)gridDim.x), me = (int)blockIdx.x;
    const long long begin = me < blocks ? stretch_begin(total, me, blocks) : total, end = me < blocks ? stretch_begin(total, me + 1, blocks) : total;
    long long before = 0;
    Start s{0, (int)(end - begin), 0, total, blocks};
    for (int b0 = 0; b0 < a.items; b0 += 32) {
      const long long mine = b0 ? tiles_of(b0 + lane) : mine0, upto = before + scan(mine);
      const unsigned m = __ballot_sync(0xffffffffu, upto > begin);
      if (m) {
        const int at = __ffs(m) - 1;
        s.item = b0 + at;
        s.offset = begin - __shfl_sync(0xffffffffu, upto - mine, at);
        break;
      }
      before = __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) *start = s;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk<QT, BN> walk(k, *start);
  Piece p;
  // The ring's units of a piece of n tiles, counted from its first: in the order in which they are used.
  auto key_unit = [](int j) { return QT == 1 ? (j == 0 ? 0 : 2 * j - 1) : 2 * j; };
  auto value_unit = [](int j, int n) { return QT == 1 ? (j == n - 1 ? 2 * n - 1 : 2 * j + 2) : 2 * j + 1; };

  if (warp == PRODUCER_WARP) {
    const int per_tile = BN / k.box_rows, loads = per_tile * k.boxes;      // a lane's box: rows and columns of the tile (16 boxes at most)
    const int rows = k.tokens * a.G;
    long long u0 = 0;
    int it = 0;
    auto stopped = [&]() { return __shfl_sync(0xffffffffu, *abort, 0) != 0; };      // the same answer for all lanes, which go on together
    while (walk.next(p) && !stopped()) {
      const int* bt = p.it.bt;
      const int row = lane / k.boxes * k.box_rows, column = lane % k.boxes;
      auto page_at = [&](int j) {
        const int key = (p.l.t_begin + p.j0 + j) * BN + row;
        return lane < loads && j < p.n ? min(max(bt[min(key / a.page_size, a.bt_stride - 1)], 0), a.pages - 1) : 0;
      };
      int page = page_at(0), before = 0;
      mbar_wait(q_empty, (it & 1) ^ 1, abort, k.status);
      if (lane == 0) {
        mbar_expect_tx(q_full, (uint32_t)(QT * k.boxes * rows * 128));
        for (int s = 0; s < QT; ++s)
          for (int c = 0; c < k.boxes; ++c)
            tma_load(q_s + s * q_bytes + c * Q_COL_BYTES, &q_map, c * BOX, p.head * a.G, p.it.row0 + (p.part * QT + s) * k.tokens, q_full);
      }
      auto load = [&](int unit, int j, int page_id, int which) {
        const long long u = u0 + unit;
        const int s = (int)(u % k.ring);
        mbar_wait(&u_empty[s], (uint32_t)((u / k.ring) & 1) ^ 1, abort, k.status);
        if (lane == 0) mbar_expect_tx(&u_full[s], (uint32_t)unit_bytes);
        __syncwarp();
        if (lane < loads && !*abort) {
          const int key = (p.l.t_begin + p.j0 + j) * BN + row;
          const int y = ((page_id * 2 + which) * a.nkv + p.head) * a.page_size + key % a.page_size;      // (fits: the launcher asks for it)
          tma_load(ring_s + s * unit_bytes + column * COL_BYTES + row * 128, &kv_map, column * BOX, y, &u_full[s]);
        }
      };
      for (int j = 0; j < p.n && !stopped(); ++j) {
        const int next = page_at(j + 1);
        load(key_unit(j), j, page, 0);
        if constexpr (QT == 1) {
          if (j > 0) load(value_unit(j - 1, p.n), j - 1, before, 1);
          if (j == p.n - 1) load(value_unit(j, p.n), j, page, 1);
        } else {
          load(value_unit(j, p.n), j, page, 1);
        }
        before = page;
        page = next;
      }
      u0 += 2 * p.n;
      ++it;
    }
  } else if (warp == MMA_WARP) {
    if (lane == 0) {
      constexpr uint32_t IDESC_S = instr_desc(BM, BN, false);
      const uint32_t idesc_pv = instr_desc(BM, k.n_out, true);
      long long u0 = 0;
      int g0 = 0, it = 0;
      auto wait_unit = [&](int unit) {
        const long long u = u0 + unit;
        mbar_wait(&u_full[(int)(u % k.ring)], (uint32_t)((u / k.ring) & 1), abort, k.status);
        return smem_u32(ring_s + (int)(u % k.ring) * unit_bytes);
      };
      auto free_unit = [&](int unit) { tc_commit(&u_empty[(int)((u0 + unit) % k.ring)]); };
      auto scores = [&](int set, int buffer, uint32_t keys) {
        const uint64_t q_desc = smem_desc(smem_u32(q_s + set * q_bytes), 16, 1024), k_desc = smem_desc(keys, 16, 1024);
        for (int s = 0; s < k.steps; ++s) {
          const int in_box = (s & 3) * 2;      // 16 columns further: 32 bytes of a row of its box
          tc_mma(tmem + S_COL + BN * buffer, q_desc + (uint64_t)((s >> 2) * (Q_COL_BYTES >> 4) + in_box),
                 k_desc + (uint64_t)((s >> 2) * (COL_BYTES >> 4) + in_box), IDESC_S, s > 0 ? 1u : 0u);
        }
        tc_commit(&s_full[buffer]);
      };
      auto add = [&](int set, int buffer, uint32_t values, bool onto) {
        const uint64_t v_desc = smem_desc(values, COL_BYTES, 1024);
        for (int s = 0; s < BN / 16; ++s)      // 16 keys further: 2048 bytes of every box
          tc_mma_ts(tmem + 128 * set, tmem + S_COL + BN * buffer + P_AT + 8 * s, v_desc + (uint64_t)(s * (2048 >> 4)), idesc_pv, (onto || s > 0) ? 1u : 0u);
        tc_commit(&o_full[buffer]);
      };
      while (walk.next(p) && !*abort) {
        const int n = p.n;
        mbar_wait(q_full, it & 1, abort, k.status);
        tc_fence_after();
        if constexpr (QT == 1) {
          auto ahead = [&](int j) {
            const uint32_t keys = wait_unit(key_unit(j));
            if (*abort) return;
            tc_fence_after();
            scores(0, (g0 + j) & 1, keys);
            free_unit(key_unit(j));
            if (j == n - 1) tc_commit(q_empty);
          };
          for (int j = 0; j < min(n, 2) && !*abort; ++j) ahead(j);
          for (int j = 0; j < n && !*abort; ++j) {
            const int g = g0 + j;
            if (j == 0 && it > 0) mbar_wait(o_free, (it - 1) & 1, abort, k.status);      // the piece before has its sums in registers
            const uint32_t values = wait_unit(value_unit(j, n));
            mbar_wait(&p_full[g & 1], (g >> 1) & 1, abort, k.status);
            if (*abort) break;
            tc_fence_after();
            add(0, g & 1, values, j > 0);
            free_unit(value_unit(j, n));
            if (j + 2 < n) ahead(j + 2);
          }
        } else {
          uint32_t keys = wait_unit(key_unit(0));
          if (*abort) break;
          tc_fence_after();
          scores(0, 0, keys);
          scores(1, 1, keys);
          free_unit(key_unit(0));
          if (n == 1) tc_commit(q_empty);
          for (int j = 0; j < n && !*abort; ++j) {
            const int g = g0 + j;
            if (j == 0 && it > 0) mbar_wait(o_free, (it - 1) & 1, abort, k.status);
            const uint32_t values = wait_unit(value_unit(j, n));
            mbar_wait(&p_full[0], g & 1, abort, k.status);
            if (*abort) break;
            tc_fence_after();
            add(0, 0, values, j > 0);
            if (j + 1 < n) {
              keys = wait_unit(key_unit(j + 1));
              if (*abort) break;
              tc_fence_after();
              scores(0, 0, keys);
            }
            mbar_wait(&p_full[1], g & 1, abort, k.status);
            if (*abort) break;
            tc_fence_after();
            add(1, 1, values, j > 0);
            free_unit(value_unit(j, n));
            if (j + 1 < n) {
              scores(1, 1, keys);
              free_unit(key_unit(j + 1));
              if (j + 2 == n) tc_commit(q_empty);
            }
          }
        }
        u0 += 2 * n;
        g0 += n;
        ++it;
      }
    }
  } else {
    // Warp w: tensor-memory lanes 32 (w % 4) .. + 31.  QT = 1: columns W (w / 4) .. of their rows; QT = 2: all columns of set w / 4's rows.
    const int quarter = warp & 3, upper = warp >> 2, half = QT == 1 ? upper : 0, set = QT == 1 ? 0 : upper, r = quarter * 32 + lane;
    const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t o_addr = t_lane + 128 * set;
    int done[BUFFERS] = {};
    auto wait_o = [&](int g) {      // P V of tile g is added
      const int b = QT == 1 ? g & 1 : set, use = QT == 1 ? g >> 1 : g;
#pragma unroll
      for (int x = 0; x < BUFFERS; ++x)
        if (x == b) {
          while (done[x] <= use) {
            mbar_wait(&o_full[x], done[x] & 1, abort, k.status);
            ++done[x];
          }
        }
      tc_fence_after();
    };
    auto meet = [&]() {      // the two warps that share rows
      if constexpr (QT == 1) asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
    };
    const float factor = a.softcap > 0.f ? 1.f : k.scale_log2;      // capped scores come in base 2
    long long u0 = 0;
    int g = 0, it = 0;
    while (walk.next(p)) {
      const int tokens_left = p.it.n - (p.part * QT + set) * k.tokens, rows = min(max(tokens_left, 0), k.tokens) * a.G;
      const bool valid = r < rows, busy = quarter * 32 < rows;      // this row exists; one of the warp's does
      const int token = min(p.it.row0 + (p.part * QT + set) * k.tokens + r / a.G, p.it.row0 + p.it.n - 1);
      const int* mask = a.mask + (size_t)token * a.words;
      const int begin = a.window > 0 ? window_begin(a, a.positions[token]) : 0;
      // keys that the mask may hide from some row: the new ones and what lies behind, with a window those that it has passed for the last token
      const int hidden_from = p.it.start, hidden_to = a.window > 0 ? p.it.start + p.it.n - a.window : 0;
      float m_run = -INFINITY, l_run = 0.f;
      int touched = 0x7fffffff;      // first key of the first tile that the mask touched
      for (int j = 0; j < p.n; ++j, ++g) {
        const int b = QT == 1 ? g & 1 : set, key0 = (p.l.t_begin + p.j0 + j) * BN;
        const bool masked = key0 + BN > hidden_from || key0 < hidden_to;
        const uint32_t s_addr = t_lane + S_COL + BN * b;
        mbar_wait(&s_full[b], QT == 1 ? (g >> 1) & 1 : g & 1, abort, k.status);
        tc_fence_after();
        if (masked) {      // values that are not finite are taken out before P V multiplies them with weights of zero
          // (behind the scores: the ring's earlier uses of this unit are over then, so the barrier's parity is this one's)
          if (touched > key0) touched = key0;
          const long long u = u0 + value_unit(j, p.n);
          mbar_wait(&u_full[(int)(u % k.ring)], (uint32_t)((u / k.ring) & 1), abort, k.status);
          unsigned char* v_s = ring_s + (int)(u % k.ring) * unit_bytes;
          bool any = false;
          for (int i = threadIdx.x; i < unit_bytes / 16; i += 32 * SOFTMAX_WARPS) {
            uint4 x = *reinterpret_cast<const uint4*>(v_s + 16 * i);
            uint32_t* w4 = &x.x;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t hit = __vcmpeq2(w4[e] & 0x7f807f80u, 0x7f807f80u);
              bad |= hit != 0;
              w4[e] &= ~hit;
            }
            if (bad) {
              *reinterpret_cast<uint4*>(v_s + 16 * i) = x;
              any = true;
            }
          }
          if (any) spoiled[it & 1] = it + 1;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          asm volatile("bar.sync 5, 256;" ::: "memory");
        }
        if (busy) {
          constexpr int N = W < 64 ? W : 64;      // columns that a thread has in registers
          auto shape = [&](float (&v)[N], int col) {
            if (a.softcap > 0.f) {
#pragma unroll
              for (int e = 0; e < N; ++e) v[e] = mi::shaped_logit2(v[e], a.scale, a.softcap, false, 0.f);
            }
            if (masked) {
#pragma unroll
              for (int e0 = 0; e0 < N; e0 += 32) {
                const uint32_t bits = seen_bits(a, p.it, key0 + col + e0, begin, mask);
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e0 + e] = (bits >> e) & 1 ? v[e0 + e] : -INFINITY;
              }
            }
          };
          auto largest = [&](const float (&v)[N]) {
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < N; e += 2) mx4[e >> 1 & 3] = mi::max_of(mx4[e >> 1 & 3], v[e], v[e + 1]);
            return fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          };
          float v[N], mx;
          if constexpr (QT == 1) {
            tmem_ld(v, s_addr + W * half);
            shape(v, W * half);
            float* maxima = row_max + (g & 1) * 2 * BM;
            mx = largest(v);
            maxima[half * BM + r] = mx;
            tc_fence_before();
            meet();      // both halves of the scores are in registers: the weights may be written over them
            tc_fence_after();
            mx = fmaxf(mx, maxima[(half ^ 1) * BM + r]);
          } else {      // the second half of the scores stays in registers, the first is read again: the weights lie over the second
            tmem_ld(v, s_addr);
            shape(v, 0);
            mx = largest(v);
            tmem_ld(v, s_addr + 64);
            shape(v, 64);
            mx = fmaxf(mx, largest(v));
          }
          const float m_new = fmaxf(m_run, mx * factor);      // the scale is positive
          const bool move = m_new > m_run;
          if (__any_sync(0xffffffffu, move)) {
            const float alpha = move ? exp2f(m_run - m_new) : 1.f;
            if (j > 0) {
              wait_o(g - 1);
#pragma unroll 1
              for (int c = half; 32 * c < k.n_out; c += HALVES) {
                float o[32];
                uint32_t x[32];
                tmem_ld(o, o_addr + 32 * c);
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                  mi::mul_pair(o[e], o[e + 1], o[e], o[e + 1], alpha);
                  x[e] = __float_as_uint(o[e]);
                  x[e + 1] = __float_as_uint(o[e + 1]);
                }
                tmem_st(o_addr + 32 * c, x);
              }
            }
            l_run *= alpha;
            if (move) m_run = m_new;
          }
          const float m_use = m_run == -INFINITY ? 0.f : m_run;
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          auto weigh = [&](float (&v)[N], uint32_t to) {      // two keys to a column
            uint32_t packed[N / 2];
#pragma unroll
            for (int e = 0; e < N; e += 2) mi::fma_pair(v[e], v[e + 1], v[e], v[e + 1], factor, -m_use);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
              packed[e] = pack_bf16(mi::ex2_fast(v[2 * e]), mi::ex2_fast(v[2 * e + 1]));      // nothing where the row may not see the key
              mi::add_pair(part[2 * e & 3], part[(2 * e + 1) & 3], __uint_as_float(packed[e] << 16), __uint_as_float(packed[e] & 0xffff0000u));
            }
            tmem_st(to, packed);
          };
          if constexpr (QT == 1) {
            weigh(v, s_addr + W / 2 * half);
          } else {
            weigh(v, s_addr + 96);
            tmem_ld(v, s_addr);
            shape(v, 0);
            weigh(v, s_addr + 64);
          }
          l_run += (part[0] + part[1]) + (part[2] + part[3]);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        if (g >= LAG) wait_o(g - LAG);      // long done: keeps this thread in step with the barrier
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[b]);
      }
#pragma unroll
      for (int back = LAG; back > 0; --back)
        if (g >= back) wait_o(g - back);
      const bool whole = p.whole;
      const bool fix = spoiled[it & 1] == it + 1;
      float l_all = l_run;
      if constexpr (QT == 1) {
        row_sum[half * BM + r] = l_run;
        meet();
        l_all = row_sum[r] + row_sum[BM + r];
      }
      const int h = p.head * a.G + r % a.G;
      float mult = 1.f;
      if (whole) {
        const float sink2 = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
        const float top = fmaxf(m_run, sink2), off = top == -INFINITY ? 0.f : top, weight = exp2f(m_run - off);
        const float total = l_all * weight + exp2f(sink2 - off);
        mult = total == 0.f ? 0.f : weight / total;      // nothing visible: zeros
      }
      const int key_end = min(p.it.ctx, (p.l.t_begin + p.j0 + p.n) * BN);
      const size_t at = (size_t)p.slot * (QT * BM) + set * BM + r;      // row of the sums
      if (busy) {
#pragma unroll 1
        for (int c = half; 32 * c < k.n_out; c += HALVES) {
          float o[32];
          tmem_ld(o, o_addr + 32 * c);
          if (valid && !*abort) {
            if (fix) {
              float more[32] = {};
              add_not_finite(a, p.it, p.head, touched, key_end, begin, mask, 32 * c, more);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] += more[e];
            }
            if (whole) {
              __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)token * a.nh * a.hd + (size_t)h * a.hd + 32 * c;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (32 * c + 8 * q < a.hd) {      // (a head size is a multiple of 16)
                  uint32_t x[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) x[e] = pack_bf16(o[8 * q + 2 * e] * mult, o[8 * q + 2 * e + 1] * mult);
                  *reinterpret_cast<uint4*>(dst + 8 * q) = make_uint4(x[0], x[1], x[2], x[3]);
                }
            } else {
              float* dst = a.part_o + at * a.hd + 32 * c;
#pragma unroll
              for (int q = 0; q < 8; ++q)
                if (32 * c + 4 * q < a.hd) *reinterpret_cast<float4*>(dst + 4 * q) = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
            }
          }
          __syncwarp();
        }
        if (!whole && valid && half == 0 && !*abort) *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(m_run, l_all);
      }
      if (threadIdx.x == 0 && p.j0 == 0) {      // the unit's pieces, for the kernel that joins them
        const int blocks = start->blocks, me = (int)blockIdx.x;
        const long long total = start->total, g_last = stretch_begin(total, me, blocks) + (start->left - walk.left) - p.n + p.l.tiles - 1;
        int last = me;
        if (!whole) {      // the block whose stretch holds the unit's last tile
          last = (int)(g_last * blocks / total);
          while (last + 1 < blocks && stretch_begin(total, last + 1, blocks) <= g_last) ++last;
        }
        k.units[((size_t)p.b * a.nkv + p.head) * k.max_parts + p.part] = make_int2(me, last - me + 1);
      }
      tc_fence_before();
      meet();      // (the sums are read too: the next piece may leave its own)
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      u0 += 2 * p.n;
      ++it;
    }
  }
  // every tensor-memory access is done, then the columns go back
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM_COLS) : "memory");
  }
}

// The pieces of units that several blocks shared, added up: grid (items * nkv * max_parts, rows / JOIN_WARPS), a warp a row, four values a lane.
constexpr int JOIN_WARPS = 8;
template <int QT>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
tree_join_kernel(const Tc k) {
  const Args& a = k.a;
  const int unit = blockIdx.x, part = unit % k.max_parts, head = unit / k.max_parts % a.nkv, b = unit / k.max_parts / a.nkv;
  const int row = blockIdx.y * JOIN_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;      // of the unit's QT * 128
  mi::grid_dependency_sync();
  const Item it = item_of(a, b);
  const int set = row / BM, r = row - set * BM, first = (part * QT + set) * k.tokens;
  if (r >= min(k.tokens, it.n - first) * a.G) return;
  const int2 u = k.units[unit];
  const int pieces = u.y;
  if (pieces <= 1) return;
  // piece s lies in block u.x + s: its first piece where the unit begins there, else the one that its stretch begins with
  auto slot = [&](int s) { return (size_t)(2 * (u.x + s) + (s == 0 ? 1 : 0)) * (QT * BM) + row; };
  const int h = head * a.G + r % a.G;
  const float sink2 = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
  float2 mine = make_float2(-INFINITY, 0.f);
  if (lane < pieces) mine = *reinterpret_cast<const float2*>(a.part_ml + 2 * slot(lane));
  float top = fmaxf(mine.x, sink2);
  for (int s = 32 + lane; s < pieces; s += 32) top = fmaxf(top, a.part_ml[2 * slot(s)]);
  top = mi::warp_max(top);
  const float off = top == -INFINITY ? 0.f : top;
  float f = exp2f(mine.x - off), total = mine.y * f;
  float acc[2][4] = {};
#pragma unroll 1
  for (int s0 = 0; s0 < pieces; s0 += 32) {
    if (s0 > 0) {
      mine = s0 + lane < pieces ? *reinterpret_cast<const float2*>(a.part_ml + 2 * slot(s0 + lane)) : make_float2(-INFINITY, 0.f);
      f = exp2f(mine.x - off);
      total += mine.y * f;
    }
    const int near = min(32, pieces - s0);
#pragma unroll 4
    for (int s = 0; s < near; ++s) {
      const float w = __shfl_sync(0xffffffffu, f, s);
      const float* src = a.part_o + slot(s0 + s) * a.hd;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (128 * c + 4 * lane < a.hd) {
          const float4 x = *reinterpret_cast<const float4*>(src + 128 * c + 4 * lane);
          acc[c][0] = fmaf(x.x, w, acc[c][0]);
          acc[c][1] = fmaf(x.y, w, acc[c][1]);
          acc[c][2] = fmaf(x.z, w, acc[c][2]);
          acc[c][3] = fmaf(x.w, w, acc[c][3]);
        }
    }
  }
  total = mi::warp_sum(total) + exp2f(sink2 - off);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) + ((size_t)(it.row0 + first + r / a.G) * a.nh + h) * a.hd;
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (128 * c + 4 * lane < a.hd)
      *reinterpret_cast<uint2*>(dst + 128 * c + 4 * lane) = make_uint2(pack_bf16(acc[c][0] * inv, acc[c][1] * inv), pack_bf16(acc[c][2] * inv, acc[c][3] * inv));
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = (EncodeFn)p;
  }
  return fn;
}

template <int QT, int BN>
int launch(Tc& k, const CUtensorMap& q_map, const CUtensorMap& kv_map, int blocks, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return mi_fail("attention_tree_tc: no current device");
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(tree_tc_kernel<QT, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess)
      return mi_fail("attention_tree_tc: %d bytes of shared memory were refused", SMEM_BYTES);
    ready[dev] = true;
  }
  k.ring = (SMEM_BYTES - 1024 - SMEM_TAIL - QT * k.boxes * BM * 128) / (k.boxes * BN * 128);
  if (k.ring > MAX_UNITS) k.ring = MAX_UNITS;
  MI_REQUIRE(k.ring >= 4, "attention_tree_tc: no room for a ring of tiles of %d boxes", k.boxes);
  if (mi::launch(tree_tc_kernel<QT, BN>, dim3(blocks), dim3(THREADS), SMEM_BYTES, stream, q_map, kv_map, k) != cudaSuccess)
    return mi_fail("attention_tree_tc: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  const Args& a = k.a;
  const int rows = a.max_q * a.G < QT * BM ? a.max_q * a.G : QT * BM;      // (a set's last rows may be empty: groups that do not divide 128)
  const int join_rows = QT == 2 && rows > BM ? QT * BM : rows;
  if (mi::launch(tree_join_kernel<QT>, dim3(a.items * a.nkv * k.max_parts, (join_rows + JOIN_WARPS - 1) / JOIN_WARPS), dim3(32 * JOIN_WARPS), 0, stream, k) != cudaSuccess)
    return mi_fail("attention_tree_tc: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  MI_LAUNCH_OK("attention_tree_tc");
  return 0;
}

// Sets of 128 rows that a block takes at a time: two once the largest item has more rows than one holds, as far as tensor memory goes.
int sets_of(int max_q, int G, int hd) { return hd <= 128 && max_q > BM / G ? 2 : 1; }

}  // namespace

// Whether the kernel takes these sizes and addresses.
MI_API int mi_attention_tree_tc_takes(const void* out, const void* qkv, const void* kv, int T, int width, int nh, int nkv, int hd, long long pages, int page_size, int max_q, float scale) {
  return nkv > 0 && nh % nkv == 0 && nh / nkv <= BM && hd % 16 == 0 && hd >= 64 && hd <= 256 && width % 8 == 0 && page_size % 16 == 0 && scale > 0.f && T > 0 &&
         (((uintptr_t)out | (uintptr_t)qkv | (uintptr_t)kv) % 16) == 0 && pages * 2 * nkv * page_size <= 0x7fffffffll && max_q > 0;
}
// Floats of scratch: the units' pieces, the sums.
MI_API long long mi_attention_tree_tc_floats(int items, int nh, int nkv, int hd, int max_q) {
  const int G = nh / nkv, qt = sets_of(max_q, G, hd), tokens = BM / G, parts = (max_q + qt * tokens - 1) / (qt * tokens);
  return 4ll * items * nkv * parts + 2ll * mi::sm_count() * qt * BM * (hd + 2);
}

// bfloat16, what mi_attention_tree_tc_takes says.  scratch: mi_attention_tree_tc_floats floats, 16-byte aligned; status: one word, set to 2 if a
// bounded wait ran out.
MI_API int mi_attention_tree_tc(void* out, const void* qkv, const void* kv, const int* block_table, int bt_stride, const int* q_start, const int* q_len,
                                const int* ctx_len, const int* seq_slot, const int* mask, int words, const int* positions, const float* sink, float* scratch,
                                int* status, int items, int T, int width, int nh, int nkv, int hd, int pages, int page_size, int window, int max_q, float scale,
                                float softcap, cudaStream_t stream) {
  MI_REQUIRE(mi_attention_tree_tc_takes(out, qkv, kv, T, width, nh, nkv, hd, pages, page_size, max_q, scale), "attention_tree_tc: sizes or addresses that it does not take");
  MI_REQUIRE(items >= 0 && bt_stride > 0 && pages > 0 && (long long)words * 32 >= max_q && ((uintptr_t)scratch % 16) == 0, "attention_tree_tc: bad sizes items=%d words=%d max_q=%d", items, words, max_q);
  if (items == 0) return 0;
  const EncodeFn encode = encoder();
  if (!encode) return mi_fail("attention_tree_tc: the driver does not offer cuTensorMapEncodeTiled");
  const int G = nh / nkv, qt = sets_of(max_q, G, hd);
  Tc k{};
  k.status = status;
  k.boxes = (hd + BOX - 1) / BOX;
  k.steps = hd / 16;
  k.n_out = k.boxes * BOX;
  k.box_rows = page_size % 64 == 0 ? 64 : page_size % 32 == 0 ? 32 : 16;
  k.tokens = BM / G;
  k.max_parts = (max_q + qt * k.tokens - 1) / (qt * k.tokens);
  k.scale_log2 = scale * 1.4426950408889634f;
  const long long units = (long long)items * nkv * k.max_parts;
  MI_REQUIRE(units <= 0x7fffffffll, "attention_tree_tc: %d items of %d heads in %d parts are too many", items, nkv, k.max_parts);
  const int blocks = mi::sm_count();
  k.units = (int2*)scratch;
  float* part_o = scratch + 4 * units;
  float* part_ml = part_o + 2ll * blocks * qt * BM * hd;
  k.a = Args{out, qkv, kv, block_table, bt_stride, q_start, q_len, ctx_len, seq_slot, mask, words, positions, sink, part_o, part_ml,
             items, T, width, nh, nkv, G, hd, pages, page_size, window, max_q, scale, softcap};
  CUtensorMap q_map, kv_map;
  {
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)nh, (cuuint64_t)T}, strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)width * 2};
    const cuuint32_t box[3] = {BOX, (cuuint32_t)G, (cuuint32_t)k.tokens}, elem[3] = {1, 1, 1};
    const CUresult r = encode(&q_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(qkv), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return mi_fail("attention_tree_tc: cuTensorMapEncodeTiled of the queries failed with code %d", (int)r);
  }
  {
    const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)pages * 2 * nkv * page_size}, strides[1] = {(cuuint64_t)hd * 2};
    const cuuint32_t box[2] = {BOX, (cuuint32_t)k.box_rows}, elem[2] = {1, 1};
    const CUresult r = encode(&kv_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(kv), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return mi_fail("attention_tree_tc: cuTensorMapEncodeTiled of the cache failed with code %d", (int)r);
  }
  if (qt == 2) return launch<2, 128>(k, q_map, kv_map, blocks, stream);
  return hd <= 128 ? launch<1, 128>(k, q_map, kv_map, blocks, stream) : launch<1, 64>(k, q_map, kv_map, blocks, stream);
}
