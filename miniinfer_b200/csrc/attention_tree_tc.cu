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
// a lane a box, the next tile's pages looked up ahead), a warp that issues all products, and two sets of four softmax warps, a thread a row, that take
// turns on the tensor cores and on the exponentials: one set's scores are made while the other's weights are.  Weights stay in tensor memory, over the scores they come
// from.  With up to 128 rows the sets are two streams of key tiles of the same rows, put together at the end of a piece; with up to 256 they are two sets of rows on
// the same tiles, whose keys and values are fetched once for both.  Heads beyond 128 leave tensor memory for one set's sums only.
//
// Weights of invisible keys are zeros in P V, so whatever is not finite among the values of a tile that the mask touches is taken out in
// shared memory first; a row that does see such a value gets it added at the end.  Only those tiles pay for it.
//
// Weights are relative to a maximum that may lag behind the row's by 2^8, so that a row of sums is rescaled a few times and not in every tile; they are
// rounded to bf16, as the tensor cores take them, and the sum that divides the row is that of the rounded ones.
//
// Measured, heads of 128: 32 trees of 64 over up to 8192 keys, 32 heads on 8 (625 MB, 105 GFLOP) 180 us in short bursts, 200 to 215 one call after the other (the power cap): 3.5 and 2.9 to 3.1 TB/s; 8 trees of 32 over up to
// 4096 keys (62 MB) 24 to 26 us, with a cap of 30 37.5, with pages of 16 30.5, heads of 64 and 256 21.8 and 40.3; one tree of 8 over 2047 keys, 16 heads on 8 (8.5 MB) 16.5 us.  The first is
// bound by the chain from scores over exponentials to weights (with a cap, whose exponentials and reciprocals come on top, 404 us): two sets of rows leave the tensor cores 35 % busy,
// without the softmax the products and copies alone took 130 us.  The others are bound by what a
// piece costs whatever its length is - its description, its queries, the first tile's latency, its sums - about 4000 cycles, and 10000 once a block.
#include <cuda.h>
#include <string.h>

#include "attention_tree.cuh"

namespace {

using namespace mi_tree;

constexpr int BM = 128, BOX = 64, BUFFERS = 2;
constexpr int TMEM_COLS = 512, S_COL = 256;
constexpr int MAX_UNITS = 12;                 // boxes of the ring: a tile's keys or its values each
constexpr int WAIT_LIMIT = 1 << 22;
constexpr int STATUS_LATE = 64, STATUS_PLACE = 128;      // bits of the status word: a bounded wait ran out; shared memory is not laid out as the kernel needs it
constexpr int SMEM_BYTES = 227 << 10;
constexpr int BARS = 80;                      // 8-byte words behind queries and ring: barriers, pieces

struct Tc {
  Args a;
  int* status;
  int* counters;                 // [items * nkv * max_parts], zero, left zero: pieces of a unit that have come; null: tree_join_kernel joins them
  int4* joins;                   // [blocks]: of the unit that begins in a block and goes on in others: pieces, first token, tokens, key/value head
  int boxes, steps, n_out;       // boxes and 16s of columns of a row, columns of P V
  int ring, box_rows;            // units of the ring; rows of a TMA box of keys
  int tokens, max_parts;         // tokens of a set of 128 rows; parts of the largest item
  float scale_log2;              // scale * log2(e)
  float cap_scale, cap_log2;     // with a cap: 2 scale log2(e) / cap, cap log2(e)
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
  atomicOr(status, STATUS_LATE);
}
// The wait at a role's end: what it has started itself, copies or products, is over before the block is.  It does not ask for `abort`, but has a limit too.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  for (int i = 0; i < WAIT_LIMIT; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    if (done) return;
  }
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
// True in one thread of a warp that is together.
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
  return yes != 0;
}
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
__device__ __forceinline__ void tmem_ld(float (&v)[16], uint32_t taddr) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
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

// The line of work: item after item, in an item head after head, in a head part after part (QT * tokens tokens each).  A unit takes its
// tiles and `overhead` more in front of them: what queries, the first copies and the results cost, as long as a block has several tiles.
// From that many tiles a block on.  24 sizes - 4 to 64 requests, trees of 8 to 64, contexts of 512 to 8192, heads of 64 to 256 - without it 2 to 16 % slower in 20, equal
// in 4; with it from none on 11 % slower at 1 to 3 tiles a block in two, 5 % faster in one.
constexpr int OVERHEAD = 4, OVERHEAD_FROM = 4;
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
// Block b's stretch: `base` places of the line, one more for the first `more` blocks; and the block that a place belongs to.
__device__ __forceinline__ int stretch_begin(int base, int more, int b) { return b * base + min(b, more); }
__device__ __forceinline__ int stretch_of(int base, int more, int place) {
  const int longer = more * (base + 1);
  return place < longer ? place / (base + 1) : more + (place - longer) / base;
}

// Where a block's stretch begins, and how long it is.
struct Start {
  Item it;                       // the first item
  int item, left, offset;        // its number; places of the stretch; places of the item before it
};

// A piece of a unit: some of its tiles, as the producer describes it to the other warps.
struct Piece {
  Item it;
  int n, key;                    // tiles (0: no piece is left), first key
  int head, first;               // key/value head; the unit's first token in the item
  int slot;                      // of the sums, where the unit goes on in other blocks; -1: it does not
  int unit, block, pieces;       // the unit's number, its first block, in how many blocks it lies
};
constexpr int PIECES = 4;        // that are described at a time: the producer is at most two ahead of the last reader

template <int QT, int BN>
struct Walk {
  const Tc& k;
  int item, left, offset, place, base, more, overhead;      // place: where on the line the walk is
  Item it;
  Line l;
  __device__ Walk(const Tc& k_, const Start& s, int place_, int base_, int more_, int overhead_)
      : k(k_), item(s.item), left(s.left), offset(s.offset), place(place_), base(base_), more(more_), overhead(overhead_), it(s.it), l(line_of<QT, BN>(k_, s.it)) {}
  __device__ bool next(Piece& p) {
    while (left > 0) {
      const int all = (l.tiles + overhead) * k.a.nkv * l.parts;
      if (offset >= all) {      // (also items without tokens)
        offset -= all;
        if (++item >= k.a.items) return false;
        it = item_of(k.a, item);
        l = line_of<QT, BN>(k, it);
        continue;
      }
      const int unit = offset / (l.tiles + overhead), at = offset - unit * (l.tiles + overhead), n = min(left, (l.tiles + overhead) - at);      // places of the unit in this stretch
      const int j0 = max(at - overhead, 0), j1 = max(at + n - overhead, 0), first_tile = place - at + overhead;
      offset += n;
      left -= n;
      place += n;
      if (j1 <= j0) continue;
      p.it = it;
      p.n = j1 - j0;
      p.key = (l.t_begin + j0) * BN;
      p.head = unit / l.parts;
      const int part = unit - p.head * l.parts;
      p.first = part * QT * k.tokens;
      p.slot = p.n == l.tiles ? -1 : 2 * (int)blockIdx.x + (j0 == 0 ? 1 : 0);
      p.unit = (item * k.a.nkv + p.head) * k.max_parts + part;
      p.block = p.n == l.tiles ? (int)blockIdx.x : stretch_of(base, more, first_tile);
      p.pieces = p.n == l.tiles ? 1 : stretch_of(base, more, first_tile + l.tiles - 1) - p.block + 1;
      return true;
    }
    return false;
  }
};

// Bits of the keys key0 .. key0 + 31 that a row sees: of the context from `begin` on, of the new ones by the token's mask (and the window).
// near: the mask's first 64 bits.
__device__ __forceinline__ uint32_t seen_bits(const Args& a, const Item& it, int key0, int begin, const int* mask, uint64_t near) {
  auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
  uint32_t bits = below(it.start - key0) & ~below(begin - key0);
  const int j0 = key0 - it.start;
  if (j0 > -32 && j0 < it.n) {
    uint32_t nodes;
    if (j0 < 0) {
      nodes = (uint32_t)near << -j0;
    } else if (it.n <= 64) {
      nodes = (uint32_t)(near >> j0);
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
__device__ __forceinline__ void add_not_finite(const Args& a, const Item& it, int head, int key_begin, int key_end, int begin, const int* mask, uint64_t near, int col, float (&o)[32]) {
  const __nv_bfloat16* kv = reinterpret_cast<const __nv_bfloat16*>(a.kv);
  for (int key0 = key_begin; key0 < key_end; key0 += 32) {
    for (uint32_t bits = seen_bits(a, it, key0, begin, mask, near); bits; bits &= bits - 1) {
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

// Row r of set `set` of a unit that lies in u.x blocks from `first` on - its first token u.y, tokens u.z, key/value head u.w -, columns 4 f0 .. 4 (f0 + F) - 1: the
// pieces' sums added up.  Piece s lies in block first + s: as that block's second of the sums where the unit begins there, else as its first.
template <int QT, int F, int AT_ONCE>
__device__ __forceinline__ void join_row(const Tc& k, int first, const int4& u, int set, int r, int f0) {
  const Args& a = k.a;
  const int row = set * BM + r, pieces = u.x, token = u.y + set * k.tokens + r / a.G, h = u.w * a.G + r % a.G;
  if (r >= min(k.tokens, u.z - set * k.tokens) * a.G || 4 * f0 >= a.hd) return;
  const float2* sums = reinterpret_cast<const float2*>(a.part_ml) + row;
  const float4* values = reinterpret_cast<const float4*>(a.part_o) + (size_t)f0 * (QT * BM) + row;
  const float sink2 = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
  float top = sink2, total = a.sink ? 1.f : 0.f;
  float acc[F][4] = {};
#pragma unroll 1
  for (int s0 = 0; s0 < pieces; s0 += AT_ONCE) {
    float2 ml[AT_ONCE];
    float4 x[AT_ONCE][F];
#pragma unroll
    for (int s = 0; s < AT_ONCE; ++s) {
      ml[s] = make_float2(-INFINITY, 0.f);
      const size_t at = 2 * (first + s0 + s) + (s0 + s == 0 ? 1 : 0);
      if (s0 + s < pieces) ml[s] = __ldcg(sums + at * (QT * BM));
#pragma unroll
      for (int f = 0; f < F; ++f) {
        x[s][f] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s0 + s < pieces) x[s][f] = __ldcg(values + (at * (k.n_out / 4) + f) * (QT * BM));
      }
    }
    float next = top;
#pragma unroll
    for (int s = 0; s < AT_ONCE; ++s) next = fmaxf(next, ml[s].x);
    const float off = next == -INFINITY ? 0.f : next, alpha = exp2f(top - off);
    top = next;
    total *= alpha;
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[f][e] *= alpha;
#pragma unroll
    for (int s = 0; s < AT_ONCE; ++s) {
      const float w = exp2f(ml[s].x - off);
      total = fmaf(ml[s].y, w, total);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        acc[f][0] = fmaf(x[s][f].x, w, acc[f][0]);
        acc[f][1] = fmaf(x[s][f].y, w, acc[f][1]);
        acc[f][2] = fmaf(x[s][f].z, w, acc[f][2]);
        acc[f][3] = fmaf(x[s][f].w, w, acc[f][3]);
      }
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;      // nothing visible: zeros
  __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) + ((size_t)token * a.nh + h) * a.hd + 4 * f0;
#pragma unroll
  for (int f = 0; f < F; f += 2)      // (a head size is a multiple of 16)
    if (4 * (f0 + f) < a.hd)
      *reinterpret_cast<uint4*>(dst + 4 * f) = make_uint4(pack_bf16(acc[f][0] * inv, acc[f][1] * inv), pack_bf16(acc[f][2] * inv, acc[f][3] * inv),
                                                          pack_bf16(acc[f + 1][0] * inv, acc[f + 1][1] * inv), pack_bf16(acc[f + 1][2] * inv, acc[f + 1][3] * inv));
}

// A wait has run out here, or in a call before that shared the counters, which are then not what they should be: all rows become NaN, and
// so do the sums that this block owes to those who join them.
template <int QT>
__device__ __forceinline__ void give_up(const Tc& k) {
  const Args& a = k.a;
#pragma unroll 1
  for (int b = 0; b < a.items; ++b) {
    const Item it = item_of(a, b);
    __nv_bfloat16* rows = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)it.row0 * a.nh * a.hd;
#pragma unroll 1
    for (size_t i = threadIdx.x; i < (size_t)it.n * a.nh * a.hd; i += blockDim.x) rows[i] = __float2bfloat16(NAN);
  }
#pragma unroll 1
  for (int i = threadIdx.x; i < 2 * QT * BM; i += blockDim.x) reinterpret_cast<float2*>(a.part_ml)[(size_t)2 * blockIdx.x * QT * BM + i] = make_float2(NAN, NAN);
}

constexpr int threads_of(int sets) { return 32 * (4 * sets + 2); }

template <int QT, int SETS, int BN, int STEPS>
__global__ void __launch_bounds__(threads_of(SETS), 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map, const Tc k) {
  constexpr int SOFTMAX_WARPS = 4 * SETS, PRODUCER_WARP = SOFTMAX_WARPS, MMA_WARP = SOFTMAX_WARPS + 1;
  constexpr int N = 64;                                 // scores in registers at a time; their weights lie over the first half of them
  constexpr int COL_BYTES = BN * 128, Q_COL_BYTES = BM * 128;
  const Args& a = k.a;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw;             // aligned, for the kernel has no other shared memory; the ring leaves no room to move
  if (smem_u32(smem) & 1023u) {
    mi::grid_dependency_sync();
    if (threadIdx.x == 0) {
      atomicOr(k.status, STATUS_PLACE);
      k.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    give_up<QT>(k);
    return;
  }
  const int q_bytes = k.boxes * Q_COL_BYTES, unit_bytes = k.boxes * COL_BYTES;      // of a set of rows; of a tile's keys or values
  unsigned char *q_s = smem, *ring_s = smem + QT * q_bytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring_s + k.ring * unit_bytes);
  uint64_t *q_full = bars, *q_empty = bars + 1, *o_free = bars + 2;
  uint64_t *piece_full = bars + 3;                       // [PIECES]: described
  uint64_t *u_full = piece_full + PIECES, *u_empty = u_full + MAX_UNITS;
  uint64_t *s_full = u_empty + MAX_UNITS, *p_full = s_full + BUFFERS, *o_full = p_full + BUFFERS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + BUFFERS);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* spoiled = abort + 1;      // [2]: the last piece, by parity, in which a value was not finite
  volatile int* last_to_come = spoiled + 2;
  uint64_t* drained = bars + 43;        // the last products are done
  Piece* pieces = reinterpret_cast<Piece*>(bars + 44);
  float2* of_set = reinterpret_cast<float2*>(bars + BARS);      // [2][BM]: a row's maximum and sum in each stream of keys, at a piece's end
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(o_free, SOFTMAX_WARPS);
    mbar_init(drained, 1);
    for (int u = 0; u < k.ring; ++u) {
      mbar_init(&u_full[u], 1);
      mbar_init(&u_empty[u], 1);
    }
    for (int i = 0; i < PIECES; ++i) mbar_init(&piece_full[i], 1);
    for (int b = 0; b < BUFFERS; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 4);      // the warps of a set
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The values of tile j of a piece of n tiles, as a unit of the ring counted from the piece's first.
  constexpr bool KEYS = QT == 1 && SETS == 2;           // the sets are streams of keys
  auto value_unit = [](int j, int n) { return KEYS ? (j == n - 1 ? 2 * n - 1 : 2 * j + 2) : 2 * j + 1; };

  if (warp == PRODUCER_WARP) {
    const int late = lane == 0 ? *reinterpret_cast<volatile int*>(k.status) : 0;      // (on its way beside the items' sizes)
    // where this block's stretch of the line begins
    int overhead = 0;
    auto places_of = [&](const Item& it) {
      const Line l = line_of<QT, BN>(k, it);
      return it.n > 0 ? (l.tiles + overhead) * a.nkv * l.parts : 0;
    };
    auto item_at = [&](int b) { return b < a.items ? item_of(a, b) : Item{0, 0, 0, 0, nullptr}; };
    auto scan = [&](int x) {      // sums up to and with this lane
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      return x;
    };
    const Item mine0 = item_at(lane);      // the first 32 items stay in registers
    auto all_places = [&]() {
      int x = places_of(mine0);
      for (int b0 = 32; b0 < a.items; b0 += 32) x += places_of(item_at(b0 + lane));
      return __reduce_add_sync(0xffffffffu, x);
    };
    int total = all_places();
    if (total >= OVERHEAD_FROM * (int)gridDim.x) {
      overhead = OVERHEAD;
      total = all_places();
    }
    const int upto0 = scan(places_of(mine0));
    const int me = (int)blockIdx.x, base = total / (int)gridDim.x, more = total - base * (int)gridDim.x;
    const int begin = stretch_begin(base, more, me);
    Start from{Item{0, 0, 0, 0, nullptr}, 0, 0, 0};
    int before = 0;
    for (int b0 = 0; b0 < a.items; b0 += 32) {
      const Item mine = b0 ? item_at(b0 + lane) : mine0;
      const int upto = b0 ? before + scan(places_of(mine)) : upto0;
      const unsigned m = __ballot_sync(0xffffffffu, upto > begin);
      if (m) {
        const int at = __ffs(m) - 1, prior = __shfl_sync(0xffffffffu, upto, max(at - 1, 0));
        from.it = Item{__shfl_sync(0xffffffffu, mine.row0, at), __shfl_sync(0xffffffffu, mine.n, at), __shfl_sync(0xffffffffu, mine.start, at),
                       __shfl_sync(0xffffffffu, mine.ctx, at), reinterpret_cast<const int*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine.bt), at))};
        from.item = b0 + at;
        from.left = base + (me < more ? 1 : 0);
        from.offset = begin - (at > 0 ? prior : before);
        break;
      }
      before = __shfl_sync(0xffffffffu, upto, 31);
    }
    Walk<QT, BN> walk(k, from, begin, base, more, overhead);
    const int per_tile = BN / k.box_rows, loads = per_tile * k.boxes;      // a lane's box: rows and columns of the tile (16 boxes at most)
    const int rows = k.tokens * a.G;
    int4 joined = make_int4(0, 0, 0, 0);      // for the kernel that joins pieces
    int slot = 0, turn = 1, it = 0;      // the ring's next unit; the parity that its barrier of free units is waited with
    int units = 0;                       // asked for so far
    auto stopped = [&]() { return __shfl_sync(0xffffffffu, *abort, 0) != 0; };      // the same answer for all lanes, which go on together
    const bool lost = __shfl_sync(0xffffffffu, late, 0) != 0;
    for (;; ++it) {
      Piece p;
      const bool more_pieces = !lost && walk.next(p);
      if (!more_pieces) p.n = 0;
      if (lost) *abort = 1;
      const int* bt = p.it.bt;
      const int row = lane / k.boxes * k.box_rows, column = lane % k.boxes;
      auto page_at = [&](int j) {
        const int key = p.key + j * BN + row;
        return lane < loads && j < p.n ? min(max(bt[min(key / a.page_size, a.bt_stride - 1)], 0), a.pages - 1) : 0;
      };
      int page = page_at(0), behind = 0;
      mbar_wait(q_empty, (it & 1) ^ 1, abort, k.status);
      if (stopped() && !lost) break;
      if (lane == 0) {
        pieces[it % PIECES] = p;
        mbar_arrive(&piece_full[it % PIECES]);
      }
      if (!more_pieces) break;
      if (lane == 0) {
        if (p.pieces > 1 && p.block == me) joined = make_int4(p.pieces, p.it.row0 + p.first, min(p.it.n - p.first, QT * k.tokens), p.head);
        mbar_expect_tx(q_full, (uint32_t)(QT * k.boxes * rows * 128));
        for (int s = 0; s < QT; ++s)
          for (int c = 0; c < k.boxes; ++c)
            tma_load(q_s + s * q_bytes + c * Q_COL_BYTES, &q_map, c * BOX, p.head * a.G, p.it.row0 + p.first + s * k.tokens, q_full);
      }
      auto load = [&](int j, int page_id, int which) {
        const int s = slot;
        mbar_wait(&u_empty[s], (uint32_t)turn, abort, k.status);
        if (stopped()) return;      // (all lanes or none: a unit whose boxes are not all on their way would never be full)
        if (++slot == k.ring) {
          slot = 0;
          turn ^= 1;
        }
        ++units;
        if (lane == 0) mbar_expect_tx(&u_full[s], (uint32_t)unit_bytes);
        __syncwarp();
        if (lane < loads) {
          const int key = p.key + j * BN + row;
          const int y = ((page_id * 2 + which) * a.nkv + p.head) * a.page_size + key % a.page_size;      // (fits: the launcher asks for it)
          tma_load(ring_s + s * unit_bytes + column * COL_BYTES + row * 128, &kv_map, column * BOX, y, &u_full[s]);
        }
      };
      for (int j = 0; j < p.n && !stopped(); ++j) {
        const int next = page_at(j + 1);
        load(j, page, 0);
        if constexpr (KEYS) {      // in the order in which they are used: keys run a tile ahead
          if (j > 0) load(j - 1, behind, 1);
          if (j == p.n - 1) load(j, page, 1);
        } else {
          load(j, page, 1);
        }
        behind = page;
        page = next;
      }
    }
    if (lane == 0) k.joins[me] = joined;
    // no copy is on its way into this block's memory when the block ends, also where a wait has run out
    for (int u = max(units - k.ring, 0); u < units; ++u) mbar_drain(&u_full[u % k.ring], (uint32_t)(u / k.ring & 1));
    if (it > 0) mbar_drain(q_full, (uint32_t)(it - 1) & 1);
  } else if (warp == MMA_WARP) {
    {      // the whole warp goes through the waits together, one elected thread issues: descriptors then stay in uniform registers
      auto stopped = [&]() { return __shfl_sync(0xffffffffu, *abort, 0) != 0; };
      constexpr uint32_t IDESC_S = instr_desc(BM, BN, false);
      const uint32_t idesc_pv = instr_desc(BM, k.n_out, true);
      int done[2] = {0, 0}, it = 0, slot = 0, turn = 0;      // tiles of a set
      auto next_unit = [&]() {      // the ring's next unit, once it is there
        const int s = slot;
        mbar_wait(&u_full[s], (uint32_t)turn, abort, k.status);
        if (++slot == k.ring) {
          slot = 0;
          turn ^= 1;
        }
        return s;
      };
      auto unit_at = [&](int s) { return smem_u32(ring_s + s * unit_bytes); };
      auto free_unit = [&](int s) {
        if (elected()) tc_commit(&u_empty[s]);
        __syncwarp();
      };
      auto scores = [&](int set, int buffer, uint32_t keys) {
        const uint64_t q_desc = smem_desc(smem_u32(q_s + set * q_bytes), 16, 1024), k_desc = smem_desc(keys, 16, 1024);
        if (elected()) {
          auto step = [&](int s) {      // 16 columns further: 32 bytes of a row of its box
            const int in_box = (s & 3) * 2;
            tc_mma(tmem + S_COL + BN * buffer, q_desc + (uint64_t)((s >> 2) * (Q_COL_BYTES >> 4) + in_box),
                   k_desc + (uint64_t)((s >> 2) * (COL_BYTES >> 4) + in_box), IDESC_S, s > 0 ? 1u : 0u);
          };
          if constexpr (STEPS > 0) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) step(s);
          } else {
            for (int s = 0; s < k.steps; ++s) step(s);
          }
          tc_commit(&s_full[buffer]);
        }
        __syncwarp();
      };
      auto add = [&](int set, int buffer, uint32_t values, bool onto) {
        const uint64_t v_desc = smem_desc(values, COL_BYTES, 1024);
        if (elected()) {
#pragma unroll
          for (int s = 0; s < BN / 16; ++s)      // 16 keys further: 2048 bytes of every box
            tc_mma_ts(tmem + 128 * set, tmem + S_COL + BN * buffer + 16 * s / 64 * 64 + 16 * s % 64 / 2, v_desc + (uint64_t)(s * (2048 >> 4)), idesc_pv, (onto || s > 0) ? 1u : 0u);
          tc_commit(&o_full[buffer]);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elected()) tc_commit(bar);
        __syncwarp();
      };
      for (;; ++it) {
        mbar_wait(&piece_full[it % PIECES], (it / PIECES) & 1, abort, k.status);
        const int n = stopped() ? 0 : pieces[it % PIECES].n;
        if (n == 0) break;
        mbar_wait(q_full, it & 1, abort, k.status);
        tc_fence_after();
        if constexpr (QT == 1) {
          auto ahead = [&](int j) {
            const int keys = next_unit();
            if (stopped()) return;
            tc_fence_after();
            scores(0, j % SETS, unit_at(keys));
            free_unit(keys);
            if (j == n - 1) commit(q_empty);
          };
          for (int j = 0; j < min(n, SETS) && !stopped(); ++j) ahead(j);
          for (int j = 0; j < n && !stopped(); ++j) {
            const int set = j % SETS;
            if (j == 0 && it > 0) mbar_wait(o_free, (it - 1) & 1, abort, k.status);      // the piece before has its sums in registers
            const int values = next_unit();
            mbar_wait(&p_full[set], done[set] & 1, abort, k.status);
            ++done[set];
            if (stopped()) break;
            tc_fence_after();
            add(set, set, unit_at(values), j >= SETS);
            free_unit(values);
            if (j + SETS < n) ahead(j + SETS);
          }
        } else {
          int keys = next_unit();
          if (stopped()) break;
          tc_fence_after();
          scores(0, 0, unit_at(keys));
          scores(1, 1, unit_at(keys));
          free_unit(keys);
          if (n == 1) commit(q_empty);
          for (int j = 0; j < n && !stopped(); ++j) {
            const int g = done[0] + j;
            if (j == 0 && it > 0) mbar_wait(o_free, (it - 1) & 1, abort, k.status);
            const int values = next_unit();
            mbar_wait(&p_full[0], g & 1, abort, k.status);
            if (stopped()) break;
            tc_fence_after();
            add(0, 0, unit_at(values), j > 0);
            if (j + 1 < n) {
              keys = next_unit();
              if (stopped()) break;
              tc_fence_after();
              scores(0, 0, unit_at(keys));
            }
            mbar_wait(&p_full[1], g & 1, abort, k.status);
            if (stopped()) break;
            tc_fence_after();
            add(1, 1, unit_at(values), j > 0);
            free_unit(values);
            if (j + 1 < n) {
              scores(1, 1, unit_at(keys));
              free_unit(keys);
              if (j + 2 == n) commit(q_empty);
            }
          }
        }
        if constexpr (QT == 2) done[0] += n;
      }
      commit(drained);      // nor does a product read it, or write tensor memory that goes back
      mbar_drain(drained, 0);
    }
  } else if (warp < SOFTMAX_WARPS) {
    // Warp w: set w / 4, tensor-memory lanes 32 (w % 4) .. + 31, a thread a row.
    const int quarter = warp & 3, set = warp >> 2, rows_set = QT == 2 ? set : 0, r = quarter * 32 + lane;
    const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16), o_addr = t_lane + 128 * set, s_addr = t_lane + S_COL + BN * set;
    auto sync_softmax = [&]() { asm volatile("bar.sync 9, %0;" ::"n"(32 * SOFTMAX_WARPS) : "memory"); };
    auto any_of_softmax = [&](bool x) {
      int any;
      asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, 9, %2, p;\n selp.b32 %0, 1, 0, q;\n}\n" : "=r"(any) : "r"((int)x), "n"(32 * SOFTMAX_WARPS) : "memory");
      return any != 0;
    };
    const float factor = a.softcap > 0.f ? 1.f : k.scale_log2;      // capped scores come in base 2
    int g = 0, it = 0, u0 = 0;      // g: tiles of the set
    for (;; ++it) {
      mbar_wait(&piece_full[it % PIECES], (it / PIECES) & 1, abort, k.status);
      if (any_of_softmax(*abort)) break;      // together: they meet at barriers below
      const Piece& p = pieces[it % PIECES];
      const int tiles = p.n;
      if (tiles == 0) break;
      const int rows = min(max(p.it.n - (p.first + rows_set * k.tokens), 0), k.tokens) * a.G;
      const bool valid = r < rows, busy = quarter * 32 < rows;      // this row exists; one of the warp's does
      const int token = min(p.it.row0 + p.first + rows_set * k.tokens + r / a.G, p.it.row0 + p.it.n - 1);
      const int* mask = a.mask + (size_t)token * a.words;
      const uint64_t near = (uint32_t)mask[0] | (a.words > 1 ? (uint64_t)(uint32_t)mask[1] << 32 : 0ull);
      const int begin = a.window > 0 ? window_begin(a, a.positions[token]) : 0;
      // keys that the mask may hide from some row: the new ones and what lies behind, with a window those that it has passed for the last token
      const int hidden_from = p.it.start, hidden_to = a.window > 0 ? p.it.start + p.it.n - a.window : 0;
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = KEYS ? set : 0; j < tiles; j += KEYS ? 2 : 1, ++g) {
        const bool first_of_set = j < (KEYS ? 2 : 1);      // of this piece's tiles; two sets of rows both begin with tile 0
        const int key0 = p.key + j * BN;
        const bool masked = key0 + BN > hidden_from || key0 < hidden_to;
        uint32_t bits[BN / 32];      // keys that the row sees
        if (masked && busy) {
#pragma unroll
          for (int i = 0; i < BN / 32; ++i) bits[i] = seen_bits(a, p.it, key0 + 32 * i, begin, mask, near);
        }
        mbar_wait(&s_full[set], g & 1, abort, k.status);
        tc_fence_after();
        if (masked) {      // values that are not finite are taken out before P V multiplies them with weights of zero
          // (behind the scores: the ring's earlier uses of this unit are over then, so the barrier's parity is this one's)
          const int u = u0 + value_unit(j, tiles), turn = u / k.ring, unit = u - turn * k.ring;
          mbar_wait(&u_full[unit], (uint32_t)(turn & 1), abort, k.status);
          unsigned char* v_s = ring_s + unit * unit_bytes;
          const __nv_bfloat162 nought = __floats2bfloat162_rn(0.f, 0.f);
          __nv_bfloat162 sum = nought;      // 0 x of all of them: a NaN where one is not finite
#pragma unroll 4
          for (int i = r; i < unit_bytes / 16; i += BM) {
            const uint4 x = *reinterpret_cast<const uint4*>(v_s + 16 * i);
            sum = __hfma2(reinterpret_cast<const __nv_bfloat162&>(x.x), nought, sum);
            sum = __hfma2(reinterpret_cast<const __nv_bfloat162&>(x.y), nought, sum);
            sum = __hfma2(reinterpret_cast<const __nv_bfloat162&>(x.z), nought, sum);
            sum = __hfma2(reinterpret_cast<const __nv_bfloat162&>(x.w), nought, sum);
          }
          if (__low2float(sum) != 0.f || __high2float(sum) != 0.f) {
            spoiled[it & 1] = it + 1;      // (first: two sets of rows on the same tile may find the other's zeros instead)
            __threadfence_block();
            for (int i = r; i < unit_bytes / 16; i += BM) {
              uint4 x = *reinterpret_cast<const uint4*>(v_s + 16 * i);
              uint32_t* w4 = &x.x;
#pragma unroll
              for (int e = 0; e < 4; ++e) w4[e] &= ~__vcmpeq2(w4[e] & 0x7f807f80u, 0x7f807f80u);
              *reinterpret_cast<uint4*>(v_s + 16 * i) = x;
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          asm volatile("bar.sync %0, %1;" ::"r"(1 + set), "n"(BM) : "memory");
        }
        if (busy) {
          // The first scores, the last ones - which stay in registers -, and once the maximum is known the first again: one piece of code three times, for
          // what runs a few times a block is bound by fetching its instructions.
          constexpr int CHUNKS = BN / N;
          float v[N], mx = -INFINITY, m_use = 0.f, part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (int step = 0; step < 2 * CHUNKS - 1; ++step) {
            const int col = step == 1 ? N : 0;
            tmem_ld(v, s_addr + col);
            if (a.softcap > 0.f) {      // cap tanh(x / cap) in base 2, as cap (1 - 2 / (1 + e^(2 x / cap))): 0 is taken off where the sum is infinite
#pragma unroll
              for (int e = 0; e < N; ++e) v[e] = k.cap_log2 - __fdividef(2.f * k.cap_log2, 1.f + mi::ex2_fast(v[e] * k.cap_scale));
            }
            if (masked) {      // -infinity where the row may not see the key
              const uint32_t b0 = step == 1 ? bits[BN / 32 - 2] : bits[0], b1 = step == 1 ? bits[BN / 32 - 1] : bits[1];
#pragma unroll
              for (int e = 0; e < N; ++e) v[e] = ((e < 32 ? b0 : b1) >> (e & 31)) & 1 ? v[e] : -INFINITY;
            }
            if (step < CHUNKS) {
              float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int e = 0; e < N; e += 2) mx4[e >> 1 & 3] = mi::max_of(mx4[e >> 1 & 3], v[e], v[e + 1]);
              mx = fmaxf(mx, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
            }
            if (step < CHUNKS - 1) continue;
            if (step == CHUNKS - 1) {
              const float m_new = fmaxf(m_run, mx * factor);      // the scale is positive
              const bool move = m_new > m_run + 8.f;      // (of the first key: from -infinity)
              if (__any_sync(0xffffffffu, move)) {
                const float alpha = move ? exp2f(m_run - m_new) : 1.f;
                if (!first_of_set) {      // (its last P V is done: this tile's scores came behind it)
#pragma unroll 1
                  for (int c = 0; 16 * c < k.n_out; ++c) {      // (16 at a time: the scores are in registers too)
                    float o[16];
                    uint32_t x[16];
                    tmem_ld(o, o_addr + 16 * c);
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                      mi::mul_pair(o[e], o[e + 1], o[e], o[e + 1], alpha);
                      x[e] = __float_as_uint(o[e]);
                      x[e + 1] = __float_as_uint(o[e + 1]);
                    }
                    tmem_st(o_addr + 16 * c, x);
                  }
                }
                l_run *= alpha;
                if (move) m_run = m_new;
              }
              m_use = m_run == -INFINITY ? 0.f : m_run;
            }
            uint32_t packed[N / 2];
#pragma unroll
            for (int e = 0; e < N; e += 2) mi::fma_pair(v[e], v[e + 1], v[e], v[e + 1], factor, -m_use);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
              packed[e] = pack_bf16(mi::ex2_fast(v[2 * e]), mi::ex2_fast(v[2 * e + 1]));      // nothing where the row may not see the key
              mi::add_pair(part[2 * e & 3], part[(2 * e + 1) & 3], __uint_as_float(packed[e] << 16), __uint_as_float(packed[e] & 0xffff0000u));
            }
            tmem_st(s_addr + col, packed);      // two keys to a column, over the first half of their scores
          }
          l_run += (part[0] + part[1]) + (part[2] + part[3]);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[set]);
      }
      const bool whole = p.slot < 0, mine = !KEYS || set < tiles;      // (a piece of one tile has no second stream)
      if (mine) {
        mbar_wait(&o_full[set], (g - 1) & 1, abort, k.status);
        tc_fence_after();
      }
      float m_all = m_run, l_all = l_run, scale0 = 1.f, scale1 = 0.f;
      if constexpr (KEYS) {      // the two streams' sums of this row
        of_set[set * BM + r] = make_float2(m_run, l_run);
        tc_fence_before();
        sync_softmax();
        tc_fence_after();
        const float2 x0 = of_set[r], x1 = of_set[BM + r];
        m_all = fmaxf(x0.x, x1.x);
        const float off = m_all == -INFINITY ? 0.f : m_all;
        scale0 = exp2f(x0.x - off);
        scale1 = exp2f(x1.x - off);
        l_all = x0.y * scale0 + x1.y * scale1;
      }
      const bool fix = spoiled[it & 1] == it + 1;
      const int h = p.head * a.G + r % a.G;
      if (whole) {
        const float sink2 = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
        const float top = fmaxf(m_all, sink2), off = top == -INFINITY ? 0.f : top, weight = exp2f(m_all - off);
        const float total = l_all * weight + exp2f(sink2 - off), mult = total == 0.f ? 0.f : weight / total;      // nothing visible: zeros
        scale0 *= mult;
        scale1 *= mult;
      }
      const int key_end = min(p.it.ctx, p.key + tiles * BN);
      if (busy) {
#pragma unroll 1
        for (int c = KEYS ? set : 0; 32 * c < k.n_out; c += KEYS ? 2 : 1) {
          float o[32];
          tmem_ld(o, (KEYS ? t_lane : o_addr) + 32 * c);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= scale0;
          if (KEYS && tiles > 1) {
            float o1[32];
            tmem_ld(o1, t_lane + 128 + 32 * c);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fmaf(o1[e], scale1, o[e]);
          }
          if (valid && !*abort) {
            if (fix) {
              float more[32] = {};
              add_not_finite(a, p.it, p.head, p.key, key_end, begin, mask, near, 32 * c, more);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] += more[e];
            }
            if (whole) {
              __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)token * a.nh * a.hd + (size_t)h * a.hd + 32 * c;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (32 * c + 8 * q < a.hd)      // (a head size is a multiple of 16)
                  *reinterpret_cast<uint4*>(dst + 8 * q) = make_uint4(pack_bf16(o[8 * q], o[8 * q + 1]), pack_bf16(o[8 * q + 2], o[8 * q + 3]),
                                                                      pack_bf16(o[8 * q + 4], o[8 * q + 5]), pack_bf16(o[8 * q + 6], o[8 * q + 7]));
            } else {      // four columns of all rows, then the next four: what a warp's lanes write lies side by side
              float4* dst = reinterpret_cast<float4*>(a.part_o) + ((size_t)p.slot * (k.n_out / 4) + 8 * c) * (QT * BM) + rows_set * BM + r;
#pragma unroll
              for (int q = 0; q < 8; ++q) dst[q * (QT * BM)] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
            }
          }
          __syncwarp();
        }
        if (!whole && valid && (!KEYS || set == 0) && !*abort) reinterpret_cast<float2*>(a.part_ml)[(size_t)p.slot * (QT * BM) + rows_set * BM + r] = make_float2(m_all, l_all);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      if (KEYS && !whole && k.counters) {      // few rows: the unit's last piece to come joins them all, a launch less
        __threadfence();
        sync_softmax();
        if (threadIdx.x == 0) {
          const bool all = atomicAdd(k.counters + p.unit, 1) == p.pieces - 1;
          if (all) k.counters[p.unit] = 0;      // ready for the next launch
          *last_to_come = all;
        }
        sync_softmax();
        if (*last_to_come) {
          __threadfence();
          const int4 u = make_int4(p.pieces, p.it.row0 + p.first, min(p.it.n - p.first, k.tokens), p.head);
          const int quarters = (min(k.tokens, u.z) * a.G + 31) / 32;      // a warp 32 rows and 8 columns at a time
#pragma unroll 1
          for (int w = warp; w < quarters * (k.n_out / 8); w += SOFTMAX_WARPS) join_row<1, 2, 8>(k, p.block, u, 0, w % quarters * 32 + lane, w / quarters * 2);
        }
      }
      u0 = (u0 + 2 * tiles) % (2 * k.ring);      // (as far as slot and parity go)
    }
  }
  // every tensor-memory access is done, then the columns go back
  tc_fence_before();
  __syncthreads();
  if (*abort) give_up<QT>(k);
  if (warp == MMA_WARP) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM_COLS) : "memory");
  }
}

// The pieces of units that several blocks shared, where the last block to come does not join them: for the unit that begins in a block and goes on in others,
// grid (blocks, QT, columns / (4 F JOIN_WARPS / 4)); a lane a row and 4 F columns, a warp 32 rows, AT_ONCE pieces on their way at a time.
constexpr int JOIN_WARPS = 8;
template <int QT, int F, int AT_ONCE>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
tree_join_kernel(const Tc k) {
  const int warp = threadIdx.x >> 5;
  mi::grid_dependency_sync();
  const int4 u = k.joins[blockIdx.x];
  if (u.x) join_row<QT, F, AT_ONCE>(k, blockIdx.x, u, blockIdx.y, warp % 4 * 32 + (threadIdx.x & 31), (blockIdx.z * (JOIN_WARPS / 4) + warp / 4) * F);
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

constexpr int NOT_TAKEN = 2, JOINED = 3;      // answers beside 0 and 1: another kernel's sizes; two launches, the second of which joins the pieces

template <int QT, int SETS, int BN, int STEPS>
int launch(Tc& k, const CUtensorMap& q_map, const CUtensorMap& kv_map, int blocks, cudaStream_t stream) {
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return mi_fail("attention_tree_tc: no current device");
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(tree_tc_kernel<QT, SETS, BN, STEPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess)
      return mi_fail("attention_tree_tc: %d bytes of shared memory were refused", SMEM_BYTES);
    ready[dev] = true;
  }
  k.ring = (SMEM_BYTES - BARS * 8 - (QT == 1 ? 2 * BM * 8 : 0) - QT * k.boxes * BM * 128) / (k.boxes * BN * 128);
  if (k.ring > MAX_UNITS) k.ring = MAX_UNITS;
  MI_REQUIRE(k.ring >= 4, "attention_tree_tc: no room for a ring of tiles of %d boxes", k.boxes);
  if (mi::launch(tree_tc_kernel<QT, SETS, BN, STEPS>, dim3(blocks), dim3(threads_of(SETS)), SMEM_BYTES, stream, q_map, kv_map, k) != cudaSuccess)
    return mi_fail("attention_tree_tc: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  if (k.counters) {
    MI_LAUNCH_OK("attention_tree_tc");
    return 0;
  }
  // Many pieces of a unit where there are fewer units than blocks: eight at a time of 8 columns; else two at a time of 32.
  const Args& a = k.a;
  const bool few = (long long)a.items * a.nkv * k.max_parts < blocks;
  const int f = few ? 2 : 8, columns = (k.n_out / 4 + f * (JOIN_WARPS / 4) - 1) / (f * (JOIN_WARPS / 4));
  auto join = few ? tree_join_kernel<QT, 2, 8> : tree_join_kernel<QT, 8, 2>;
  if (mi::launch(join, dim3(blocks, QT, columns), dim3(32 * JOIN_WARPS), 0, stream, k) != cudaSuccess)
    return mi_fail("attention_tree_tc: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  MI_LAUNCH_OK("attention_tree_tc");
  return JOINED;
}

// A unit's last block to come joins its pieces where that is a moment's work for one block: 32 rows, of heads that leave it both sets of softmax
// warps, and so many bytes.  On the device, inside and by a kernel of its own (which takes a launch, 5 us of the host's time, more): 8 requests, groups of 4,
// 4 pieces of 16, 32, 48, 96 rows of 128 columns 23.9, 23.7, 25.9, 29.2 and 23.9, 24.0, 24.6, 25.5 us; one request, groups of 2, 20 pieces of 8, 16, 32, 64
// rows (80 KB to 640) 16.2, 16.6, 17.5, 23.9 and 16.4 to 16.7, of 64 columns 12.7, 13.0, 13.5, 16.9 and 15.0 to 15.4, of 256 columns 43 and 24.7.
constexpr int JOIN_INSIDE_ROWS = 32;
constexpr long long JOIN_INSIDE_BYTES = 192 << 10;

// Sets of 128 rows that a block takes at a time: two once the largest item has more rows than one holds, as far as tensor memory goes.
int sets_of(int max_q, int G, int hd) { return hd <= 128 && max_q > BM / G ? 2 : 1; }

}  // namespace

// Floats of scratch - what is to be joined, the sums -, 0 for sizes that the kernel does not take.
MI_API long long mi_attention_tree_tc_floats(int nh, int nkv, int hd, int page_size, int max_q) {
  if (!(nkv > 0 && nh > 0 && nh % nkv == 0 && nh / nkv <= BM && hd % 16 == 0 && hd >= 64 && hd <= 256 && page_size > 0 && page_size % 16 == 0 && max_q > 0)) return 0;
  const long long blocks = mi::sm_count();
  return 4 * blocks + 2 * blocks * sets_of(max_q, nh / nkv, hd) * BM * ((hd + BOX - 1) / BOX * BOX + 2);
}

// bfloat16.  scratch: mi_attention_tree_tc_floats floats, 16-byte aligned; counters: a zero word for each item, key/value head and set of
// 128 / G tokens of max_q, left zero; status: one word, which gets STATUS_LATE or
// STATUS_PLACE.  Answers NOT_TAKEN for sizes or addresses that it does not take, JOINED if it has launched two kernels instead of one.
MI_API int mi_attention_tree_tc(void* out, const void* qkv, const void* kv, const int* block_table, int bt_stride, const int* q_start, const int* q_len,
                                const int* ctx_len, const int* seq_slot, const int* mask, int words, const int* positions, const float* sink, float* scratch,
                                int* counters, int* status, int items, int T, int width, int nh, int nkv, int hd, int pages, int page_size, int window, int max_q, float scale,
                                float softcap, cudaStream_t stream) {
  MI_REQUIRE(items >= 0 && T >= 0 && nkv > 0 && nh % nkv == 0 && bt_stride > 0 && pages > 0 && (long long)words * 32 >= max_q, "attention_tree_tc: bad sizes items=%d T=%d words=%d max_q=%d", items, T, words, max_q);
  if (mi_attention_tree_tc_floats(nh, nkv, hd, page_size, max_q) == 0 || width % 8 != 0 || !(scale > 0.f) || T == 0 ||
      ((uintptr_t)out | (uintptr_t)qkv | (uintptr_t)kv | (uintptr_t)scratch) % 16 != 0 || (long long)pages * 2 * nkv * page_size > 0x7fffffffll ||
      ((long long)bt_stride * page_size / 64 + 2 + OVERHEAD) * items * nkv * (max_q / (BM / (nh / nkv)) + 1) > 0x7fffffffll)      // the last: the line of tiles
    return NOT_TAKEN;
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
  k.cap_log2 = softcap * 1.4426950408889634f;
  k.cap_scale = softcap > 0.f ? 2.f * k.scale_log2 / softcap : 0.f;
  const int blocks = mi::sm_count();
  // Pieces are joined by the unit's last block to come, a launch less, where that is little for one block to do; else by a kernel of their own.
  const long long units = (long long)items * nkv * k.max_parts, rows = (long long)max_q * G, pieces = blocks / units + 2;
  k.counters = hd <= 128 && rows <= JOIN_INSIDE_ROWS && pieces * rows * hd * 4 <= JOIN_INSIDE_BYTES ? counters : nullptr;
  k.joins = (int4*)scratch;
  float* part_o = scratch + 4ll * blocks;
  float* part_ml = part_o + 2ll * blocks * qt * BM * k.n_out;
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
  // heads of 64, 128 and 256 with the products' steps written out
  if (qt == 2) {
    if (hd == 128) return launch<2, 2, 128, 8>(k, q_map, kv_map, blocks, stream);
    return hd == 64 ? launch<2, 2, 128, 4>(k, q_map, kv_map, blocks, stream) : launch<2, 2, 128, 0>(k, q_map, kv_map, blocks, stream);
  }
  if (hd == 128) return launch<1, 2, 128, 8>(k, q_map, kv_map, blocks, stream);
  if (hd < 128) return hd == 64 ? launch<1, 2, 128, 4>(k, q_map, kv_map, blocks, stream) : launch<1, 2, 128, 0>(k, q_map, kv_map, blocks, stream);
  return hd == 256 ? launch<1, 1, 64, 16>(k, q_map, kv_map, blocks, stream) : launch<1, 1, 64, 0>(k, q_map, kv_map, blocks, stream);
}
