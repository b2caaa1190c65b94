// Attention of a tree of new tokens over the paged cache, for any head size up to 640, any page size, float32 or bf16 storage, float32
// arithmetic: the 32-bit path, and what the tensor-core kernel (attention_tree_tc.cu) does not take.  attention_tree.cuh says which keys a row
// sees.
//
// A block has up to 32 query rows of one (item, key/value head) and a piece of the item's keys, walked in tiles of BK: an online softmax in base 2,
// scores and weighted values by FMAs from shared memory, four rows a warp and BK / 32 keys (then values) a lane, so a value read from shared
// memory serves four products.  The rows of a head group lie side by side: a key is fetched once for all of them.  With 16 rows or fewer a
// tile's keys are dealt out to several warps a row group, each with an online softmax of its own, put together at the end of the piece.  Pieces give
// a small step enough blocks; more than one of them leave sums that tree_merge_kernel puts together.
//
// How many pieces there are follows from the step's items, longest context and the SMs, how many warps share a row from the largest item: unlike
// attention_f32.cu, whose segments are fixed, the last bits of a row may differ with what else is in the batch, within the bound that the tests derive.
//
// A key that a row does not see has the weight -1, which the weighted values leave out: a zero would make a NaN of an infinity there.
//
// What bounds it: shared memory, whose 16 bytes of a key or value serve four rows - 16 FMAs a lane to five wavefronts and more, where the FMAs take four
// cycles -, and with few rows the fetching of tiles, of which a block has one on its way.  Measured in float32: 3 trees of 13 over about 1000 keys, 16 heads on
// 8, 22 us (the bytes 2.2); 8 single tokens over 4000 keys 82 us, 49 % of the bytes' rate (135 with all of a row's keys in one warp); 8 trees of 8 over 2000
// keys 81 us, the FMAs 15.  In bf16, with pages of 24 that the tensor-core kernel leaves to this one, 8 trees of 32 over up to 4096 keys, 32 heads on 8, 441 us.
#include "attention_tree.cuh"

namespace {

using namespace mi_tree;

// RG groups of four rows, KS warps a group.
constexpr int threads_of(int RG, int KS) { return 32 * RG * KS; }

template <typename T>
__device__ __forceinline__ void load_row4(float4& v, const T* p, int left, bool wide) {      // four values, zeros past the row
  if (wide) {
    if constexpr (sizeof(T) == 4) {
      v = *reinterpret_cast<const float4*>(p);
    } else {
      const uint2 raw = *reinterpret_cast<const uint2*>(p);
      v = make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xffff0000u));
    }
  } else {
    v = make_float4(mi::to_float(p[0]), left > 1 ? mi::to_float(p[1]) : 0.f, left > 2 ? mi::to_float(p[2]) : 0.f, left > 3 ? mi::to_float(p[3]) : 0.f);
  }
}

// grid: (pieces, row tiles * nkv, items)
template <typename T, int RG, int KS, int BK, int HD>
__global__ void __launch_bounds__(threads_of(RG, KS))
tree_kernel(Args a, int chunk, int pieces, int wide) {
  constexpr int THREADS = threads_of(RG, KS), TX = 32, BR = 4 * RG, COLS = HD / (4 * TX);
  constexpr int OWN = BK / KS;                              // keys of a tile that a warp has
  constexpr int L = OWN < TX ? TX / OWN : 1, KEYS = OWN < TX ? 1 : OWN / TX;      // lanes that share a key's columns; keys of a lane
  static_assert(BK % KS == 0 && OWN * L == TX * KEYS && L <= 4 && HD % (4 * TX) == 0, "a row's keys of a tile are a warp's lanes'");
  extern __shared__ __align__(16) float smem[];
  const int hd4 = (a.hd + 3) / 4, stride = 4 * hd4 + 4;      // a row in shared memory, 16 bytes on for the banks
  float *q_s = smem, *k_s = q_s + BR * stride, *v_s = k_s + BK * stride, *p_s = v_s + BK * stride;      // [BR, stride], [BK, stride] twice, [BR, BK + 4]
  constexpr int PS = BK + 4;
  __shared__ const T* rows_of[2][BK];      // of this tile's keys and of the next one's: where in the cache the key lies; the values so much further on
  const size_t to_values = (size_t)a.nkv * a.page_size * a.hd;
  const int piece = blockIdx.x, head = blockIdx.y % a.nkv, r0 = blockIdx.y / a.nkv * BR;
  mi::grid_dependency_sync();
  const Item it = item_of(a, blockIdx.z);
  const int rows = it.n * a.G;
  if (r0 >= rows) return;
  const int key_end = piece == pieces - 1 ? it.ctx : min(it.ctx, (piece + 1) * chunk);
  const int key_begin = max(piece * chunk, window_begin(a, it.start));      // (no new token's position is below the context's length)
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX % RG, split = threadIdx.x / TX / RG, own = split * OWN;
  const int kx = tx % (TX / L), dx = tx / (TX / L);      // of the warp's keys; of the columns
  const bool busy = r0 + 4 * ty < rows;      // one of the warp's rows exists; the other warps fetch only
  const T* qkv = reinterpret_cast<const T*>(a.qkv);
  const T* kv = reinterpret_cast<const T*>(a.kv);

  for (int i = threadIdx.x; i < BR * hd4; i += THREADS) {
    const int r = i / hd4, d = 4 * (i - r * hd4), row = r0 + r;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < rows) load_row4(v, qkv + (size_t)(it.row0 + row / a.G) * a.width + (size_t)(head * a.G + row % a.G) * a.hd + d, a.hd - d, wide);
    *reinterpret_cast<float4*>(q_s + r * stride + d) = v;
  }
  // of this thread's four rows: the token's mask, and where its window begins
  const int* mask[4];
  int token[4], begin[4], pos[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    token[i] = min(r0 + 4 * ty + i, rows - 1) / a.G;
    mask[i] = a.mask + (size_t)(it.row0 + token[i]) * a.words;
    pos[i] = a.window > 0 ? a.positions[it.row0 + token[i]] : 0;
    begin[i] = window_begin(a, pos[i]);
  }
  float m[4], l[4], acc[4][COLS][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < COLS; ++c) acc[i][c][0] = acc[i][c][1] = acc[i][c][2] = acc[i][c][3] = 0.f;
  }
  auto find_rows = [&](int key0, int buffer) {
    for (int k = threadIdx.x; k < BK; k += THREADS) {
      const int key = key0 + k;
      rows_of[buffer][k] = key < key_end ? kv + (((size_t)page_of(a, it, key) * 2 * a.nkv + head) * a.page_size + key % a.page_size) * a.hd : nullptr;
    }
  };
  // A tile's keys or values on their way (float32 by asynchronous copies, where a row is whole 16 bytes); zeros past the piece.
  auto load_tile = [&](float* to, int buffer, size_t further) {
#pragma unroll 4
    for (int i = threadIdx.x; i < BK * hd4; i += THREADS) {
      const int k = i / hd4, d = 4 * (i - k * hd4);
      const T* from = rows_of[buffer][k];
      float* dst = to + k * stride + d;
      if (sizeof(T) == 4 && wide) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(from ? from + further + d : kv), "r"(from ? 16 : 0) : "memory");
      } else {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (from) load_row4(v, from + further + d, a.hd - d, wide);
        *reinterpret_cast<float4*>(dst) = v;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the keys of a tile are on their way while the values of the tile before are worked on, its values while its scores are made
  find_rows(key_begin, 0);
  __syncthreads();
  load_tile(k_s, 0, 0);
  load_tile(v_s, 0, to_values);
  int buffer = 0;
  for (int key0 = key_begin; key0 < key_end; key0 += BK, buffer ^= 1) {
    const bool more = key0 + BK < key_end;
    if (more) find_rows(key0 + BK, buffer ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");      // the keys are there
    __syncthreads();
    if (busy) {
      float s[4][KEYS];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < KEYS; ++j) s[i][j] = 0.f;
#pragma unroll 2
      for (int d = 4 * dx; d < 4 * hd4; d += 4 * L) {
        float4 q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(q_s + (4 * ty + i) * stride + d);
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
          const float4 k = *reinterpret_cast<const float4*>(k_s + (own + kx + TX * j) * stride + d);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[i][j] = fmaf(q[i].w, k.w, fmaf(q[i].z, k.z, fmaf(q[i].y, k.y, fmaf(q[i].x, k.x, s[i][j]))));
        }
      }
#pragma unroll
      for (int o = TX / L; o < TX; o <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < KEYS; ++j) s[i][j] += __shfl_xor_sync(0xffffffffu, s[i][j], o);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float top = -INFINITY;
        bool see[KEYS];
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
          const int key = key0 + own + kx + TX * j, node = key - it.start;
          see[j] = key < key_end;
          if (node < 0) {
            see[j] = see[j] && key >= begin[i];
          } else if (see[j]) {
            see[j] = (mask[i][node >> 5] >> (node & 31)) & 1;
            if (a.window > 0) see[j] = see[j] && a.positions[it.row0 + node] >= begin[i];
          }
          s[i][j] = logit2_exact(s[i][j], a.scale, a.softcap);
          if (see[j]) top = fmaxf(top, s[i][j]);
        }
#pragma unroll
        for (int o = TX / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float next = fmaxf(m[i], top), off = next == -INFINITY ? 0.f : next, alpha = exp2f(m[i] - off);
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < KEYS; ++j) {
          const float p = exp2f(s[i][j] - off);
          if (see[j] && dx == 0) part += p;
          if (dx == 0) p_s[(4 * ty + i) * PS + own + kx + TX * j] = see[j] ? p : -1.f;
        }
        m[i] = next;
        l[i] = l[i] * alpha + part;      // (this thread's keys; the row's threads are added up at the end)
#pragma unroll
        for (int c = 0; c < COLS; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][c][e] *= alpha;
      }
    }
    __syncthreads();      // (scores made, weights written)
    if (more) {
      load_tile(k_s, buffer ^ 1, 0);
      asm volatile("cp.async.wait_group 1;" ::: "memory");      // the values are there
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const bool all = key0 + BK <= min(it.start, key_end) && a.window <= 0;      // every row sees every key of the tile
    const int near = busy ? min(own + OWN, key_end - key0) : 0;
    for (int k0 = own; k0 < near; k0 += 4) {      // (past `near` all weights are -1)
      float4 p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(p_s + (4 * ty + i) * PS + k0);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          const int d = 4 * (tx + TX * c);
          if (d < 4 * hd4) {
            const float4 v = *reinterpret_cast<const float4*>(v_s + (k0 + k) * stride + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float w = k == 0 ? p[i].x : k == 1 ? p[i].y : k == 2 ? p[i].z : p[i].w;
              if (all || !(w < 0.f)) {
                acc[i][c][0] = fmaf(w, v.x, acc[i][c][0]);
                acc[i][c][1] = fmaf(w, v.y, acc[i][c][1]);
                acc[i][c][2] = fmaf(w, v.z, acc[i][c][2]);
                acc[i][c][3] = fmaf(w, v.w, acc[i][c][3]);
              }
            }
          }
        }
    }
    if (more) {
      __syncthreads();
      load_tile(v_s, buffer ^ 1, to_values);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int o = TX / 2; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
  if constexpr (KS > 1) {      // the row group's warps put together: warp `split` the rows split, split + KS, ..
    float* acc_s = k_s;                                     // [KS, BR, stride], over the tiles
    float2* ml_s = reinterpret_cast<float2*>(p_s);          // [KS, BR]
    static_assert(KS * BR <= 2 * BK && 2 * KS <= PS, "the sums lie where the tiles were");
    asm volatile("cp.async.wait_all;" ::: "memory");        // (those of a piece without keys)
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = split * BR + 4 * ty + i;
      if (tx == 0) ml_s[at] = make_float2(m[i], l[i]);
#pragma unroll
      for (int c = 0; c < COLS; ++c)
        if (4 * (tx + TX * c) < 4 * hd4) *reinterpret_cast<float4*>(acc_s + at * stride + 4 * (tx + TX * c)) = make_float4(acc[i][c][0], acc[i][c][1], acc[i][c][2], acc[i][c][3]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i % KS != split) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < KS; ++w) top = fmaxf(top, ml_s[w * BR + 4 * ty + i].x);
      const float off = top == -INFINITY ? 0.f : top;
      m[i] = top;
      l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < COLS; ++c) acc[i][c][0] = acc[i][c][1] = acc[i][c][2] = acc[i][c][3] = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        const int at = w * BR + 4 * ty + i;
        const float2 x = ml_s[at];
        const float weight = exp2f(x.x - off);
        l[i] = fmaf(x.y, weight, l[i]);
#pragma unroll
        for (int c = 0; c < COLS; ++c)
          if (4 * (tx + TX * c) < 4 * hd4) {
            const float4 v = *reinterpret_cast<const float4*>(acc_s + at * stride + 4 * (tx + TX * c));
            acc[i][c][0] = fmaf(v.x, weight, acc[i][c][0]);
            acc[i][c][1] = fmaf(v.y, weight, acc[i][c][1]);
            acc[i][c][2] = fmaf(v.z, weight, acc[i][c][2]);
            acc[i][c][3] = fmaf(v.w, weight, acc[i][c][3]);
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + 4 * ty + i;
    if (row >= rows || i % KS != split) continue;
    const int h = head * a.G + row % a.G;
    const size_t at = (size_t)(it.row0 + token[i]) * a.nh + h;
    if (pieces > 1) {
      const size_t slot = at * pieces + piece;
      if (tx == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * slot) = make_float2(m[i], l[i]);
#pragma unroll
      for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * (tx + TX * c) + e < a.hd) a.part_o[slot * a.hd + 4 * (tx + TX * c) + e] = acc[i][c][e];
      continue;
    }
    const float sink2 = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
    const float top = fmaxf(m[i], sink2), off = top == -INFINITY ? 0.f : top, weight = exp2f(m[i] - off);
    const float total = l[i] * weight + exp2f(sink2 - off), factor = total == 0.f ? 0.f : weight / total;      // nothing visible: zeros
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * (tx + TX * c) + e < a.hd) reinterpret_cast<T*>(a.out)[at * a.hd + 4 * (tx + TX * c) + e] = mi::from_float<T>(acc[i][c][e] * factor);
  }
}

// The pieces of a row added up, a warp per (token, head): grid (T, ceil(nh / 4)).  Rows that belong to no item are left as they were.
template <typename T>
__global__ void __launch_bounds__(128)
tree_merge_kernel(Args a, int chunk, int pieces) {
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, t = blockIdx.x;
  mi::grid_dependency_sync();
  if (h >= a.nh) return;
  int ctx = -1;
  for (int b = lane; b < a.items; b += 32) {
    const Item it = item_of(a, b);
    if (t >= it.row0 && t < it.row0 + it.n) ctx = it.ctx;
  }
  ctx = __reduce_max_sync(0xffffffffu, ctx);
  if (ctx < 0) return;
  const int n = min((ctx + chunk - 1) / chunk, pieces);
  const size_t at = (size_t)t * a.nh + h;
  const float sink2 = a.sink ? a.sink[h] * 1.4426950408889634f : -INFINITY;
  constexpr int AT_ONCE = 8, COLS = 4;      // pieces and 32s of columns that are on their way at a time
  for (int d0 = lane; d0 < a.hd; d0 += 32 * COLS) {
    float top = sink2, total = a.sink ? 1.f : 0.f, sum[COLS] = {};
    for (int s0 = 0; s0 < n; s0 += AT_ONCE) {
      float2 ml[AT_ONCE];
      float x[AT_ONCE][COLS];
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) {
        const bool there = s0 + s < n;
        ml[s] = there ? *reinterpret_cast<const float2*>(a.part_ml + 2 * (at * pieces + s0 + s)) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int c = 0; c < COLS; ++c) x[s][c] = there && d0 + 32 * c < a.hd ? a.part_o[(at * pieces + s0 + s) * a.hd + d0 + 32 * c] : 0.f;
      }
      float next = top;
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) next = fmaxf(next, ml[s].x);
      const float off = next == -INFINITY ? 0.f : next, alpha = exp2f(top - off);
      top = next;
      total *= alpha;
#pragma unroll
      for (int c = 0; c < COLS; ++c) sum[c] *= alpha;
#pragma unroll
      for (int s = 0; s < AT_ONCE; ++s) {
        const float w = exp2f(ml[s].x - off);
        total = fmaf(ml[s].y, w, total);
#pragma unroll
        for (int c = 0; c < COLS; ++c) sum[c] = fmaf(x[s][c], w, sum[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < COLS; ++c)
      if (d0 + 32 * c < a.hd) reinterpret_cast<T*>(a.out)[at * a.hd + d0 + 32 * c] = mi::from_float<T>(total == 0.f ? 0.f : sum[c] / total);
  }
}

template <typename T, int RG, int KS, int BK, int HD>
int launch(const Args& a, int chunk, int pieces, bool wide, cudaStream_t stream) {
  constexpr int BR = 4 * RG;
  const int stride = (a.hd + 3) / 4 * 4 + 4;
  const size_t smem = ((size_t)(BR + 2 * BK) * stride + BR * (BK + 4)) * sizeof(float);
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return mi_fail("attention_tree: no current device");
  if (!ready[dev]) {
    const size_t most = ((size_t)(BR + 2 * BK) * (HD + 4) + BR * (BK + 4)) * sizeof(float);
    if (cudaFuncSetAttribute(tree_kernel<T, RG, KS, BK, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess)
      return mi_fail("attention_tree: %zu bytes of shared memory were refused", most);
    ready[dev] = true;
  }
  const int tiles = (a.max_q * a.G + BR - 1) / BR;
  MI_REQUIRE((long long)tiles * a.nkv <= 65535, "attention_tree: %d rows of %d heads are too many for one launch", a.max_q * a.G, a.nkv);
  if (mi::launch(tree_kernel<T, RG, KS, BK, HD>, dim3(pieces, tiles * a.nkv, a.items), dim3(threads_of(RG, KS)), smem, stream, a, chunk, pieces, (int)wide) != cudaSuccess)
    return mi_fail("attention_tree: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  if (pieces > 1 && mi::launch(tree_merge_kernel<T>, dim3(a.T, (a.nh + 3) / 4), dim3(128), 0, stream, a, chunk, pieces) != cudaSuccess)
    return mi_fail("attention_tree: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  MI_LAUNCH_OK("attention_tree");
  return 0;
}

// All eight warps have a row group each, or with few rows several of them share a group's keys (three rows, heads of 256: 98 us instead of 181; 16 rows, heads of
// 128: 81 instead of 90).
template <typename T, int HD>
int launch_rows(const Args& a, int chunk, int pieces, bool wide, cudaStream_t stream) {
  const int rows = a.max_q * a.G;
  if (rows <= 4) return launch<T, 1, 8, 64, HD>(a, chunk, pieces, wide, stream);
  if (rows <= 8) return launch<T, 2, 4, 64, HD>(a, chunk, pieces, wide, stream);
  if (rows <= 16) return launch<T, 4, 2, 64, HD>(a, chunk, pieces, wide, stream);
  return launch<T, 8, 1, 64, HD>(a, chunk, pieces, wide, stream);
}
template <typename T>
int launch_sized(const Args& a, int chunk, int pieces, bool wide, cudaStream_t stream) {
  if (a.hd <= 128) return launch_rows<T, 128>(a, chunk, pieces, wide, stream);
  if (a.hd <= 256) return launch_rows<T, 256>(a, chunk, pieces, wide, stream);
  return launch<T, 4, 1, 32, 640>(a, chunk, pieces, wide, stream);
}

}  // namespace

// Every item with up to max_q new tokens.  chunk: keys of a piece; pieces: of an item, whose last one takes all
// keys that are left.
// scratch: T * nh * pieces * (hd + 2) floats, 8-byte aligned; unused with one piece.
MI_API int mi_attention_tree(void* out, const void* qkv, int dtype, const void* kv, const int* block_table, int bt_stride, const int* q_start,
                             const int* q_len, const int* ctx_len, const int* seq_slot, const int* mask, int words, const int* positions,
                             const float* sink, float* scratch, int items, int T, int width, int nh, int nkv, int hd, int pages, int page_size,
                             int window, int max_q, float scale, float softcap, int chunk, int pieces, cudaStream_t stream) {
  MI_REQUIRE(items >= 0 && items <= 65535 && T >= 0 && nh > 0 && nkv > 0 && nh % nkv == 0 && hd > 0 && hd <= 640 && pages > 0 && page_size > 0 && bt_stride > 0,
             "attention_tree: bad sizes items=%d T=%d heads=%d/%d hd=%d pages=%d of %d", items, T, nh, nkv, hd, pages, page_size);
  MI_REQUIRE(max_q >= 0 && (long long)words * 32 >= max_q && chunk > 0 && pieces > 0 && pieces <= 65535 && (long long)max_q * (nh / nkv) <= 1 << 24, "attention_tree: bad sizes max_q=%d words=%d chunk=%d pieces=%d", max_q, words, chunk, pieces);
  if (items == 0 || T == 0 || max_q == 0) return 0;
  Args a{out, qkv, kv, block_table, bt_stride, q_start, q_len, ctx_len, seq_slot, mask, words, positions, sink,
         scratch + (size_t)T * nh * pieces * 2, scratch, items, T, width, nh, nkv, nh / nkv, hd, pages, page_size, window, max_q, scale, softcap};
  const int size = dtype == MI_F32 ? 4 : 2;
  const bool wide = hd % 4 == 0 && (long long)width % 4 == 0 && (((uintptr_t)qkv | (uintptr_t)kv) % (4 * size)) == 0;
  MI_REQUIRE(dtype == MI_F32 || dtype == MI_BF16, "attention_tree: unknown type");
  if (dtype == MI_F32) return launch_sized<float>(a, chunk, pieces, wide, stream);
  return launch_sized<__nv_bfloat16>(a, chunk, pieces, wide, stream);
}
