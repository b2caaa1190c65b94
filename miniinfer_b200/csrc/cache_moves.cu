// Copies inside caches and per-request states: what a request with several continuations needs when it forks, when its beams
// change places and when the accepted path of a drafted tree moves to the front of the tree's rows.
//
//   places    base[l, dst[k], :] = base[l, src[k], :]          rows of a state, or pages of a pool (whole or as far as filled)
//   rows      pool[l, page, w, h, offset, :] of a place dst[k] = that of src[k], all layers, keys and values, all heads
//
// Every source is read before any destination is written - among all pairs of a call, and in `rows` among the pairs of a group -, so
// a permutation needs no second buffer: a block takes the same few columns of ALL pairs, copies them to shared memory, waits, and
// writes them out.  Different blocks touch different columns, so no block can overwrite what another still has to read.  A pair whose
// places are equal costs nothing; one whose source or destination is out of range (a padded one: -1) is left out.
//
// Nothing is computed; the bytes are the bound.  Loads are asynchronous copies of 16 bytes into shared memory (of 4 or 2 where rows
// or the base are not aligned to more), so what a block has on its way is its whole share and not its registers.
//
// Measured: 96 pages of 28 layers (1.41 GB read and written) 216 us, 6.5 TB/s, the rate of a plain copy; paths of 8 of 64 tokens for 64 requests (117 MB)
// 20.5 us, 5.7 TB/s; 32 states of 12 layers of 1 MB 81 us (what keeps its place costs nothing); 3 pages (15 MB) 6.9 us; calls of a MB or less 1.7 to 2.5 us,
// which a launch takes.  Rows that are not whole 16 bytes are copied by 4 or 2 bytes: 32 states of 12 layers of 95151 float32 77 us, 38 % of the bytes' rate.
#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int MAX_PAIRS = 4096;                // of one call of `places`: a column of 16 bytes of each fits a block's shared memory
constexpr int SMEM_WANTED = 32 << 10;          // six blocks of this size share an SM and take turns at reading and writing (0.12 GB of rows: 20.5 us; by 48 KB 22.9)
constexpr int SMEM_MOST = 200 << 10;

template <typename U>
__device__ __forceinline__ void copy_to_shared(U* dst, const U* src) {
  if constexpr (sizeof(U) == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
  } else if constexpr (sizeof(U) == 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
  } else {
    *dst = *src;
  }
}
__device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
}

struct Places {
  void* base;
  const int *src, *dst, *filled;      // [n]; filled or null: the first filled[k] of a place's `page` rows only
  long long places, row_units;        // places of a layer; units of a place
  int n, log_columns;                 // pairs; columns (units) of a block, a power of two
  int page, token_units;              // rows of a head's part of a place, units of such a row
};

// One block: a few columns of layer blockIdx.y, of all pairs.  A thread stays in its column; 2^log_columns threads side by side take a pair.
template <typename U>
__global__ void __launch_bounds__(THREADS) move_places_kernel(Places a) {
  extern __shared__ __align__(16) unsigned char smem[];
  U* stage = reinterpret_cast<U*>(smem);                                                     // [n, columns]
  const int columns = 1 << a.log_columns, c = threadIdx.x & (columns - 1), k0 = threadIdx.x >> a.log_columns, step = THREADS >> a.log_columns;
  const long long at = ((long long)blockIdx.x << a.log_columns) + c;
  U* column = reinterpret_cast<U*>(a.base) + (long long)blockIdx.y * a.places * a.row_units + at;
  mi::grid_dependency_sync();
  if (at < a.row_units) {
#pragma unroll 4
    for (int k = k0; k < a.n; k += step) {
      const int from = a.src[k], to = a.dst[k];
      const bool wanted = (unsigned)from < (unsigned long long)a.places && (unsigned)to < (unsigned long long)a.places && from != to;
      if (wanted) copy_to_shared(stage + (k << a.log_columns) + c, column + from * a.row_units);
    }
  }
  copies_done();
  if (at < a.row_units) {
#pragma unroll 4
    for (int k = k0; k < a.n; k += step) {
      const int from = a.src[k], to = a.dst[k];
      const bool wanted = (unsigned)from < (unsigned long long)a.places && (unsigned)to < (unsigned long long)a.places && from != to;
      if (wanted) column[to * a.row_units] = stage[(k << a.log_columns) + c];
    }
  }
}

// The same for places that are filled in part: a block lists the pairs that have something in its columns first, for half of them as a rule have not
// (465 pairs of pages filled to any length, 20 layers, 152 MB: 32 us instead of 67; 3 pairs of 28 layers 6.9 instead of 7.6).
template <typename U>
__global__ void __launch_bounds__(THREADS) move_filled_kernel(Places a) {
  extern __shared__ __align__(16) unsigned char smem[];
  int* list = reinterpret_cast<int*>(smem);                                                  // [3][n]: from, to, filled
  U* stage = reinterpret_cast<U*>(smem + (a.n * 12 + 15) / 16 * 16);                         // [n, columns]
  __shared__ int count;
  const unsigned columns = 1u << a.log_columns, c = threadIdx.x & (columns - 1), first = blockIdx.x << a.log_columns, at = first + c;
  const int k0 = threadIdx.x >> a.log_columns, step = THREADS >> a.log_columns;
  const unsigned token_first = first / a.token_units, token_last = (min(first + columns, (unsigned)a.row_units) - 1) / a.token_units, token = at / a.token_units;
  const int row = token % a.page, lowest = token_first / a.page == token_last / a.page ? token_first % a.page : 0;      // of the thread's column; of the block's
  U* column = reinterpret_cast<U*>(a.base) + (long long)blockIdx.y * a.places * a.row_units + at;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  mi::grid_dependency_sync();
  for (int k = threadIdx.x; k < a.n; k += THREADS) {
    const int from = a.src[k], to = a.dst[k], filled = a.filled[k];
    if ((unsigned)from < (unsigned long long)a.places && (unsigned)to < (unsigned long long)a.places && from != to && lowest < filled) {
      const int i = atomicAdd(&count, 1);      // (in any order: destinations differ)
      list[i] = from;
      list[a.n + i] = to;
      list[2 * a.n + i] = filled;
    }
  }
  __syncthreads();
  const int n = at < a.row_units ? count : 0;
#pragma unroll 4
  for (int k = k0; k < n; k += step)
    if (row < list[2 * a.n + k]) copy_to_shared(stage + (k << a.log_columns) + c, column + list[k] * a.row_units);
  copies_done();
#pragma unroll 4
  for (int k = k0; k < n; k += step)
    if (row < list[2 * a.n + k]) column[list[a.n + k] * a.row_units] = stage[(k << a.log_columns) + c];
}

struct Rows {
  void* base;
  const int *src, *dst, *start;       // places page * page_size + offset; start [groups + 1]
  long long pages;
  int pairs, planes, plane_step;      // pairs in all; (layer, key or value, head) triples, and how many of them a block takes
  int heads2, page, row_units, most;  // key and value heads of a layer; units of a row; rows of a group that are moved at a time
  int columns, log_lanes;             // units of a row that are moved at a time, all of them where they fit; 2^log_lanes threads side by side take them
};

// One block: plane_step planes of group blockIdx.y, `most` rows at a time.  An address is the sum of two numbers, of the pair and of the plane: tables, for
// divisions would cost more than the copies.
template <typename U>
__global__ void __launch_bounds__(THREADS) move_rows_kernel(Rows a) {
  extern __shared__ __align__(16) unsigned char smem[];
  longlong2* of_pair = reinterpret_cast<longlong2*>(smem);                                   // [most]: from, to; -1: nothing to do
  long long* of_plane = reinterpret_cast<long long*>(of_pair + a.most);                      // [plane_step]
  U* stage = reinterpret_cast<U*>(smem + (a.most * 16 + a.plane_step * 8 + 15) / 16 * 16);   // [planes of the block, rows, columns]
  const int p0 = blockIdx.x * a.plane_step, planes = min(a.plane_step, a.planes - p0);
  const int lane = threadIdx.x & ((1 << a.log_lanes) - 1), first = threadIdx.x >> a.log_lanes, step = THREADS >> a.log_lanes;
  for (int p = threadIdx.x; p < planes; p += THREADS)
    of_plane[p] = ((long long)((p0 + p) / a.heads2) * a.pages * a.heads2 + (p0 + p) % a.heads2) * a.page * a.row_units;
  mi::grid_dependency_sync();
  const int lo = max(a.start[blockIdx.y], 0), hi = min(a.start[blockIdx.y + 1], a.pairs);
  const long long limit = a.pages * a.page;
  U* base = reinterpret_cast<U*>(a.base);
  auto of_place = [&](int place) { return ((long long)(place / a.page) * a.heads2 * a.page + place % a.page) * a.row_units; };
  for (int k0 = lo; k0 < hi; k0 += a.most) {
    const int rows = min(a.most, hi - k0), total = planes * rows;
    for (int k = threadIdx.x; k < rows; k += THREADS) {
      const int from = a.src[k0 + k], to = a.dst[k0 + k];
      const bool wanted = (unsigned)from < limit && (unsigned)to < limit && from != to;
      of_pair[k] = wanted ? make_longlong2(of_place(from), of_place(to)) : make_longlong2(-1, -1);
    }
    __syncthreads();
    for (int c0 = 0; c0 < a.row_units; c0 += a.columns) {
      const int columns = min(a.columns, a.row_units - c0);
#pragma unroll 4
      for (int i = first; i < total; i += step) {
        const int p = i / rows;
        const long long from = of_pair[i - p * rows].x;
        if (from >= 0)
          for (int u = lane; u < columns; u += 1 << a.log_lanes) copy_to_shared(stage + i * a.columns + u, base + of_plane[p] + from + c0 + u);
      }
      copies_done();
#pragma unroll 4
      for (int i = first; i < total; i += step) {
        const int p = i / rows;
        const long long to = of_pair[i - p * rows].y;
        if (to >= 0)
          for (int u = lane; u < columns; u += 1 << a.log_lanes) base[of_plane[p] + to + c0 + u] = stage[i * a.columns + u];
      }
      __syncthreads();
    }
  }
}

// The widest unit that divides every one of the sizes and the address.
int unit_of(const void* base, long long bytes) {
  const unsigned long long x = (unsigned long long)(uintptr_t)base | (unsigned long long)bytes;
  return x % 16 == 0 ? 16 : x % 4 == 0 ? 4 : x % 2 == 0 ? 2 : 1;
}

template <typename K>
int allow_shared(K kernel, bool* ready) {      // more shared memory than a kernel gets without asking; asked once per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return mi_fail("cache moves: no current device");
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST);
    if (e != cudaSuccess) return mi_fail("cache moves: %d bytes of shared memory were refused: %s", SMEM_MOST, cudaGetErrorString(e));
    ready[dev] = true;
  }
  return 0;
}

template <typename U, bool FILLED>
int launch_places(Places a, int layers, cudaStream_t stream) {
  static bool ready[64] = {};
  auto kernel = FILLED ? move_filled_kernel<U> : move_places_kernel<U>;
  if (allow_shared(kernel, ready)) return 1;
  // columns: what the wanted shared memory holds, at least 8 (128 bytes in a row) as long as the most allows, no more than a place or the threads have,
  // and few enough that small calls are spread over the GPU
  const long long list = FILLED ? (a.n * 12ll + 15) / 16 * 16 : 0, per = (long long)a.n * sizeof(U), spread = (a.row_units * layers + 4 * mi::sm_count() - 1) / (4 * mi::sm_count());
  long long most = SMEM_WANTED / per;
  if (most < 8) most = 8;
  if (most > (SMEM_MOST - list) / per) most = (SMEM_MOST - list) / per;
  if (most > (spread > 16 ? spread : 16)) most = spread > 16 ? spread : 16;
  a.log_columns = 0;
  while ((2ll << a.log_columns) <= most && (2 << a.log_columns) <= THREADS && (1ll << a.log_columns) < a.row_units) ++a.log_columns;
  const long long c = 1ll << a.log_columns, blocks = (a.row_units + c - 1) / c;
  MI_REQUIRE(blocks <= 0x7fffffffll && layers <= 65535, "cache moves: %lld blocks of %d layers are too many for one launch", blocks, layers);
  if (mi::launch(kernel, dim3((unsigned)blocks, layers), dim3(THREADS), (size_t)(list + per * c), stream, a) != cudaSuccess)
    return mi_fail("cache moves: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  MI_LAUNCH_OK("cache moves");
  return 0;
}

template <typename U>
int launch_rows(Rows a, int groups, cudaStream_t stream) {
  static bool ready[64] = {};
  if (allow_shared(move_rows_kernel<U>, ready)) return 1;
  // columns: whole rows, or where `most` of them do not fit as much of each as does: units are moved one by one, so what is read before what stays so
  const long long units = (SMEM_MOST - 64 - 16ll * a.most) / (a.most * (long long)sizeof(U));
  MI_REQUIRE(units >= 1, "move_cache_rows: most=%d rows at a time are too many", a.most);
  a.columns = units < a.row_units ? (int)units : a.row_units;
  const long long per = (long long)a.columns * sizeof(U) * a.most + 8, spread = ((long long)a.planes * groups + 4 * mi::sm_count() - 1) / (4 * mi::sm_count());
  long long step = SMEM_WANTED / per;
  if (step > spread) step = spread;
  if (step < 1) step = 1;
  a.plane_step = (int)step;
  a.log_lanes = 0;
  while ((1 << a.log_lanes) < a.columns && (2 << a.log_lanes) <= THREADS) ++a.log_lanes;
  if (mi::launch(move_rows_kernel<U>, dim3((unsigned)((a.planes + step - 1) / step), groups), dim3(THREADS), (size_t)(per * step + a.most * 16 + 16), stream, a) != cudaSuccess)
    return mi_fail("move_cache_rows: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  MI_LAUNCH_OK("move_cache_rows");
  return 0;
}

}  // namespace

// base [layers, places, place_bytes].  filled (or null) [n]: only the rows below it of each of a place's parts of `page` rows of
// token_bytes are copied.
MI_API int mi_move_places(void* base, int layers, long long places, long long place_bytes, const int* src, const int* dst, const int* filled,
                          int page, long long token_bytes, int n, cudaStream_t stream) {
  MI_REQUIRE(layers >= 0 && places >= 0 && place_bytes >= 0 && n >= 0, "cache moves: bad sizes layers=%d places=%lld bytes=%lld n=%d", layers, places, place_bytes, n);
  MI_REQUIRE(n <= MAX_PAIRS, "cache moves: %d pairs, at most %d go in one call", n, MAX_PAIRS);
  if (layers == 0 || places == 0 || place_bytes == 0 || n == 0) return 0;
  MI_REQUIRE(places <= 0x7fffffffll, "cache moves: %lld places are too many", places);
  if (filled) MI_REQUIRE(page > 0 && token_bytes > 0 && place_bytes % (page * token_bytes) == 0, "cache moves: a place of %lld bytes is not made of %d rows of %lld", place_bytes, page, token_bytes);
  if (filled) MI_REQUIRE(place_bytes <= 0x7fffffffll, "cache moves: a place of %lld bytes is too large to be copied in part", place_bytes);
  const int unit = unit_of(base, filled ? (place_bytes | token_bytes) : place_bytes);
  Places a{base, src, dst, filled, places, place_bytes / unit, n, 0, page, filled ? (int)(token_bytes / unit) : 1};
  if (filled) {
    if (unit == 16) return launch_places<uint4, true>(a, layers, stream);
    if (unit == 4) return launch_places<uint32_t, true>(a, layers, stream);
    if (unit == 2) return launch_places<uint16_t, true>(a, layers, stream);
    return launch_places<uint8_t, true>(a, layers, stream);
  }
  if (unit == 16) return launch_places<uint4, false>(a, layers, stream);
  if (unit == 4) return launch_places<uint32_t, false>(a, layers, stream);
  if (unit == 2) return launch_places<uint16_t, false>(a, layers, stream);
  return launch_places<uint8_t, false>(a, layers, stream);
}

// base [layers, pages, 2, heads, page, row_bytes]; src, dst [pairs]; start [groups + 1]; most: rows of a group that are moved at a time.
MI_API int mi_move_cache_rows(void* base, int layers, long long pages, int heads, int page, long long row_bytes, const int* src, const int* dst,
                              const int* start, int pairs, int groups, int most, cudaStream_t stream) {
  MI_REQUIRE(layers >= 0 && pages >= 0 && heads > 0 && page > 0 && row_bytes > 0 && pairs >= 0 && groups >= 0 && most > 0, "move_cache_rows: bad sizes");
  if (layers == 0 || pages == 0 || pairs == 0 || groups == 0) return 0;
  MI_REQUIRE(pages * page <= 0x7fffffffll && 2ll * layers * heads <= 0x7fffffffll && groups <= 65535, "move_cache_rows: %lld pages of %d rows or %d groups are too many", pages, page, groups);
  const int unit = unit_of(base, row_bytes);
  if (most > pairs) most = pairs;
  Rows a{base, src, dst, start, pages, pairs, 2 * layers * heads, 0, 2 * heads, page, (int)(row_bytes / unit), most, 0, 0};
  if (unit == 16) return launch_rows<uint4>(a, groups, stream);
  if (unit == 4) return launch_rows<uint32_t>(a, groups, stream);
  if (unit == 2) return launch_rows<uint16_t>(a, groups, stream);
  return launch_rows<uint8_t>(a, groups, stream);
}
