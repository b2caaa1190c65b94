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
#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int MAX_PAIRS = 4096;                // of one call of `places`: a column of 16 bytes of each fits a block's shared memory
constexpr int SMEM_WANTED = 48 << 10;          // four blocks of this size share an SM and take turns at reading and writing
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
  int n, columns;                     // pairs; columns (units) of a block
  int page, token_units;              // rows of a head's part of a place, units of such a row
};

// One block: columns blockIdx.x * columns .. of layer blockIdx.y, of all pairs.
template <typename U, bool FILLED>
__global__ void __launch_bounds__(THREADS) move_places_kernel(Places a) {
  extern __shared__ __align__(16) unsigned char smem[];
  U* stage = reinterpret_cast<U*>(smem);                                                     // [n, columns]
  const long long c0 = (long long)blockIdx.x * a.columns;
  const int cols = (int)min((long long)a.columns, a.row_units - c0), total = a.n * cols;
  U* layer = reinterpret_cast<U*>(a.base) + (long long)blockIdx.y * a.places * a.row_units + c0;
  mi::grid_dependency_sync();
  auto wanted = [&](int k, int c, int from, int to) {
    if ((unsigned)from >= (unsigned long long)a.places || (unsigned)to >= (unsigned long long)a.places || from == to) return false;
    return !FILLED || (int)((c0 + c) / a.token_units % a.page) < a.filled[k];
  };
  for (int i = threadIdx.x; i < total; i += THREADS) {
    const int k = i / cols, c = i - k * cols, from = a.src[k];
    if (wanted(k, c, from, a.dst[k])) copy_to_shared(stage + i, layer + from * a.row_units + c);
  }
  copies_done();
  for (int i = threadIdx.x; i < total; i += THREADS) {
    const int k = i / cols, c = i - k * cols, to = a.dst[k];
    if (wanted(k, c, a.src[k], to)) layer[to * a.row_units + c] = stage[i];
  }
}

struct Rows {
  void* base;
  const int *src, *dst, *start;       // places page * page_size + offset; start [groups + 1]
  long long pages;
  int pairs, planes, plane_step;      // pairs in all; (layer, key or value, head) triples, and how many of them a block takes
  int heads2, page, row_units, most;  // key and value heads of a layer; units of a row; rows of a group that are moved at a time
};

// One block: plane_step planes of group blockIdx.y, `most` rows at a time.
template <typename U>
__global__ void __launch_bounds__(THREADS) move_rows_kernel(Rows a) {
  extern __shared__ __align__(16) unsigned char smem[];
  U* stage = reinterpret_cast<U*>(smem);                                                     // [planes of the block, most, row_units]
  const int p0 = blockIdx.x * a.plane_step, planes = min(a.plane_step, a.planes - p0);
  mi::grid_dependency_sync();
  const int lo = max(a.start[blockIdx.y], 0), hi = min(a.start[blockIdx.y + 1], a.pairs);
  const long long limit = a.pages * a.page;
  auto at = [&](int plane, int place) {      // of (layer, w * heads + h)
    const long long page = (long long)(plane / a.heads2) * a.pages + place / a.page;
    return ((page * a.heads2 + plane % a.heads2) * a.page + place % a.page) * a.row_units;
  };
  U* base = reinterpret_cast<U*>(a.base);
  for (int k0 = lo; k0 < hi; k0 += a.most) {
    const int rows = min(a.most, hi - k0), width = rows * a.row_units, total = planes * width;
    for (int i = threadIdx.x; i < total; i += THREADS) {
      const int p = i / width, k = k0 + (i - p * width) / a.row_units, u = i % a.row_units, from = a.src[k], to = a.dst[k];
      if ((unsigned)from < limit && (unsigned)to < limit && from != to) copy_to_shared(stage + i, base + at(p0 + p, from) + u);
    }
    copies_done();
    for (int i = threadIdx.x; i < total; i += THREADS) {
      const int p = i / width, k = k0 + (i - p * width) / a.row_units, u = i % a.row_units, from = a.src[k], to = a.dst[k];
      if ((unsigned)from < limit && (unsigned)to < limit && from != to) base[at(p0 + p, to) + u] = stage[i];
    }
    __syncthreads();
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
  if (allow_shared(move_places_kernel<U, FILLED>, ready)) return 1;
  // columns: what the wanted shared memory holds, at least 8 (128 bytes in a row) as long as the most allows, and few enough that small
  // calls are spread over the GPU
  const long long per = (long long)a.n * sizeof(U), spread = (a.row_units * layers + 4 * mi::sm_count() - 1) / (4 * mi::sm_count());
  long long c = SMEM_WANTED / per;
  if (c < 8) c = 8;
  if (c > SMEM_MOST / per) c = SMEM_MOST / per;
  const long long least = spread > 16 ? spread : 16;
  if (c > least) c = least;
  if (c > a.row_units) c = a.row_units;
  a.columns = (int)c;
  const long long blocks = (a.row_units + c - 1) / c;
  MI_REQUIRE(blocks <= 0x7fffffffll && layers <= 65535, "cache moves: %lld blocks of %d layers are too many for one launch", blocks, layers);
  if (mi::launch(move_places_kernel<U, FILLED>, dim3((unsigned)blocks, layers), dim3(THREADS), (size_t)(per * c), stream, a) != cudaSuccess)
    return mi_fail("cache moves: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  MI_LAUNCH_OK("cache moves");
  return 0;
}

template <typename U>
int launch_rows(Rows a, int groups, cudaStream_t stream) {
  static bool ready[64] = {};
  if (allow_shared(move_rows_kernel<U>, ready)) return 1;
  const long long row = (long long)a.row_units * sizeof(U);
  MI_REQUIRE(row <= SMEM_MOST, "move_cache_rows: rows of %lld bytes are too long", row);
  if (a.most > SMEM_MOST / row) a.most = (int)(SMEM_MOST / row);
  const long long per = row * a.most, spread = ((long long)a.planes * groups + 4 * mi::sm_count() - 1) / (4 * mi::sm_count());
  long long step = SMEM_WANTED / per;
  if (step > spread) step = spread;
  if (step < 1) step = 1;
  a.plane_step = (int)step;
  if (mi::launch(move_rows_kernel<U>, dim3((unsigned)((a.planes + step - 1) / step), groups), dim3(THREADS), (size_t)(per * step), stream, a) != cudaSuccess)
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
  Rows a{base, src, dst, start, pages, pairs, 2 * layers * heads, 0, 2 * heads, page, (int)(row_bytes / unit), most};
  if (unit == 16) return launch_rows<uint4>(a, groups, stream);
  if (unit == 4) return launch_rows<uint32_t>(a, groups, stream);
  if (unit == 2) return launch_rows<uint16_t>(a, groups, stream);
  return launch_rows<uint8_t>(a, groups, stream);
}
