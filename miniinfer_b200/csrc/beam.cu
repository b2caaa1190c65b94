// Beam search's selection: the n best continuations of a request over all of its beams and the vocabulary.
//
//   score(r, v) = cum[r] + x[r, v] - log(sum_u exp(x[r, u]))          r: a row of logits, one per beam
//
// The best score comes first; of equal ones the lower row, in a row the larger logit and then the lower token.  A score that is no number
// or minus infinity is no candidate (a forbidden token, a beam that has ended, a row with a logit that is no number); places that no
// candidate fills get token -1, parent -1, score -inf.
//
// One launch, one pass over the logits.  A block walks a stretch of a row in tiles of 4096, three tiles on their way in shared memory while one is
// in registers: a running maximum and sum of exp(x - maximum) a thread, and the stretch's n best logits so far - a row's order does not depend on its
// normaliser.  Past the first tile hardly a value beats the n-th best, and a tile costs its exponentials; warps go through the tiles without waiting for one
// another.  The last block of a request to finish puts the pieces together: the rows' normalisers, then the n best of (stretches x n) candidates.
//
// The n best of a tile without sorting it: a thread's best of its own 16, and of each warp's 32 the ceil(n / 8)-th - eight warps make n of them -; the
// least of these eight bounds the tile's n-th best from below.  What is not below it - 2 or 3 n, as a rule - is collected in shared memory and ranked
// by counting.  Should many more come (equal values, a tile of which a warp has only poor ones or none), the n-th best of the 256 threads'
// bests is found exactly: at most n times a thread's 16 values are not below that.
//
// Float32 holds a value and a row's sum of exponentials, made by the hardware's exponential: a normaliser errs by up to 3.5e-6 (derived beside the tests).
// From there on - its logarithm, the scores and their order - all is in 64 bits, and the score that is handed out is rounded once.  So a row's own candidates
// are always in their order, and those of different beams wherever their scores are further apart than two normalisers may err.
//
// Measured: 64 requests, 263 rows of 151936 float32 (160 MB) 45 us, 3.5 TB/s (49 us with a barrier in each tile): the walk itself takes 23 us, the memory's
// full rate, but 5 us pass before the first tile is ranked and 14 in the last ranking and joining, chains of short steps with nothing on its way.  4 rows of one request 13.2 to 13.7 us for
// 2.4 MB: that chain and little else.  In bf16 41 and 13.8 us, bound by the instructions a value takes.  Rows whose bytes are not a multiple of 16 are read value by
// value, with nothing on its way ahead: 263 rows of 151935 62 us in float32, 119 in bf16.
#include "attention_scores.cuh"
#include "common.cuh"

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, ITEMS = 16, TILE = THREADS * ITEMS;
constexpr int STAGES = 4;                     // tiles in shared memory: three on their way, one that was just read
constexpr int MAX_BEST = 128;
constexpr int ROOM = MAX_BEST * (ITEMS + 1) + 384;      // candidates: the n best so far and a tile's on top; what is over lets a few tiles come before they are thinned out
// (263 rows of 151936: 48 us; 2, which are one and a half rounds of blocks: 63.  As many stretches as two blocks an SM in one round allow: 1 to 7 rows 15 to 56 us instead of 12 to
// 22, for more pieces take longer to join than the walk gains; 8 and 24 to 48 rows up to 18 % slower or as now, 16 and 64 rows 16.7 and 20.8 instead of 18.9 and 27.0)
constexpr int BLOCKS_WANTED = 1;
constexpr int MANY = 256;                     // candidates of a tile that are ranked without a second thought
constexpr unsigned FULL = 0xffffffffu;

// Rises with the value; minus and plus zero are one.  (Values that are no numbers never come here.)
__device__ __forceinline__ uint32_t rising(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
// A logit and its token as one number: larger logit first, lower token first.  0: none.
__device__ __forceinline__ uint64_t key_of(float v, int token) { return v > -INFINITY ? (uint64_t)rising(v) << 32 | (0x7fffffffu - (uint32_t)token) : 0ull; }
__device__ __forceinline__ int token_of(uint64_t key) { return (int)(0x7fffffffu - (uint32_t)key); }
__device__ __forceinline__ uint64_t rising64(double d) {
  const uint64_t u = (uint64_t)__double_as_longlong(d + 0.0);
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double score_of(uint64_t image) { return __longlong_as_double((long long)((image >> 63) ? (image & 0x7fffffffffffffffull) : ~image)); }

// The warp's 32 values, falling from lane 0 to lane 31.
__device__ __forceinline__ uint64_t sorted_in_warp(uint64_t x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const uint64_t other = __shfl_xor_sync(FULL, x, j);
      const bool larger = ((lane & j) == 0) == ((lane & k) == 0);      // this lane keeps the larger of the two
      x = (other > x) == larger ? other : x;
    }
  return x;
}

// The k-th largest of the warp's 32 numbers, or 0.
__device__ __forceinline__ uint32_t kth_of_warp(uint32_t x, int k) {
  uint32_t largest = 0;
#pragma unroll 1
  for (int i = 0; i < k; ++i) {
    largest = __reduce_max_sync(FULL, x);
    const int at = __ffs(__ballot_sync(FULL, x == largest)) - 1;
    if ((int)(threadIdx.x & 31) == at) x = 0;
  }
  return largest;
}
// The least of the warps' ceil(n / WARPS)-th largest: at least n of the block's THREADS numbers are not below it.
__device__ __forceinline__ uint32_t quick_bound(uint32_t x, int n, uint32_t* of_warp /* WARPS */) {
  const uint32_t mine = kth_of_warp(x, (n + WARPS - 1) / WARPS);
  if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = mine;
  __syncthreads();
  uint32_t bound = of_warp[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) bound = min(bound, of_warp[w]);
  return bound;
}

// The n-th largest of the block's THREADS keys (n <= THREADS; 0 where fewer are not 0).  A key's rank is its place in its own warp's order and, by
// halving, in the other warps'; of equal ones the lower warp's comes first.
// (not inlined, like what else is done once a block: a second copy of the code would have to be fetched as well)
__device__ __noinline__ uint64_t nth_best(uint64_t key, int n, uint64_t* lists /* THREADS */, uint64_t* result) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t mine = sorted_in_warp(key);
  lists[threadIdx.x] = mine;
  __syncthreads();
  int place[WARPS];      // of each list: how many come before mine
#pragma unroll
  for (int w = 0; w < WARPS; ++w) place[w] = 0;
#pragma unroll
  for (int half = 16; half > 0; half >>= 1)
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const uint64_t x = lists[32 * w + place[w] + half - 1];
      if (x > mine || (x == mine && w < warp)) place[w] += half;
    }
  int rank = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {      // (31 looked at; the last of a list)
    if (place[w] == 31) {
      const uint64_t x = lists[32 * w + 31];
      if (x > mine || (x == mine && w < warp)) place[w] = 32;
    }
    rank += w == warp ? lane : place[w];
  }
  if (rank == n - 1) *result = mine;
  __syncthreads();
  return *result;
}

// The candidates of the block ranked; the n best stay, in their order.  (All that have been found are there: a barrier lies behind them.)  Answers what a
// value has to beat from here on.
__device__ __noinline__ float keep_best(uint64_t* pool, int* count, int n, uint64_t* ranked /* MAX_BEST at least */) {
  const int got = *count;
#pragma unroll 1
  for (int i = threadIdx.x; i < got; i += THREADS) {
    const uint64_t key = pool[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < got; ++j) rank += pool[j] > key;
    if (rank < n) ranked[rank] = key;
  }
  __syncthreads();
  const int kept = min(got, n);
  for (int i = threadIdx.x; i < kept; i += THREADS) pool[i] = ranked[i];
  if (threadIdx.x == 0) *count = kept;
  const float bar = got >= n ? value_of(ranked[n - 1]) : -INFINITY;
  __syncthreads();
  return bar;
}

struct Args {
  int *tokens, *parents;         // [requests, n]
  float* scores;
  const void* logits;            // [R, V]
  const float* cum;              // [R]
  const int* start;              // [requests + 1]
  float2* sums;                  // [R, stretches]: maximum, sum of exp(x - maximum)
  uint64_t* best;                // [R, stretches, n]: keys, 0 where there is none
  double2* norm;                 // [R]: the maximum, cum minus the log of the sum
  int* arrivals;                 // [requests + 1], zero; left zero: blocks of a request that have come, and of all rows
  int R, V, requests, n, stretches, tiles;      // tiles of a stretch
};

// The request that row r belongs to, or -1; by a warp.
__device__ __forceinline__ int request_of(const Args& a, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.requests;      // the answer lies in lo .. hi - 1: the last request whose start is not past r
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned m = __ballot_sync(FULL, at < hi && a.start[at] <= r);
    if (m == 0) return -1;
    const int last = 31 - __clz(m);
    lo += last * step;
    hi = min(hi, lo + step);
  }
  return a.start[lo] <= r && r < a.start[lo + 1] ? lo : -1;
}

// The token of a thread's j-th value; they rise with j.
template <typename T, bool WIDE>
__device__ __forceinline__ int token_at(int begin, int j) {
  constexpr int PER = WIDE ? 16 / sizeof(T) : 1;
  return begin + (j / PER * THREADS + (int)threadIdx.x) * PER + j % PER;
}
// A thread fetches what it will read itself, so no barrier stands between the copy and the reading.  stage, from: of the thread's first 16 bytes; left: values
// of the row from there on.
template <typename T>
__device__ __forceinline__ void fetch(uint32_t stage, const T* from, int left) {
  constexpr int PER = 16 / sizeof(T);
  if (left >= TILE) {      // (the tile's last 16 bytes lie at most that far on)
#pragma unroll
    for (int j = 0; j < ITEMS / PER; ++j)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(stage + j * THREADS * 16), "l"(from + j * THREADS * PER) : "memory");
  } else {
#pragma unroll 1
    for (int j = 0; j < ITEMS / PER && j * THREADS * PER < left; ++j)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(stage + j * THREADS * 16), "l"(from + j * THREADS * PER) : "memory");
  }
}
template <typename T, bool WIDE>
__device__ __forceinline__ void read_tile(float (&v)[ITEMS], const unsigned char* stage, const T* row, int begin, int end) {
  if constexpr (WIDE) {
    constexpr int PER = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < ITEMS / PER; ++j) {
      const uint4 raw = *reinterpret_cast<const uint4*>(stage + (j * THREADS + threadIdx.x) * 16);
      const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int e = 0; e < PER; ++e) v[j * PER + e] = mi::to_float(x[e]);
    }
    if (begin + TILE > end) {
#pragma unroll
      for (int j = 0; j < ITEMS; ++j)
        if (token_at<T, WIDE>(begin, j) >= end) v[j] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int at = begin + j * THREADS + (int)threadIdx.x;
      v[j] = at < end ? mi::to_float(row[at]) : -INFINITY;
    }
  }
}

// A block has come, one of all: the last finds all others before it.  (The counter goes back to zero by itself.)
__device__ __forceinline__ bool last_of_all(const Args& a) {
  const unsigned others = gridDim.x * a.R - 1;
  return atomicInc(reinterpret_cast<unsigned*>(&a.arrivals[a.requests]), others) == others;
}
// The very last of all blocks leaves the requests' counters at zero, also where a list that does not rise has sent a request fewer blocks than it counts
// on.  (Up to `step` requests without a loop, whose instructions would have to be fetched: 64 requests 45.2 us, with a loop alone 45.6, without all this 44.7.)
__device__ __forceinline__ void clear_counters(const Args& a, int first, int step) {
  if (first < a.requests) a.arrivals[first] = 0;
  if (a.requests > step)
#pragma unroll 1
    for (int q = first + step; q < a.requests; q += step) a.arrivals[q] = 0;
}

// Puts a request's pieces together; by the whole block.  `stages`: NEAR candidates' keys and images.  `shared`: room for `room` candidates' images, keys
// and rows.  A candidate's order: the score's image, then the lower row, then the row's key.
constexpr int NEAR = 4096;
__device__ __noinline__ void finish(const Args& a, int request, int r0, int r1, uint32_t* of_warp, unsigned char* stages, unsigned char* shared, int room, uint64_t* lists, uint64_t* nth, int* count) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pieces = (r1 - r0) * a.stretches, total = pieces * a.n;
  const uint64_t* keys = a.best + (size_t)r0 * a.stretches * a.n;
  // the best of every piece first, then the second of every piece, ...: the first of a thread's candidates are good ones
  auto place_of = [&](int i) { return keys + (size_t)(i % pieces) * a.n + i / pieces; };
  uint64_t *near_key = reinterpret_cast<uint64_t*>(stages), *near_image = near_key + NEAR;
  auto sums_of = [&](int r) { return r < r1 && lane < a.stretches ? __ldcg(&a.sums[(size_t)r * a.stretches + lane]) : make_float2(-INFINITY, 0.f); };
  float2 near = sums_of(r0 + warp);
  float cum = r0 + warp < r1 ? a.cum[r0 + warp] : 0.f;
  const bool last = threadIdx.x == 0 && last_of_all(a);      // (on its way beside the loads)
#pragma unroll 4
  for (int i = threadIdx.x; i < min(total, NEAR); i += THREADS) near_key[i] = __ldcg(place_of(i));
#pragma unroll 1
  for (int r = r0 + warp; r < r1; r += WARPS) {      // normalisers: a warp a row
    const float2* sums = a.sums + (size_t)r * a.stretches;
    if (r != r0 + warp) {
      near = sums_of(r);
      cum = a.cum[r];
    }
    float m = near.x;
    for (int t = lane + 32; t < a.stretches; t += 32) m = fmaxf(m, __ldcg(&sums[t].x));
    m = mi::warp_max(m);
    double s = near.y != 0.f ? (double)(near.y * expf(near.x - m)) : 0.0;      // (a stretch without weight has no maximum either)
    for (int t = lane + 32; t < a.stretches; t += 32) {
      const float2 p = __ldcg(&sums[t]);
      if (p.y != 0.f) s += (double)(p.y * expf(p.x - m));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
    if (lane == 0) a.norm[r] = make_double2((double)m, (double)cum - log(s));
  }
  if (threadIdx.x == 0) *count = 0;
  if (__syncthreads_or(last)) clear_counters(a, threadIdx.x, THREADS);
  auto row_of = [&](int i) { return r0 + i % pieces / a.stretches; };
  auto score_image = [&](int i, uint64_t key) {      // 0: no candidate
    if (key == 0) return (uint64_t)0;
    // the maximum first: of a row of lowest values (-3.4e38), nothing else would be left of the score
    const double2 norm = a.norm[row_of(i)];
    const double s = ((double)value_of(key) - norm.x) + norm.y;
    return s > -INFINITY ? rising64(s) : (uint64_t)0;      // (also where the score is no number)
  };
  // a bound of the n-th best: images alone, so that candidates equal to it stay
  uint64_t mine = 0;
#pragma unroll 1
  for (int i = threadIdx.x; i < total; i += THREADS) {
    const uint64_t image = score_image(i, i < NEAR ? near_key[i] : __ldcg(place_of(i)));
    if (i < NEAR) near_image[i] = image;
    mine = image > mine ? image : mine;
  }
  uint64_t bound = (uint64_t)quick_bound((uint32_t)(mine >> 32), a.n, of_warp) << 32;
  auto key_at = [&](int i) { return i < NEAR ? near_key[i] : __ldcg(place_of(i)); };
  auto image_at = [&](int i) { return i < NEAR ? near_image[i] : score_image(i, __ldcg(place_of(i))); };
  uint64_t* images = reinterpret_cast<uint64_t*>(shared);
  uint64_t* their_keys = images + room;
  int* rows = reinterpret_cast<int*>(their_keys + room);
#pragma unroll 1
  for (bool again = false;; again = true) {
#pragma unroll 1
    for (int at = threadIdx.x; at < total; at += THREADS) {
      const uint64_t image = image_at(at);
      if (image && image >= bound) {
        const int i = atomicAdd(count, 1);
        if (i < room) {
          images[i] = image;
          their_keys[i] = key_at(at);
          rows[i] = row_of(at);
        }
      }
    }
    __syncthreads();
    if (again || *count <= room) break;
    bound = nth_best(mine, a.n, lists, nth);      // more than there is room for: the exact bound of the threads' bests
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
  }
  const int got = *count;
  int *tokens = a.tokens + (size_t)request * a.n, *parents = a.parents + (size_t)request * a.n;
  float* scores = a.scores + (size_t)request * a.n;
  auto before = [&](uint64_t image, int row, uint64_t key, uint64_t than_image, int than_row, uint64_t than_key) {
    if (image != than_image) return image > than_image;
    return row != than_row ? row < than_row : key > than_key;
  };
  if (got <= room) {
    for (int i = threadIdx.x; i < got; i += THREADS) {
      const uint64_t image = images[i], key = their_keys[i];
      const int row = rows[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < got; ++j) {
        const uint64_t x = images[j];
        rank += x > image;
        if (x == image && j != i) rank += before(x, rows[j], their_keys[j], image, row, key);
      }
      if (rank < a.n) {
        tokens[rank] = token_of(key);
        parents[rank] = row;
        scores[rank] = (float)score_of(image);
      }
    }
    for (int i = got + threadIdx.x; i < a.n; i += THREADS) {
      tokens[i] = parents[i] = -1;
      scores[i] = -INFINITY;
    }
    return;
  }
  // more candidates than there is room for (many equal scores): one place at a time
  uint64_t last_image = ~0ull, last_key = ~0ull;
  int last_row = -1;
  for (int place = 0; place < a.n; ++place) {
    uint64_t image = 0, key = 0;
    int row = 0x7fffffff;
#pragma unroll 1
    for (int at = threadIdx.x; at < total; at += THREADS) {
      const uint64_t x = image_at(at), k = key_at(at);
      if (x && before(last_image, last_row, last_key, x, row_of(at), k) && before(x, row_of(at), k, image, row, key)) {
        image = x;
        key = k;
        row = row_of(at);
      }
    }
    __syncthreads();
    images[threadIdx.x] = image;
    their_keys[threadIdx.x] = key;
    rows[threadIdx.x] = row;
    __syncthreads();
    for (int o = THREADS / 2; o > 0; o >>= 1) {
      const int t = threadIdx.x, u = t + o;
      if (t < o && before(images[u], rows[u], their_keys[u], images[t], rows[t], their_keys[t])) {
        images[t] = images[u];
        rows[t] = rows[u];
        their_keys[t] = their_keys[u];
      }
      __syncthreads();
    }
    const bool live = images[0] != 0;
    last_image = images[0];
    last_key = their_keys[0];
    last_row = live ? rows[0] : 0x7fffffff;      // none left: nor for the places behind
    if (threadIdx.x == 0) {
      tokens[place] = live ? token_of(last_key) : -1;
      parents[place] = live ? last_row : -1;
      scores[place] = live ? (float)score_of(last_image) : -INFINITY;
    }
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS)
beam_select_kernel(Args a) {
  extern __shared__ __align__(16) unsigned char stages[];      // [STAGES][TILE]
  __shared__ __align__(16) uint64_t pool[ROOM];
  __shared__ uint64_t lists[THREADS], s_nth;
  __shared__ float s_max[WARPS], s_sum[WARPS];
  __shared__ uint32_t of_warp[WARPS];
  __shared__ int s_count, s_request, s_rows[2], s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.y, stretch = blockIdx.x;
  mi::grid_dependency_sync();
  if (row == a.R) {      // requests without rows: nobody else answers for them
    for (int q = stretch * WARPS + warp; q < a.requests; q += gridDim.x * WARPS)
      if (max(a.start[q], 0) >= min(a.start[q + 1], a.R))
        for (int i = lane; i < a.n; i += 32) {
          a.tokens[(size_t)q * a.n + i] = a.parents[(size_t)q * a.n + i] = -1;
          a.scores[(size_t)q * a.n + i] = -INFINITY;
        }
    return;
  }
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.V;
  const int first = stretch * a.tiles * TILE, end = (int)min((long long)a.V, (long long)first + (long long)a.tiles * TILE), tiles = (end - first + TILE - 1) / TILE;
  constexpr int STAGE_BYTES = TILE * sizeof(T);
  constexpr int PER = 16 / sizeof(T);
  const uint32_t my_stage = (uint32_t)__cvta_generic_to_shared(stages) + threadIdx.x * 16;
  const int mine0 = first + (int)threadIdx.x * PER;      // the thread's first value of the first tile
  auto fetch_first = [&]() {
    if constexpr (WIDE) {
#pragma unroll
      for (int t = 0; t < STAGES - 1; ++t) {
        fetch<T>(my_stage + t * STAGE_BYTES, x + mine0 + t * TILE, end - mine0 - t * TILE);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
    }
  };
  fetch_first();
  if (warp == 0) {
    const int q = request_of(a, row);
    if (lane == 0) {
      s_request = q;
      s_rows[0] = q < 0 ? 0 : max(a.start[q], 0);
      s_rows[1] = q < 0 ? 0 : min(a.start[q + 1], a.R);
      s_count = 0;
    }
  }
  float m = -INFINITY, sum = 0.f;      // of this thread's values
  float bar = -INFINITY;               // what a value has to beat: the n-th best so far, if there are n
  int most = 0;
  auto thin_out = [&]() {
    const float b = keep_best(pool, &s_count, a.n, lists);
    if (b > bar) bar = b;
  };
  // Warps collect what beats the bar as it comes, each at its own pace; they meet where the bar rises.  Should there be no room for all (a row whose tiles get
  // better and better), the stretch is walked once more, all threads' candidates of a tile counted before they are collected.
#pragma unroll 1
  for (bool counted = false;; counted = true) {
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      const int begin = first + t * TILE;
      if constexpr (WIDE) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      float v[ITEMS];
      read_tile<T, WIDE>(v, stages + t % STAGES * STAGE_BYTES, x, begin, end);
      if constexpr (WIDE) {      // into the stage that was read a tile ago
        const int ahead = (t + STAGES - 1) * TILE;
        fetch<T>(my_stage + (t + STAGES - 1) % STAGES * STAGE_BYTES, x + mine0 + ahead, end - mine0 - ahead);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      float top = v[0];
#pragma unroll
      for (int j = 1; j < ITEMS - 1; j += 2) top = mi::max_of(top, v[j], v[j + 1]);
      top = fmaxf(top, v[ITEMS - 1]);
      if (top > m) {
        sum *= mi::ex2_fast((m - top) * 1.4426950408889634f);
        m = top;
      }
      const float off = m == -INFINITY ? 0.f : -m;
      float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < ITEMS; j += 2) {      // (the difference first: values may be as large as they get)
        float d0 = v[j], d1 = v[j + 1];
        mi::add_pair(d0, d1, off, off);
        mi::mul_pair(d0, d1, d0, d1, 1.4426950408889634f);
        mi::add_pair(part[j & 2], part[(j & 2) + 1], mi::ex2_fast(d0), mi::ex2_fast(d1));
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
      int beating = 0;
      if (counted || t == 0) {
        // who has a value that beats the bar; `most`: the candidates that may be there by now, counted without asking (a barrier less)
        beating = __syncthreads_count(top > bar);
        if (beating == 0) continue;
        if (most + beating * ITEMS > ROOM && most > a.n) {
          thin_out();
          most = a.n;
          beating = __syncthreads_count(top > bar);
        }
      }
      uint32_t hits = 0;
      if (top > bar) {
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) hits |= (v[j] > bar ? 1u : 0u) << j;
      }
      // (values by their number out of the stage or the row: registers cannot be asked by number)
      auto key_by_number = [&](int j) {
        const int token = token_at<T, WIDE>(begin, j);
        if constexpr (WIDE) {
          return key_of(mi::to_float(reinterpret_cast<const T*>(stages + t % STAGES * STAGE_BYTES)[(j / PER * THREADS + (int)threadIdx.x) * PER + j % PER]), token);
        } else {
          return key_of(mi::to_float(x[token]), token);
        }
      };
      const bool bounded = t == 0 || (counted && most + beating * ITEMS > ROOM);      // (the first tile has no bar: all of a small vocabulary would be ranked)
      if (bounded) {
        const int before = s_count;
        const uint32_t high = top > -INFINITY ? rising(top) : 0;
        uint64_t bound = (uint64_t)quick_bound(high, a.n, of_warp) << 32;
#pragma unroll 1
        for (bool again = false;; again = true) {
          const float least = bound ? value_of(bound) : -INFINITY;
          uint32_t mine = 0;
#pragma unroll
          for (int j = 0; j < ITEMS; ++j) mine |= (v[j] >= least ? 1u : 0u) << j;
          mine &= hits;
#pragma unroll 1
          for (uint32_t todo = mine; todo; todo &= todo - 1)      // (of equal values the lower tokens)
            if (key_by_number(__ffs(todo) - 1) < bound) mine &= ~(todo & -todo);
          int i = mine ? atomicAdd(&s_count, __popc(mine)) : 0;
#pragma unroll 1
          for (; mine && i < ROOM; mine &= mine - 1) pool[i++] = key_by_number(__ffs(mine) - 1);
          __syncthreads();
          if (again || s_count - before <= MANY) break;
          uint64_t best = 0;      // more than are ranked in a moment: the exact bound of the threads' bests
#pragma unroll
          for (int j = ITEMS - 1; j >= 0; --j)
            if (v[j] == top && top > bar) best = key_of(top, token_at<T, WIDE>(begin, j));
          bound = nth_best(best, a.n, lists, &s_nth);
          if (threadIdx.x == 0) s_count = before;
          __syncthreads();
        }
      } else if (hits) {
        int i = atomicAdd(&s_count, __popc(hits));
#pragma unroll 1
        for (; hits && i < ROOM; hits &= hits - 1) pool[i++] = key_by_number(__ffs(hits) - 1);
      }
      most = bounded ? ROOM : most + beating * ITEMS;
      if (t == 0 || t == 3 || t == 15) {      // the bar rises as the tiles say less
        __syncthreads();
        if (s_count > ROOM) break;
        thin_out();
        most = a.n;
      }
    }
    __syncthreads();
    if (counted || s_count <= ROOM) break;
    __syncthreads();
    if (threadIdx.x == 0) s_count = 0;
    m = bar = -INFINITY;
    sum = 0.f;
    if constexpr (WIDE) asm volatile("cp.async.wait_all;" ::: "memory");
    fetch_first();
  }
  thin_out();
  const int got = s_count;
  uint64_t* best = a.best + ((size_t)row * a.stretches + stretch) * a.n;
  for (int i = threadIdx.x; i < a.n; i += THREADS) best[i] = i < got ? pool[i] : 0;
  // the threads' sums
  const float wm = mi::warp_max(m);
  if (lane == 0) s_max[warp] = wm;
  __syncthreads();
  float all = s_max[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) all = fmaxf(all, s_max[w]);
  const float ws = mi::warp_sum(sum != 0.f ? sum * mi::ex2_fast((m - all) * 1.4426950408889634f) : 0.f);
  if (lane == 0) s_sum[warp] = ws;
  __threadfence();      // the stretch's best, before the block counts as arrived
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = s_sum[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) t += s_sum[w];
    a.sums[(size_t)row * a.stretches + stretch] = make_float2(all, t);
    s_last = 0;
    const int q = s_request;
    if (q >= 0) {
      __threadfence();
      const int blocks = (s_rows[1] - s_rows[0]) * a.stretches;
      if (atomicAdd(&a.arrivals[q], 1) == blocks - 1) {
        a.arrivals[q] = 0;      // ready for the next launch
        s_last = 1;
      }
    }
  }
  __syncthreads();
  if (!s_last) {
    if (warp == 0) {
      bool last = false;
      if (lane == 0) {
        __threadfence();
        last = last_of_all(a);
      }
      if (__shfl_sync(FULL, last, 0)) clear_counters(a, lane, 32);
    }
    return;
  }
  __threadfence();
  finish(a, s_request, s_rows[0], s_rows[1], of_warp, stages, reinterpret_cast<unsigned char*>(pool), ROOM * 8 / 20, lists, &s_nth, &s_count);
}

template <typename T, bool WIDE>
int launch(const Args& a, cudaStream_t stream) {
  const size_t tiles = WIDE ? (size_t)STAGES * TILE * sizeof(T) : 0, smem = tiles > NEAR * 16 ? tiles : NEAR * 16;
  static bool ready[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return mi_fail("beam_select: no current device");
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(beam_select_kernel<T, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return mi_fail("beam_select: %zu bytes of shared memory were refused: %s", smem, cudaGetErrorString(e));
    ready[dev] = true;
  }
  if (mi::launch(beam_select_kernel<T, WIDE>, dim3(a.stretches, a.R + 1), dim3(THREADS), smem, stream, a) != cudaSuccess)
    return mi_fail("beam_select: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  MI_LAUNCH_OK("beam_select");
  return 0;
}

}  // namespace

// Tiles of a block's stretch: as many as leave BLOCKS_WANTED blocks an SM (two fit at a time), a block a row at least.
static int beam_tiles(int R, int V) {
  const long long tiles = ((long long)V + TILE - 1) / TILE, wanted = (long long)BLOCKS_WANTED * mi::sm_count();
  const long long stretches = R > 0 ? (wanted + R - 1) / R : 1;
  return (int)((tiles + stretches - 1) / (stretches < tiles ? stretches : tiles));
}

// 64-bit words of scratch for R rows of V logits and n places.
MI_API long long mi_beam_select_words(int R, int V, int n) {
  const long long per = (long long)TILE * beam_tiles(R, V);
  return (long long)R * ((V + per - 1) / per) * (n + 1) + 2ll * R + 1;
}

// scratch: mi_beam_select_words words, 8-byte aligned; arrivals: one zero word a request and one more, left zero.
MI_API int mi_beam_select(int* tokens, int* parents, float* scores, const void* logits, int dtype, const float* cum, const int* start, void* scratch,
                          int* arrivals, int R, int V, int requests, int n, cudaStream_t stream) {
  MI_REQUIRE(R >= 0 && V > 0 && requests >= 0 && n >= 1 && n <= MAX_BEST, "beam_select: bad sizes R=%d V=%d requests=%d n=%d (n is at most %d)", R, V, requests, n, MAX_BEST);
  MI_REQUIRE(V <= 1 << 30, "beam_select: a vocabulary of %d", V);
  MI_REQUIRE(R < 65535, "beam_select: %d rows are too many for one launch", R);
  MI_REQUIRE(dtype == MI_F32 || dtype == MI_BF16, "beam_select: unknown type of logits");
  if (requests == 0) return 0;
  const int size = dtype == MI_F32 ? 4 : 2, tiles = beam_tiles(R, V);
  const long long per = (long long)TILE * tiles, stretches = (V + per - 1) / per;
  MI_REQUIRE((long long)R * stretches * n <= 0x7fffffffll, "beam_select: %lld candidates of %d rows are too many for one launch", stretches * n, R);
  Args a{tokens, parents, scores, logits, cum, start, nullptr, nullptr, nullptr, arrivals, R, V, requests, n, (int)stretches, tiles};
  a.best = (uint64_t*)scratch;
  a.sums = (float2*)(a.best + (size_t)R * a.stretches * n);
  a.norm = (double2*)(((uintptr_t)(a.sums + (size_t)R * a.stretches) + 15) / 16 * 16);
  const bool wide = (uintptr_t)logits % 16 == 0 && (long long)V * size % 16 == 0;
  if (dtype == MI_F32) return wide ? launch<float, true>(a, stream) : launch<float, false>(a, stream);
  return wide ? launch<__nv_bfloat16, true>(a, stream) : launch<__nv_bfloat16, false>(a, stream);
}
