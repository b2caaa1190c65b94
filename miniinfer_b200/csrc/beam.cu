// Beam search's selection: the n best continuations of a request over all of its beams and the vocabulary.
//
//   score(r, v) = cum[r] + x[r, v] - log(sum_u exp(x[r, u]))          r: a row of logits, one per beam
//
// The best score comes first; of equal ones the lower row, in a row the larger logit and then the lower token.  A score that is no number
// or minus infinity is no candidate (a forbidden token, a beam that has ended, a row with a logit that is no number); places that no
// candidate fills get token -1, parent -1, score -inf.
//
// One launch, one pass over the logits.  A block has a tile of a row in registers: its maximum m and sum of exp(x - m), and its n best
// logits - a row's order does not depend on its normaliser.  The last block of a request to finish puts the pieces together: the rows'
// normalisers, then the n best of (tiles x n) candidates.
//
// The n best of a tile without sorting it: a thread's best of its own values; every warp sorts its 32 (by value, then lower token); with
// 8 warps the ceil(n / 8)-th of each of them makes 8 ceil(n / 8) >= n values, so the least of those eight bounds the n-th best from
// below.  What is not below it - twice n, as a rule - is collected in shared memory and ranked by counting.  Should more come
// than there is room for (a tile of which a warp has only poor values), the n-th best of the 256 threads' is counted out, which bounds the
// number by n times a thread's values.
//
// Float32 holds a value and a piece's sum; normalisers and scores are made in 64 bits, so that candidates of different beams, which may lie
// closer than a float32 of their size tells apart, are put in the right order.  The score that is handed out is rounded once.
#include "attention_scores.cuh"
#include "common.cuh"

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_BEST = 128;
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

struct Args {
  int *tokens, *parents;         // [requests, n]
  float* scores;
  const void* logits;            // [R, V]
  const float* cum;              // [R]
  const int* start;              // [requests + 1]
  float2* sums;                  // [R, tiles]: maximum, sum of exp(x - maximum)
  uint64_t* best;                // [R, tiles, n]: keys, 0 where there is none
  double2* norm;                 // [R]: the maximum, cum minus the log of the sum
  int* arrivals;                 // [requests], zero; left zero
  int R, V, requests, n, tiles;
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

template <typename T, int ITEMS, bool WIDE>
__device__ __forceinline__ void load_tile(float (&v)[ITEMS], const T* row, int begin, int V) {
  constexpr int PER = 16 / sizeof(T);      // values of a wide load
  if constexpr (WIDE) {
    uint4 raw[ITEMS / PER];
#pragma unroll
    for (int j = 0; j < ITEMS / PER; ++j) {
      const int at = begin + (j * THREADS + (int)threadIdx.x) * PER;
      raw[j] = at < V ? __ldg(reinterpret_cast<const uint4*>(row + at)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < ITEMS / PER; ++j) {
      const int at = begin + (j * THREADS + (int)threadIdx.x) * PER;
      const T* x = reinterpret_cast<const T*>(&raw[j]);
#pragma unroll
      for (int e = 0; e < PER; ++e) v[j * PER + e] = at < V ? mi::to_float(x[e]) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int at = begin + j * THREADS + (int)threadIdx.x;
      v[j] = at < V ? mi::to_float(row[at]) : -INFINITY;
    }
  }
}
// The token of a thread's j-th value; they rise with j.
template <typename T, bool WIDE>
__device__ __forceinline__ int token_at(int begin, int j) {
  constexpr int PER = WIDE ? 16 / sizeof(T) : 1;
  return begin + (j / PER * THREADS + (int)threadIdx.x) * PER + j % PER;
}

// A candidate of the last step: the score's image, then the lower row, then the row's key.
struct Candidate {
  uint64_t score, key;
  int row;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  if (a.score != b.score) return a.score > b.score;
  if (a.row != b.row) return a.row < b.row;
  return a.key > b.key;
}

// Puts a request's pieces together; by the whole block.  `pool`: shared memory for `room` candidates.
__device__ void finish(const Args& a, int request, Candidate* pool, int room, uint64_t* scratch /* THREADS */, int* count) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = max(a.start[request], 0), r1 = min(a.start[request + 1], a.R);
  for (int r = r0 + warp; r < r1; r += WARPS) {      // normalisers: a warp a row
    float m = -INFINITY;
    for (int t = lane; t < a.tiles; t += 32) m = fmaxf(m, __ldcg(&a.sums[(size_t)r * a.tiles + t].x));
    m = mi::warp_max(m);
    double s = 0.0;
    for (int t = lane; t < a.tiles; t += 32) {
      const float2 p = __ldcg(&a.sums[(size_t)r * a.tiles + t]);
      if (p.y != 0.f) s += (double)p.y * exp((double)p.x - (double)m);      // (a tile without weight has no maximum either)
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(FULL, s, o);
    if (lane == 0) a.norm[r] = make_double2((double)m, (double)a.cum[r] - log(s));
  }
  __syncthreads();
  const long long total = (long long)(r1 - r0) * a.tiles * a.n, per_row = (long long)a.tiles * a.n;
  const uint64_t* keys = a.best + (size_t)r0 * per_row;
  auto candidate = [&](long long i) {
    Candidate c{0, __ldcg(keys + i), r0 + (int)(i / per_row)};
    if (c.key) {
      // the maximum first: of a row of lowest values (-3.4e38), nothing else would be left of the score
      const double s = ((double)value_of(c.key) - a.norm[c.row].x) + a.norm[c.row].y;
      if (s > -INFINITY) c.score = rising64(s);      // (also false where the score is no number)
    }
    return c;
  };
  // a bound of the n-th best, as for a tile; images alone, so that candidates equal to it stay
  uint64_t mine = 0;
  for (long long i = threadIdx.x; i < total; i += THREADS) {
    const Candidate c = candidate(i);
    mine = c.score > mine ? c.score : mine;
  }
  const uint64_t sorted = sorted_in_warp(mine);
  if (lane == (a.n + WARPS - 1) / WARPS - 1) scratch[warp] = sorted;
  if (threadIdx.x == 0) *count = 0;
  __syncthreads();
  uint64_t bound = scratch[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) bound = scratch[w] < bound ? scratch[w] : bound;
  for (long long i = threadIdx.x; i < total; i += THREADS) {
    const Candidate c = candidate(i);
    if (c.score && c.score >= bound) {
      const int at = atomicAdd(count, 1);
      if (at < room) pool[at] = c;
    }
  }
  __syncthreads();
  const int got = *count;
  int *tokens = a.tokens + (size_t)request * a.n, *parents = a.parents + (size_t)request * a.n;
  float* scores = a.scores + (size_t)request * a.n;
  if (got <= room) {
    for (int i = threadIdx.x; i < got; i += THREADS) {
      const Candidate c = pool[i];
      int rank = 0;
      for (int j = 0; j < got; ++j) rank += before(pool[j], c);
      if (rank < a.n) {
        tokens[rank] = token_of(c.key);
        parents[rank] = c.row;
        scores[rank] = (float)score_of(c.score);
      }
    }
    for (int i = got + threadIdx.x; i < a.n; i += THREADS) {
      tokens[i] = parents[i] = -1;
      scores[i] = -INFINITY;
    }
    return;
  }
  // more candidates than there is room for (many equal scores, or all of the best in few threads' share): one place at a time
  Candidate last{~0ull, ~0ull, -1};
  for (int place = 0; place < a.n; ++place) {
    Candidate b{0, 0, 0x7fffffff};
    for (long long i = threadIdx.x; i < total; i += THREADS) {
      const Candidate c = candidate(i);
      if (c.score && before(last, c) && before(c, b)) b = c;
    }
    __syncthreads();
    pool[threadIdx.x] = b;
    __syncthreads();
    for (int o = THREADS / 2; o > 0; o >>= 1) {
      if (threadIdx.x < o && before(pool[threadIdx.x + o], pool[threadIdx.x])) pool[threadIdx.x] = pool[threadIdx.x + o];
      __syncthreads();
    }
    last = pool[0];
    if (threadIdx.x == 0) {
      const bool live = last.score != 0;
      tokens[place] = live ? token_of(last.key) : -1;
      parents[place] = live ? last.row : -1;
      scores[place] = live ? (float)score_of(last.score) : -INFINITY;
    }
    if (!last.score) last = Candidate{0, 0, 0x7fffffff};      // none left: nor for the places behind
  }
}

template <typename T, int ITEMS, bool WIDE>
__global__ void __launch_bounds__(THREADS)
beam_select_kernel(Args a) {
  constexpr int ROOM = MAX_BEST * ITEMS > 4096 ? 4096 : MAX_BEST * ITEMS;      // n of the threads' bests are not below the counted bound: n * ITEMS values
  static_assert(MAX_BEST * ITEMS <= ROOM, "the counted bound has to fit");
  __shared__ __align__(16) uint64_t pool[ROOM];
  __shared__ uint64_t scratch[THREADS];
  __shared__ float s_red[WARPS + 1];
  __shared__ int s_count, s_request, s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.y, tile = blockIdx.x;
  mi::grid_dependency_sync();
  if (row == a.R) {      // requests without rows: nobody else answers for them
    for (int q = tile * WARPS + warp; q < a.requests; q += gridDim.x * WARPS)
      if (max(a.start[q], 0) >= min(a.start[q + 1], a.R))
        for (int i = lane; i < a.n; i += 32) {
          a.tokens[(size_t)q * a.n + i] = a.parents[(size_t)q * a.n + i] = -1;
          a.scores[(size_t)q * a.n + i] = -INFINITY;
        }
    return;
  }
  const int begin = tile * THREADS * ITEMS;
  float v[ITEMS];
  load_tile<T, ITEMS, WIDE>(v, reinterpret_cast<const T*>(a.logits) + (size_t)row * a.V, begin, a.V);
  if (warp == 0) {
    const int q = request_of(a, row);
    if (lane == 0) {
      s_request = q;
      s_count = 0;
    }
  }
  // the thread's best, the tile's maximum and sum
  float top = -INFINITY;
  int at = 0;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    if (v[j] > top) {
      top = v[j];
      at = j;
    }
  float m = mi::warp_max(top);
  const uint64_t mine = key_of(top, token_at<T, WIDE>(begin, at));
  const uint64_t sorted = sorted_in_warp(mine);
  if (lane == 0) s_red[warp] = m;
  if (lane == (a.n + WARPS - 1) / WARPS - 1) scratch[warp] = sorted;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_red[w]);
  uint64_t bound = scratch[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) bound = scratch[w] < bound ? scratch[w] : bound;
  const float off = m == -INFINITY ? 0.f : m;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) sum[j & 3] += mi::ex2_fast((v[j] - off) * 1.4426950408889634f);
  const float total = mi::warp_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
  // what is not below the bound
  auto collect = [&]() {
    const float bv = bound ? value_of(bound) : -INFINITY;
    if (top >= bv) {
#pragma unroll
      for (int j = 0; j < ITEMS; ++j)
        if (v[j] >= bv) {
          const uint64_t key = key_of(v[j], token_at<T, WIDE>(begin, j));
          if (key && key >= bound) {
            const int i = atomicAdd(&s_count, 1);
            if (i < ROOM) pool[i] = key;
          }
        }
    }
    __syncthreads();
  };
  collect();
  if (s_count > ROOM) {      // the n-th best of the threads' bests, counted out
    __syncthreads();
    scratch[threadIdx.x] = mine;
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    int rank = 0;
    for (int t = 0; t < THREADS; ++t) rank += scratch[t] > mine;
    __syncthreads();
    if (rank == a.n - 1 && mine) scratch[0] = mine;      // (keys differ, but for those of threads without a value; more than ROOM values fill n threads)
    __syncthreads();
    bound = scratch[0];
    collect();
  }
  const int got = min(s_count, ROOM);
  uint64_t* best = a.best + ((size_t)row * a.tiles + tile) * a.n;
  for (int i = threadIdx.x; i < got; i += THREADS) {
    const uint64_t key = pool[i];
    int rank = 0;
    for (int j = 0; j < got; ++j) rank += pool[j] > key;
    if (rank < a.n) best[rank] = key;
  }
  for (int i = got + threadIdx.x; i < a.n; i += THREADS) best[i] = 0;
  if (lane == 0) s_red[warp] = total;
  __threadfence();      // the tile's best, before the block counts as arrived
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = s_red[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) t += s_red[w];
    a.sums[(size_t)row * a.tiles + tile] = make_float2(m, t);
    s_last = 0;
    const int q = s_request;
    if (q >= 0) {
      __threadfence();
      const int blocks = (min(a.start[q + 1], a.R) - max(a.start[q], 0)) * a.tiles;
      if (atomicAdd(&a.arrivals[q], 1) == blocks - 1) {
        a.arrivals[q] = 0;      // ready for the next launch
        s_last = 1;
      }
    }
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  finish(a, s_request, reinterpret_cast<Candidate*>(pool), ROOM * (int)sizeof(uint64_t) / (int)sizeof(Candidate), scratch, &s_count);
}

template <typename T, int ITEMS>
int launch(const Args& a, bool wide, cudaStream_t stream) {
  auto kernel = wide ? beam_select_kernel<T, ITEMS, true> : beam_select_kernel<T, ITEMS, false>;
  if (mi::launch(kernel, dim3(a.tiles, a.R + 1), dim3(THREADS), 0, stream, a) != cudaSuccess)
    return mi_fail("beam_select: launch failed: %s", cudaGetErrorString(cudaGetLastError()));
  MI_LAUNCH_OK("beam_select");
  return 0;
}

}  // namespace

// Logits of a block's tile.  A thread's 32 values are what keeps HBM busy; where that leaves less than two blocks an SM, 8.
static int beam_items(int R, int V) { return (long long)R * ((V + THREADS * 32 - 1) / (THREADS * 32)) >= 2 * mi::sm_count() ? 32 : 8; }

// 64-bit words of scratch for R rows of V logits and n places.
MI_API long long mi_beam_select_words(int R, int V, int n) {
  const int per = THREADS * beam_items(R, V);
  return (long long)R * ((V + per - 1) / per) * (n + 1) + 2ll * R + 1;
}

// scratch: mi_beam_select_words words, 8-byte aligned; arrivals: one zero word a request, left zero.
MI_API int mi_beam_select(int* tokens, int* parents, float* scores, const void* logits, int dtype, const float* cum, const int* start, void* scratch,
                          int* arrivals, int R, int V, int requests, int n, cudaStream_t stream) {
  MI_REQUIRE(R >= 0 && V > 0 && requests >= 0 && n >= 1 && n <= MAX_BEST, "beam_select: bad sizes R=%d V=%d requests=%d n=%d (n is at most %d)", R, V, requests, n, MAX_BEST);
  MI_REQUIRE(R < 65535, "beam_select: %d rows are too many for one launch", R);
  MI_REQUIRE(dtype == MI_F32 || dtype == MI_BF16, "beam_select: unknown type of logits");
  if (requests == 0) return 0;
  const int items = beam_items(R, V), size = dtype == MI_F32 ? 4 : 2, per = THREADS * items;
  Args a{tokens, parents, scores, logits, cum, start, nullptr, nullptr, nullptr, arrivals, R, V, requests, n, (V + per - 1) / per};
  a.best = (uint64_t*)scratch;
  a.sums = (float2*)(a.best + (size_t)R * a.tiles * n);
  a.norm = (double2*)(((uintptr_t)(a.sums + (size_t)R * a.tiles) + 15) / 16 * 16);
  const bool wide = (uintptr_t)logits % 16 == 0 && (long long)V * size % 16 == 0;
  if (dtype == MI_F32) return items == 32 ? launch<float, 32>(a, wide, stream) : launch<float, 8>(a, wide, stream);
  return items == 32 ? launch<__nv_bfloat16, 32>(a, wide, stream) : launch<__nv_bfloat16, 8>(a, wide, stream);
}
