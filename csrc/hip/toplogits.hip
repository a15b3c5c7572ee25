// The K largest logits of every row and their classes, in descending order,
// equal values by class number (ops.loss.top_logits).
//
// Order: NaN before everything, +0 equal to -0, otherwise by value; equal
// values lowest class first.  With key(z) an unsigned integer that increases
// with that order, element j is the 64-bit number key << 32 | ~j: all distinct,
// so "the K largest" has one answer and any way of finding them gives it.
//
// A row is read once, into the registers of a block.  Selection by filter:
// each wave finds the ceil(K / waves)-th largest of its threads' maxima, the
// smallest of these bounds is at most the K-th largest element, and only the
// elements that reach it (some tens for K = 10, some hundreds for K = 200) go
// to LDS to be ordered.  Rows that defeat the filter -- NaN, or so many equal
// values that the candidates overflow -- are narrowed by a radix search over
// the 64-bit numbers instead: exact for any input, slower.
//
// What bounds it: the one read of the logits.  Rows longer than a block's
// registers, and long rows that are too few to fill the chip, are cut into
// chunks; a chunk hands on its candidates unordered (or its K largest, if those
// are too many) and top_merge selects among them in the same way.
#include "nodes_api.h"
#include "rowreg.h"

constexpr int TOP_KMAX = 1024;
constexpr int TOP_CAND = 4096;       // most candidates in LDS

struct TopP {
  const void* z;
  int64_t ldz;
  void* val;             // [G][B][K]
  int* idx;
  uint64_t* list;        // chunked: [rows][chunks][room]
  int B, G, N, K, chunks, chunk, room;
  int cand;              // candidates in LDS
};

__device__ __forceinline__ uint32_t key_of(float z) {
  uint32_t u = __float_as_uint(z);
  if (z != z) return 0xffffffffu;
  if (z == 0.f) u = 0;
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ uint64_t number_of(float z, int j) {
  return ((uint64_t)key_of(z) << 32) | (uint32_t)~j;
}

// x and y in descending (else ascending) order
__device__ __forceinline__ void exchange(uint64_t& x, uint64_t& y, bool desc) {
  if ((x < y) == desc) {
    const uint64_t t = x;
    x = y;
    y = t;
  }
}

// s[0 .. n) in descending order; n a power of two from 256, all TH threads.  Two
// steps of the network in one pass: a thread takes the 4 numbers that exchange at
// distances j and j / 2 (256 rows of 1000 fp32 logits in order: one step a pass
// 24.3 us, two 16.3).  At distances of up to 128 a wave's groups of 4 stay inside
// its own 256 numbers, pass after pass: those passes need no barrier of the block.
template <int TH>
__device__ __forceinline__ void bitonic(uint64_t* s, int n) {
  __syncthreads();
  for (int i = threadIdx.x; i < n / 4; i += TH) {       // sequences of 2, then of 4
    uint64_t* p = s + 4 * i;
    uint64_t x0 = p[0], x1 = p[1], x2 = p[2], x3 = p[3];
    const bool desc = (i & 1) == 0;
    exchange(x0, x1, true);
    exchange(x2, x3, false);
    exchange(x0, x2, desc);
    exchange(x1, x3, desc);
    exchange(x0, x1, desc);
    exchange(x2, x3, desc);
    p[0] = x0;
    p[1] = x1;
    p[2] = x2;
    p[3] = x3;
  }
  bool wide = false;
  for (int k = 8, steps = 3; k <= n; k <<= 1, ++steps) {
    // an odd number of steps begins with one alone
    bool two = (steps & 1) == 0;
    for (int j = k >> 1; j > 0; j >>= two ? 2 : 1, two = true) {
      if (wide || j > 128) {
        __syncthreads();
      } else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
      wide = j > 128;
      const int h = j >> 1;
      for (int i = threadIdx.x; i < n / 4; i += TH) {
        const int a = 4 * i - 3 * (i & (h - 1));
        const bool desc = (a & k) == 0;
        uint64_t x0 = s[a], x1 = s[a + h], x2 = s[a + 2 * h], x3 = s[a + 3 * h];
        exchange(x0, x2, desc);
        exchange(x1, x3, desc);
        if (two) {
          exchange(x0, x1, desc);
          exchange(x2, x3, desc);
        }
        s[a] = x0;
        s[a + h] = x1;
        s[a + 2 * h] = x2;
        s[a + 3 * h] = x3;
      }
    }
  }
  __syncthreads();
}

// The C numbers in s (room for the next power of two, above 256) in descending
// order to out(rank, number) for rank < K.
template <int TH, typename F>
__device__ __forceinline__ void ordered(uint64_t* s, int* rk, int C, int K, F out) {
  if (C <= 256) {
    // few: every number counts the larger ones; several threads share a number
    const int ce = (C + 1) & ~1;
    if (threadIdx.x == 0 && ce > C) s[C] = 0;
    int cp = 64;
    while (cp < C) cp <<= 1;
    if (cp > TH) cp = TH;
    const int parts = TH / cp;
    for (int i = threadIdx.x; i < C; i += TH) rk[i] = 0;
    __syncthreads();
    const int part = threadIdx.x / cp, len = (ce / 2 + parts - 1) / parts * 2;
    const int c0 = part * len, c1 = min(ce, c0 + len);
    for (int i = threadIdx.x & (cp - 1); i < C; i += cp) {
      const uint64_t me = s[i];
      int larger = 0;
#pragma unroll 4
      for (int c = c0; c < c1; c += 2) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(s + c);
        larger += (x.x > me ? 1 : 0) + (x.y > me ? 1 : 0);
      }
      atomicAdd(&rk[i], larger);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < C; i += TH)
      if (rk[i] < K) out(rk[i], s[i]);
    return;
  }
  int n = 512;
  while (n < C) n <<= 1;
  for (int i = C + threadIdx.x; i < n; i += TH) s[i] = 0;
  bitonic<TH>(s, n);
  for (int i = threadIdx.x; i < K; i += TH) out(i, s[i]);
}

// a lower bound (upper 16 bits: all of a bf16) of the kw-th largest of a wave's
// keys, kw <= 64
__device__ __forceinline__ uint32_t wave_bound(uint32_t mk, int kw) {
  uint32_t t = 0;
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t c = t | (1u << bit);
    if (__popcll(__ballot(mk >= c)) >= kw) t = c;
  }
  return t;
}

// the same of the K-th largest of a block's GR keys a thread; cnt: 16 zeros,
// ordered before by a barrier
template <int GR>
__device__ __forceinline__ uint32_t block_bound(const uint32_t* mk, int K, int* cnt) {
  uint32_t t = 0;
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t c = t | (1u << bit);
    int reach = 0;
#pragma unroll
    for (int q = 0; q < GR; ++q) reach += __popcll(__ballot(mk[q] >= c));
    if ((threadIdx.x & 63) == 0 && reach) atomicAdd(&cnt[bit - 16], reach);
    __syncthreads();
    if (cnt[bit - 16] >= K) t = c;
  }
  return t;
}

// Radix search for the K-th largest of number(0 .. n), 8 bits at a time from the
// top, until what reaches the prefix fits `room`; those go to cand.
template <int TH, typename F>
__device__ __noinline__ int radix_candidates(F number, int n, int K, uint64_t* cand, int room,
                                             int* hist, int* count) {
  const int tid = threadIdx.x;
  uint64_t prefix = 0;
  int above = 0;                       // elements above the prefix
  for (int sh = 56; sh >= 0; sh -= 8) {
    __syncthreads();
    for (int i = tid; i < 256; i += TH) hist[i] = 0;
    __syncthreads();
    for (int j = tid; j < n; j += TH) {
      const uint64_t x = number(j);
      if (sh == 56 || (x >> (sh + 8)) == (prefix >> (sh + 8)))
        atomicAdd(&hist[(int)(x >> sh) & 255], 1);
    }
    __syncthreads();
    // hist[d] = elements with the prefix and a digit >= d
    for (int o = 1; o < 256; o <<= 1) {
      int add[(256 + TH - 1) / TH];
#pragma unroll
      for (int i = 0; i < (256 + TH - 1) / TH; ++i) {
        const int d = tid + i * TH;
        add[i] = d + o < 256 ? hist[d + o] : 0;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < (256 + TH - 1) / TH; ++i) {
        const int d = tid + i * TH;
        if (d < 256) hist[d] += add[i];
      }
      __syncthreads();
    }
    // the largest digit that K elements reach
    int lo_d = 0, hi_d = 255;
    while (lo_d < hi_d) {
      const int mid = (lo_d + hi_d + 1) >> 1;
      if (above + hist[mid] >= K) lo_d = mid;
      else hi_d = mid - 1;
    }
    prefix |= (uint64_t)lo_d << sh;
    const int reach = above + hist[lo_d];
    if (reach <= room) break;
    if (lo_d < 255) above += hist[lo_d + 1];
  }
  __syncthreads();
  if (tid == 0) *count = 0;
  __syncthreads();
  for (int j = tid; j < n; j += TH) {
    const uint64_t x = number(j);
    if (x >= prefix) cand[atomicAdd(count, 1)] = x;
  }
  __syncthreads();
  return *count;
}

template <typename T, int TH, int R>
__global__ __launch_bounds__(TH) void top_rows(const TopP P) {
  constexpr int W = TH / 64, V = RowRegs<T, TH, R>::V, CAP = RowRegs<T, TH, R>::CAP;
  // keys a thread brings to the bound: one maximum, or for larger K the maxima of
  // 4 parts of its elements, or all of them where it has one vector
  constexpr int GR = R == 1 ? V : R >= 4 ? 4 : 1;
  constexpr bool SHORT = CAP <= 512;          // the whole row fits: no search is ever needed
  extern __shared__ __attribute__((aligned(16))) uint64_t cand[];
  __shared__ uint32_t bound[16];
  __shared__ int hist[SHORT ? 1 : 256], rk[256], cnt[16], count, nanflag;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / P.chunks, ch = blockIdx.x - row * P.chunks;
  const int g = row / P.B, b = row - g * P.B;
  const int lo = ch * P.chunk, n = min(P.chunk, P.N - lo);
  const T* zr = reinterpret_cast<const T*>(P.z) + (int64_t)b * P.ldz + (int64_t)g * P.N + lo;
  RowRegs<T, TH, R> regs;
  if (tid == 0) {
    count = 0;
    nanflag = 0;
  }
  if (tid < 16) cnt[tid] = 0;
  regs.load(zr, n, tid);
  const int K = min(P.K, n);
  const int kw = (K + W - 1) / W;
  __syncthreads();

  // maxima of GR groups of this thread's elements; NaN is only noted
  float m[GR];
#pragma unroll
  for (int q = 0; q < GR; ++q) m[q] = -INFINITY;
  bool nan = regs.edge != regs.edge;
  m[0] = fmaxf(m[0], regs.edge);
  regs.vecs(tid, [&](int r, int, const float* z) {
    float t = -INFINITY;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      nan |= z[e] != z[e];
      if constexpr (R == 1) m[e] = fmaxf(m[e], z[e]);
      else t = fmaxf(t, z[e]);
    }
    if constexpr (R > 1) m[r % GR] = fmaxf(m[r % GR], t);
  });
  if (__ballot(nan) && lane == 0) nanflag = 1;
  // A small share per wave: the smallest of the waves' own bounds, which lets
  // some more through but needs one barrier.  A large one: the block's bound,
  // found with a barrier a bit (K 256 of 1000: 258 candidates, not all 1000).
  uint32_t lim;
  if (kw <= 16) {
#pragma unroll
    for (int q = 1; q < GR; ++q) m[0] = fmaxf(m[0], m[q]);
    const uint32_t t = wave_bound(key_of(m[0]), kw);
    if (lane == 0) bound[wave] = t;
    __syncthreads();
    lim = bound[0];
#pragma unroll
    for (int w = 1; w < W; ++w) lim = min(lim, bound[w]);
  } else {
    uint32_t mk[GR];
#pragma unroll
    for (int q = 0; q < GR; ++q) mk[q] = key_of(m[q]);
    lim = block_bound<GR>(mk, K, cnt);
  }
  const bool has_nan = nanflag != 0;
  int C = P.cand + 1;
  if (!has_nan || SHORT) {
    // a bound below -inf's key takes every element; so does a short row with NaN
    const float fl = has_nan || lim <= 0x007fffffu ? -INFINITY : key_value(lim);
    auto push = [&](int j, float z) {
      if (!(z < fl) && j < n) {
        const int at = atomicAdd(&count, 1);
        if (at < P.cand) cand[at] = number_of(z, lo + j);
      }
    };
    regs.vecs(tid, [&](int, int j, const float* z) {
      bool any = false;
#pragma unroll
      for (int e = 0; e < V; ++e) any |= !(z[e] < fl);
      if (__ballot(any)) {
#pragma unroll
        for (int e = 0; e < V; ++e) push(j + e, z[e]);
      }
    });
    push(regs.ej >= 0 ? regs.ej : 0x7fffffff, regs.edge);
    __syncthreads();
    C = count;
  }
  if constexpr (!SHORT) {
    // from memory: one of the last levels of cache has the row
    if (C > P.cand)
      C = radix_candidates<TH>([=](int j) { return number_of(ld1(zr + j), lo + j); }, n, K, cand,
                               P.cand, hist, &count);
  }
  if (P.chunks == 1) {
    T* val = reinterpret_cast<T*>(P.val) + (int64_t)row * P.K;
    int* idx = P.idx + (int64_t)row * P.K;
    ordered<TH>(cand, rk, C, K, [&](int k, uint64_t x) {
      const int j = (int)~(uint32_t)x;
      idx[k] = j;
      val[k] = zr[j];
    });
  } else {
    uint64_t* out = P.list + (int64_t)blockIdx.x * P.room;
    int filled = C;
    if (C <= P.room) {
      for (int k = tid; k < C; k += TH) out[k] = cand[k];
    } else {
      ordered<TH>(cand, rk, C, K, [&](int k, uint64_t x) { out[k] = x; });
      filled = K;
    }
    for (int k = filled + tid; k < P.room; k += TH) out[k] = 0;
  }
}

// the chunks' lists of a row (zeros are no entries) to its result
constexpr int TM_TH = 1024;
template <typename T>
__global__ __launch_bounds__(TM_TH) void top_merge(const TopP P) {
  constexpr int GR = 4;
  __shared__ __attribute__((aligned(16))) uint64_t cand[TOP_CAND];
  __shared__ int hist[256], rk[256], cnt[16], count;
  const int tid = threadIdx.x, row = blockIdx.x;
  const int n = P.chunks * P.room, K = P.K;
  const uint64_t* src = P.list + (int64_t)row * n;
  if (tid == 0) count = 0;
  if (tid < 16) cnt[tid] = 0;
  uint32_t mk[GR] = {0, 0, 0, 0};
  for (int i = tid; i < n; i += GR * TM_TH) {
#pragma unroll
    for (int q = 0; q < GR; ++q) {
      const int j = i + q * TM_TH;
      if (j < n) mk[q] = max(mk[q], (uint32_t)(src[j] >> 32));
    }
  }
  __syncthreads();
  uint32_t lim = block_bound<GR>(mk, K, cnt);
  if (lim == 0) lim = 1;                       // zeros stay out
  for (int i = tid; i < n; i += TM_TH) {
    const uint64_t x = src[i];
    if ((uint32_t)(x >> 32) >= lim) {
      const int at = atomicAdd(&count, 1);
      if (at < TOP_CAND) cand[at] = x;
    }
  }
  __syncthreads();
  int C = count;
  if (C > TOP_CAND)
    C = radix_candidates<TM_TH>([=](int j) { return src[j]; }, n, K, cand, TOP_CAND, hist, &count);
  const int g = row / P.B, b = row - g * P.B;
  const T* zr = reinterpret_cast<const T*>(P.z) + (int64_t)b * P.ldz + (int64_t)g * P.N;
  T* val = reinterpret_cast<T*>(P.val) + (int64_t)row * K;
  int* idx = P.idx + (int64_t)row * K;
  ordered<TM_TH>(cand, rk, C, K, [&](int k, uint64_t x) {
    const int j = (int)~(uint32_t)x;
    idx[k] = j;
    val[k] = zr[j];
  });
}

template <typename T>
static int top_chunk(int64_t rows, int N, int K) {
  constexpr int V = 16 / (int)sizeof(T);
  int c = N;
  if (N > 1024 * 16 * V) c = 1024 * 16 * V;
  // few rows: shorter chunks put more of the chip to work
  const int few = K <= 256 ? 256 * 8 * V : 512 * 16 * V;
  if (rows < 128 && N > few && few < c) c = few;
  return c;
}

static inline bool top_sizes(int B, int G, int N, int K) {
  return B > 0 && G > 0 && N > 0 && N < 0x7ffffff0 && K > 0 && K <= N && K <= TOP_KMAX &&
         (int64_t)B * G <= 0x7fffffff;
}

template <typename T>
static int top_threads(int chunk) {
  constexpr int V = 16 / (int)sizeof(T);
  return chunk <= 64 * V ? 64 : chunk <= 256 * 8 * V ? 256 : chunk <= 512 * 16 * V ? 512 : 1024;
}

static inline int top_room(int K) { return K < 32 ? 64 : 2 * K; }

// 64-bit numbers of workspace, -1 for sizes out of range
template <typename T>
static int64_t top_ws(int B, int G, int N, int K) {
  if (!top_sizes(B, G, N, K)) return -1;
  const int64_t rows = (int64_t)B * G;
  const int c = top_chunk<T>(rows, N, K);
  const int64_t chunks = (N + c - 1) / c;
  if (!grid_fits(rows * chunks, top_threads<T>(c)) || !grid_fits(rows, chunks > 1 ? TM_TH : 1)) return -1;
  return chunks > 1 ? rows * chunks * top_room(K) : 0;
}

CER_API int64_t cer_top_ws(int B, int G, int N, int K, int is_bf16) {
  return is_bf16 ? top_ws<bf16_t>(B, G, N, K) : top_ws<float>(B, G, N, K);
}

template <typename T>
static int top_launch(const T* z, int64_t ldz, T* val, int* idx, int B, int G, int N, int K,
                      uint64_t* ws, int64_t ws_n, hipStream_t st) {
  const int64_t need = top_ws<T>(B, G, N, K);
  if (need < 0 || ws_n < need || !z || !val || !idx || ldz < (int64_t)G * N)
    return (int)hipErrorInvalidValue;
  const int64_t rows = (int64_t)B * G;
  TopP P = {};
  P.z = z; P.ldz = ldz; P.val = val; P.idx = idx;
  P.B = B; P.G = G; P.N = N; P.K = K;
  P.chunk = top_chunk<T>(rows, N, K);
  P.chunks = (N + P.chunk - 1) / P.chunk;
  P.list = ws;
  P.room = top_room(K);
  const int grid = (int)(rows * P.chunks);
  const int n = P.chunk;
  constexpr int V = 16 / (int)sizeof(T);
  // room for a multiple of K, a power of two for the sort; little LDS leaves more
  // blocks on a CU
  P.cand = n <= 64 * V ? 512 : K <= 256 ? 1024 : TOP_CAND;
#define CER_TOP(TH, R) top_rows<T, TH, R><<<grid, TH, P.cand * sizeof(uint64_t), st>>>(P)
  // (top_threads knows these)
  if (n <= 64 * V) CER_TOP(64, 1);
  else if (n <= 256 * V) CER_TOP(256, 1);
  else if (n <= 256 * 4 * V) CER_TOP(256, 4);
  else if (n <= 256 * 8 * V) CER_TOP(256, 8);
  else if (n <= 512 * 8 * V) CER_TOP(512, 8);
  else if (n <= 512 * 16 * V) CER_TOP(512, 16);
  else CER_TOP(1024, 16);
#undef CER_TOP
  if (P.chunks > 1) top_merge<T><<<(int)rows, TM_TH, 0, st>>>(P);
  return (int)hipGetLastError();
}

CER_API CER_TOP_LOGITS(cer_top_logits) {
  return top_launch((const bf16_t*)z, ldz, (bf16_t*)val, idx, B, G, N, K, (uint64_t*)ws, ws_n, st);
}

CER_API CER_TOP_LOGITS(cer_top_logits_f32) {
  return top_launch((const float*)z, ldz, (float*)val, idx, B, G, N, K, (uint64_t*)ws, ws_n, st);
}
