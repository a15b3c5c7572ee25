// Cross-entropy on labels mixed with distillation from a teacher known by its
// top logits, G packed configurations (ops.loss.distill_ce).
//
// Row (g, b) with logits z[N], label y or none, teacher entries (i_k, v_k):
//
//   hard = lse(z) - z_y
//   p = softmax_k(v_k / tau),  q = softmax(z / tau)
//   soft = sum_k p_k (log p_k - log q_{i_k})
//   row  = (1 - alpha) hard + alpha tau^2 soft,   loss_g = mean_b row
//   dz_j = [(1 - alpha)(softmax(z)_j - [j = y])
//           + alpha tau (q_j - sum_{k: i_k = j} p_k)] dloss_g / B
//
// An entry with a negative class or a value of -inf is absent; a row without
// entries has no soft term, one without a label no hard term, and a term that
// is absent or has weight zero is not computed at all (what the row holds then
// does not matter).  A class or label >= N makes its row NaN.
//
// What bounds it: the logits are read once and the gradient written once.  The
// row stays in registers between the maximum, the two sums and the gradient
// (distill_row); rows beyond what a block's registers hold are cut into slices
// (distill_stats, distill_rows, distill_grad) and read twice.  All statistics
// are fp32, the sums over the batch fp64 in a fixed order: no atomics.
#include "nodes_api.h"
#include "rowreg.h"

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KMAX = 1024;     // teacher entries of a row

struct DistP {
  const void* z;
  int64_t ldz;                 // elements from row b to row b + 1
  const int* labels;           // [G][B]
  const void* val;             // teacher values: config, row strides; entries adjacent
  int val_f32;                 // fp32 values (else bf16), whatever the logits are
  int64_t val_gs, val_bs;
  const int* idx;
  int64_t idx_gs, idx_bs;
  const float* alpha;          // [G], or null: alpha0
  const float* tau;            // [G], or null: tau0
  float alpha0, tau0;
  const float* dloss;          // [G] or null (ones)
  void* dz;                    // [B][G N] or null
  float* rowloss;              // [G][B]
  int* rowhit;                 // bit 0 top-1, bit 1 top-5
  float* stats;                // [G][B][4]: max, sum at 1, sum at tau, rank (or null)
  float* part;                 // [slices][G][B][4]
  int B, G, N, K, slices, slice;
};

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^(k (z - m)); the difference first: a row (or slice) of the type's lowest
// value has m k beyond the type
struct Expo {
  float k, m;
  __device__ __forceinline__ Expo(float k_, float m_) : k(k_), m(m_) {}
  __device__ __forceinline__ float operator()(float z) const { return ex2((z - m) * k); }
};

// sums of three values over the block
template <int TH>
__device__ __forceinline__ void block_sum3(float& a, float& b, float& c, float* sm) {
  a = warp_sum(a);
  b = warp_sum(b);
  c = warp_sum(c);
  if constexpr (TH > 64) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 0) {
      sm[w] = a;
      sm[16 + w] = b;
      sm[32 + w] = c;
    }
    __syncthreads();
    a = b = c = 0.f;
#pragma unroll
    for (int i = 0; i < TH / 64; ++i) {
      a += sm[i];
      b += sm[16 + i];
      c += sm[32 + i];
    }
  }
}

template <int TH>
__device__ __forceinline__ float block_max1(float a, float* sm) {
  a = warp_max(a);
  if constexpr (TH > 64) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 0) sm[w] = a;
    __syncthreads();
    a = sm[0];
#pragma unroll
    for (int i = 1; i < TH / 64; ++i) a = fmaxf(a, sm[i]);
  }
  return a;
}

// which terms a row has, and their weights
struct RowW {
  bool hard, soft, bad;
  float a, tau, itau;
};

// The teacher's entries of a row: classes and, with `probs`, probabilities into
// LDS (absent ones as class -1, probability 0); sum_k p_k log p_k in plogp.
template <int TH>
__device__ __forceinline__ RowW teacher(const DistP& P, int g, int b, int lab, int* ti, float* tp,
                                        float* sm, float& plogp, int& nthere) {
  RowW w;
  w.a = P.alpha ? P.alpha[g] : P.alpha0;
  w.tau = P.tau ? P.tau[g] : P.tau0;
  w.itau = 1.f / w.tau;
  const int64_t v0 = g * P.val_gs + b * P.val_bs;
  const int* ix = P.idx + g * P.idx_gs + b * P.idx_bs;
  float mx = -INFINITY, there = 0.f, bad = lab >= P.N ? 1.f : 0.f;
  const bool want = w.a != 0.f;
  for (int k = threadIdx.x; k < P.K; k += TH) {
    int i = want ? ix[k] : -1;
    float x = -INFINITY;
    if (i >= 0)
      x = P.val_f32 ? reinterpret_cast<const float*>(P.val)[v0 + k]
                    : bf2f(reinterpret_cast<const bf16_t*>(P.val)[v0 + k]);
    if (i >= P.N) bad = 1.f;
    if (x == -INFINITY || i >= P.N) i = -1;
    ti[k] = i;
    tp[k] = i >= 0 ? x : 0.f;
    if (i >= 0) {
      mx = fmaxf(mx, x);
      there += 1.f;
    }
  }
  float dummy = 0.f;
  mx = block_max1<TH>(mx, sm);
  block_sum3<TH>(there, bad, dummy, sm);
  nthere = (int)there;
  w.bad = bad > 0.f;
  w.soft = nthere > 0;
  w.hard = lab >= 0 && w.a != 1.f;
  plogp = 0.f;
  if (w.soft) {
    float s = 0.f, t = 0.f, u = 0.f;
    for (int k = threadIdx.x; k < P.K; k += TH) {
      if (ti[k] >= 0) {
        const float x = (tp[k] - mx) * w.itau;
        const float e = ex2(x * LOG2E);
        s += e;
        if (e > 0.f) t += e * x;
        tp[k] = e;
      }
    }
    block_sum3<TH>(s, t, u, sm);
    const float is = 1.f / s;
    for (int k = threadIdx.x; k < P.K; k += TH) tp[k] *= is;
    plogp = t * is - logf(s);
  }
  return w;
}

// sum_k p_k log q_{i_k}: every thread gets it
template <typename T, int TH>
__device__ __forceinline__ float cross(const DistP& P, const T* zr, const int* ti, const float* tp,
                                       const RowW& w, float mx, float s2, float* sm) {
  float c = 0.f, d0 = 0.f, d1 = 0.f;
  const float l2 = logf(s2);
  for (int k = threadIdx.x; k < P.K; k += TH)
    if (ti[k] >= 0 && tp[k] > 0.f) c += tp[k] * ((ld1(zr + ti[k]) - mx) * w.itau - l2);
  block_sum3<TH>(c, d0, d1, sm);
  return c;
}

// thread 0: the row's loss and hits
__device__ __forceinline__ void row_result(const DistP& P, int g, int b, int lab, const RowW& w,
                                           float plogp, float c, float mx, float s1, float zl,
                                           float cnt) {
  float row = 0.f;
  if (w.hard) row += (1.f - w.a) * (logf(s1) + (mx - zl));
  if (w.soft) row += w.a * w.tau * w.tau * (plogp - c);
  if (w.bad) row = NAN;
  const int64_t o = (int64_t)g * P.B + b;
  P.rowloss[o] = row;
  // two classes have no fifth place: every row counts, as in softmax_ce
  const bool lb = lab >= 0 && lab < P.N;
  P.rowhit[o] = (lb && cnt < 1.f ? 1 : 0) | ((P.N > 2 ? (lb && cnt < 5.f) : true) ? 2 : 0);
}

// coefficients of a row's gradient: before the entries it is
// c1 2^((z - mx) log2 e) + c2 2^((z - mx) k2).  The factors stay out of the exponents,
// whose rounding is relative to their size: log2(c / s) of -16 to -32 there made
// every term 2^-20 wrong (fp32 8192 x 1000: 2.9e-7 from 64 bits, so 0.5e-7).
struct GradW {
  float mx, k2, c1, c2, ch, cs;
  bool hard, soft, one;
};

__device__ __forceinline__ GradW grad_weights(const DistP& P, const RowW& w, int g, float mx,
                                              float s1, float s2) {
  GradW q;
  float sc = (P.dloss ? P.dloss[g] : 1.f) / (float)P.B;
  if (w.bad) sc = NAN;
  q.hard = w.hard || w.bad;
  q.soft = w.soft;
  q.k2 = LOG2E * w.itau;
  q.ch = (1.f - w.a) * sc;
  q.cs = w.a * w.tau * sc;
  q.mx = mx;
  // at tau = 1 both terms have one exponential
  q.one = q.hard && q.soft && w.tau == 1.f;
  q.c1 = (q.one ? q.ch + q.cs : q.ch) / s1;
  q.c2 = q.cs / s2;
  return q;
}

template <bool HARD, bool SOFT>
__device__ __forceinline__ float grad_of(const GradW& q, float z) {
  const float x = z - q.mx;
  float d = 0.f;
  if (HARD) d = q.c1 * ex2(x * LOG2E);
  if (SOFT) d = HARD ? fmaf(q.c2, ex2(x * q.k2), d) : q.c2 * ex2(x * q.k2);
  return d;
}

__device__ __forceinline__ float grad_base(const GradW& q, float z) {
  return q.hard ? (q.soft && !q.one ? grad_of<true, true>(q, z) : grad_of<true, false>(q, z))
                : (q.soft ? grad_of<false, true>(q, z) : 0.f);
}

// The label's and the teacher's classes in [lo, hi): written whole, after the
// rest of the row (the caller's barrier orders the two).  A class that is named
// several times gets the sum of its entries in their order, from each of them.
template <typename T, int TH>
__device__ __forceinline__ void grad_entries(const DistP& P, const GradW& q, const T* zr, T* dr,
                                             const int* ti, const float* tp, int lab, int lo,
                                             int hi) {
  const int n = P.K + 1;
  for (int k = threadIdx.x; k < n; k += TH) {
    const bool is_lab = k == P.K;
    const int j = is_lab ? (q.hard ? lab : -1) : (q.soft ? ti[k] : -1);
    if (j < lo || j >= hi) continue;
    float d = grad_base(q, ld1(zr + j));
    if (q.hard && j == lab) d -= q.ch;
    if (q.soft) {
      float p = 0.f;
      for (int i = 0; i < P.K; ++i) p += ti[i] == j ? tp[i] : 0.f;
      d = fmaf(-q.cs, p, d);
    }
    st1(dr + j, d);
  }
}

// the gradient's rows need not have the logits' alignment
typedef uint32_t u32x4_a __attribute__((ext_vector_type(4), aligned(2)));

template <typename T, int TH, int R, typename F>
__device__ __forceinline__ void write_row(const RowRegs<T, TH, R>& row, T* dr, F f) {
  constexpr int V = RowRegs<T, TH, R>::V;
  row.vecs(threadIdx.x, [&](int r, int, const float* z) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (V == 4) w[e] = __float_as_uint(f(z[e]));
      else w[e] = cvt_pk_bf16(f(z[2 * e]), f(z[2 * e + 1]));
    }
    const int i = threadIdx.x + r * TH;
    if (i < row.nv)
      *reinterpret_cast<u32x4_a*>(dr + row.head + (int64_t)i * V) = u32x4_a{w[0], w[1], w[2], w[3]};
  });
  if (row.ej >= 0) st1(dr + row.ej, f(row.edge));
}

template <typename T, int TH, int R>
__device__ __forceinline__ void grad_row(const RowRegs<T, TH, R>& row, const GradW& q, T* dr) {
  if (!q.hard && !q.soft)
    write_row(row, dr, [&](float) { return 0.f; });
  else if (q.hard && q.soft && !q.one)
    write_row(row, dr, [&](float z) { return grad_of<true, true>(q, z); });
  else if (q.hard)
    write_row(row, dr, [&](float z) { return grad_of<true, false>(q, z); });
  else
    write_row(row, dr, [&](float z) { return grad_of<false, true>(q, z); });
}

// maximum, both sums and the label's rank (exact up to 4, at least 5 beyond) of
// the elements in `row`, which start at class j0 of the logits row; all threads
// get them.  A whole row of -inf has sums of NaN, a SLICE of nothing but -inf sums
// of zero.
template <typename T, int TH, int R, bool SLICE>
__device__ __forceinline__ void row_stats(const RowRegs<T, TH, R>& row, int j0, int lab, float zl,
                                          bool hard, bool soft, float itau, float* sm, float& mx,
                                          float& s1, float& s2, float& cnt) {
  constexpr int V = RowRegs<T, TH, R>::V;
  float m = row.edge;
  int before = 0;
  if (lab >= 0) {
    // the maximum, and how many come before the label: counted a wave at a time
    // in scalar registers, until a wave has seen the five that put the label
    // behind both places (4096 x 49999 bf16, random labels: 220 -> 205 us); equal
    // values are looked at only where there are any
    const int l = lab - j0;
    row.vecs(threadIdx.x, [&](int, int j, const float* z) {
#pragma unroll
      for (int e = 0; e < V; ++e) m = fmaxf(m, z[e]);
      if (before < 5) {
        uint64_t eq = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          before += __popcll(__ballot(z[e] > zl));
          eq |= __ballot(z[e] == zl);
        }
        if (eq) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            before += __popcll(__ballot((z[e] == zl) & (j + e < l)));
        }
      }
    });
    const int je = row.ej >= 0 ? row.ej : 0x7fffffff;
    before += __popcll(__ballot((row.edge > zl) | ((row.edge == zl) & (je < l))));
  } else {
    row.each(threadIdx.x, [&](int, float z) { m = fmaxf(m, z); });
  }
  mx = block_max1<TH>(m, sm);
  s1 = s2 = 0.f;
  cnt = (threadIdx.x & 63) == 0 ? (float)before : 0.f;
  const float mm = SLICE && mx == -INFINITY ? 0.f : mx;
  const Expo q1(LOG2E, mm), q2(LOG2E * itau, mm);
  if (hard && soft && itau != 1.f) {
    row.each(threadIdx.x, [&](int, float z) {
      s1 += q1(z);
      s2 += q2(z);
    });
  } else if (hard || itau == 1.f) {
    row.each(threadIdx.x, [&](int, float z) { s1 += q1(z); });
    s2 = s1;                     // used where the soft term is there: tau is 1 then
  } else if (soft) {
    row.each(threadIdx.x, [&](int, float z) { s2 += q2(z); });
  }
  block_sum3<TH>(s1, s2, cnt, sm);
}

template <typename T, int TH, int R>
__global__ __launch_bounds__(TH) void distill_row(const DistP P) {
  __shared__ int ti[KMAX];
  __shared__ float tp[KMAX];
  __shared__ float sm[48];
  const int b = blockIdx.x, g = blockIdx.y;
  const T* zr = reinterpret_cast<const T*>(P.z) + (int64_t)b * P.ldz + (int64_t)g * P.N;
  RowRegs<T, TH, R> row;
  row.load(zr, P.N, threadIdx.x);
  const int lab = P.labels[(int64_t)g * P.B + b];
  const float zl = lab >= 0 && lab < P.N ? ld1(zr + lab) : 0.f;
  float plogp, mx, s1, s2, cnt;
  int nthere;
  const RowW w = teacher<TH>(P, g, b, lab, ti, tp, sm, plogp, nthere);
  row_stats<T, TH, R, false>(row, 0, lab, zl, w.hard, w.soft, w.itau, sm, mx, s1, s2, cnt);
  const float c = w.soft ? cross<T, TH>(P, zr, ti, tp, w, mx, s2, sm) : 0.f;
  if (threadIdx.x == 0) {
    row_result(P, g, b, lab, w, plogp, c, mx, s1, zl, cnt);
    if (P.stats) {
      float* s = P.stats + ((int64_t)g * P.B + b) * 4;
      s[0] = mx;
      s[1] = s1;
      s[2] = s2;
    }
  }
  if (P.dz) {
    const GradW q = grad_weights(P, w, g, mx, s1, s2);
    T* dr = reinterpret_cast<T*>(P.dz) + (int64_t)b * P.G * P.N + (int64_t)g * P.N;
    grad_row<T, TH, R>(row, q, dr);
    __syncthreads();
    grad_entries<T, TH>(P, q, zr, dr, ti, tp, lab, 0, P.N);
  }
}

// slices of long rows: 256 threads x R vectors
constexpr int SL_TH = 256, SL_R = 8;

template <typename T>
__global__ __launch_bounds__(SL_TH) void distill_stats(const DistP P) {
  __shared__ float sm[48];
  const int b = blockIdx.x / P.slices, s = blockIdx.x - b * P.slices, g = blockIdx.y;
  const T* zr = reinterpret_cast<const T*>(P.z) + (int64_t)b * P.ldz + (int64_t)g * P.N;
  const int lo = s * P.slice, n = min(P.slice, P.N - lo);
  RowRegs<T, SL_TH, SL_R> row;
  row.load(zr + lo, n, threadIdx.x);
  const int lab = P.labels[(int64_t)g * P.B + b];
  const float zl = lab >= 0 && lab < P.N ? ld1(zr + lab) : 0.f;
  float mx, s1, s2, cnt;
  row_stats<T, SL_TH, SL_R, true>(row, lo, lab, zl, true, true, 1.f / (P.tau ? P.tau[g] : P.tau0), sm, mx, s1, s2, cnt);
  if (threadIdx.x == 0) {
    float* p = P.part + (((int64_t)s * P.G + g) * P.B + b) * 4;
    p[0] = mx;
    p[1] = s1;
    p[2] = s2;
    p[3] = cnt;
  }
}

template <typename T>
__global__ __launch_bounds__(SL_TH) void distill_rows(const DistP P) {
  __shared__ int ti[KMAX];
  __shared__ float tp[KMAX];
  __shared__ float sm[48];
  const int b = blockIdx.x, g = blockIdx.y;
  const T* zr = reinterpret_cast<const T*>(P.z) + (int64_t)b * P.ldz + (int64_t)g * P.N;
  const int lab = P.labels[(int64_t)g * P.B + b];
  float plogp;
  int nthere;
  const RowW w = teacher<SL_TH>(P, g, b, lab, ti, tp, sm, plogp, nthere);
  // join the slices in their order; one of nothing but -inf brings its sums
  // (zero, or NaN where it holds NaN) as they are, unless the whole row is
  float mx = -INFINITY, s1 = 0.f, s2 = 0.f, cnt = 0.f;
  const int64_t st = (int64_t)P.G * P.B * 4;
  const float* p = P.part + ((int64_t)g * P.B + b) * 4;
  for (int s = 0; s < P.slices; ++s) mx = fmaxf(mx, p[s * st]);
  for (int s = 0; s < P.slices; ++s) {
    const float m = p[s * st], x = m - mx;
    const bool none = m == -INFINITY && mx != -INFINITY;
    s1 += p[s * st + 1] * (none ? 1.f : ex2(x * LOG2E));
    s2 += p[s * st + 2] * (none ? 1.f : ex2(x * LOG2E * w.itau));
    cnt += p[s * st + 3];
  }
  const float c = w.soft ? cross<T, SL_TH>(P, zr, ti, tp, w, mx, s2, sm) : 0.f;
  if (threadIdx.x == 0) {
    const float zl = lab >= 0 && lab < P.N ? ld1(zr + lab) : 0.f;
    row_result(P, g, b, lab, w, plogp, c, mx, s1, zl, cnt);
    float* q = P.stats + ((int64_t)g * P.B + b) * 4;
    q[0] = mx;
    q[1] = s1;
    q[2] = s2;
  }
}

template <typename T, int TH, int R>
__global__ __launch_bounds__(TH) void distill_grad(const DistP P) {
  __shared__ int ti[KMAX];
  __shared__ float tp[KMAX];
  __shared__ float sm[48];
  const int b = blockIdx.x / P.slices, s = blockIdx.x - b * P.slices, g = blockIdx.y;
  const int64_t z0 = (int64_t)g * P.N;
  const T* zr = reinterpret_cast<const T*>(P.z) + (int64_t)b * P.ldz + z0;
  T* dr = reinterpret_cast<T*>(P.dz) + (int64_t)b * P.G * P.N + z0;
  const int lo = s * P.slice, n = min(P.slice, P.N - lo);
  RowRegs<T, TH, R> row;
  row.load(zr + lo, n, threadIdx.x);
  const int lab = P.labels[(int64_t)g * P.B + b];
  float plogp;
  int nthere;
  const RowW w = teacher<TH>(P, g, b, lab, ti, tp, sm, plogp, nthere);
  const float* st = P.stats + ((int64_t)g * P.B + b) * 4;
  const GradW q = grad_weights(P, w, g, st[0], st[1], st[2]);
  grad_row<T, TH, R>(row, q, dr + lo);
  __syncthreads();
  grad_entries<T, TH>(P, q, zr, dr, ti, tp, lab, lo, lo + n);
}

// per configuration: mean loss, and acc += (sum of row losses, top-1, top-5, B)
template <int TH>
__global__ __launch_bounds__(TH) void distill_sum(const float* __restrict__ rowloss,
                                                  const int* __restrict__ rowhit,
                                                  float* __restrict__ loss,
                                                  float* __restrict__ acc, int B) {
  constexpr int W = TH / 64;
  __shared__ double sd[W];
  __shared__ int s1[W], s5[W];
  const int g = blockIdx.x, t = threadIdx.x;
  double s = 0.0;
  int h1 = 0, h5 = 0;
#pragma unroll 4
  for (int b = t; b < B; b += TH) {
    s += (double)rowloss[(int64_t)g * B + b];
    const int h = rowhit[(int64_t)g * B + b];
    h1 += h & 1;
    h5 += h >> 1;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o);
    h1 += __shfl_xor(h1, o);
    h5 += __shfl_xor(h5, o);
  }
  if ((t & 63) == 0) {
    sd[t >> 6] = s;
    s1[t >> 6] = h1;
    s5[t >> 6] = h5;
  }
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < W; ++w) {
      s += sd[w];
      h1 += s1[w];
      h5 += s5[w];
    }
    loss[g] = (float)(s / (double)B);
    acc[g * 4 + 0] += (float)s;
    acc[g * 4 + 1] += (float)h1;
    acc[g * 4 + 2] += (float)h5;
    acc[g * 4 + 3] += (float)B;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename T>
static int64_t slice_of(int N) {
  // longest row of distill_row: 1024 threads x 16 vectors
  return N <= RowRegs<T, 1024, 16>::CAP ? 0 : RowRegs<T, SL_TH, SL_R>::CAP;
}

// Threads and vectors of the block for a row of N.  Few waves with long rows
// rather than many with short ones: the row's reductions are barriers, and
// blocks of 256 leave several of them on a CU (8192 x 16000 bf16: 512 x 8 253 us,
// 256 x 8 150 us; 4096 x 30000: 512 x 8 186 us, 256 x 16 141 us).  26 vectors are the
// most that three such blocks can hold on a CU (166 of 168 registers a lane); with
// more, two fit, and 512 threads are better.  us, unit gradient, 4096 rows of
//   bf16:     33000  40000  49999  53000  54000  60000  65536
//   256 x 26    152    167    202    211
//   512 x 16    179    197    231    231    237    251    261
//   256 x 32    184    205    241    245    250    268    281
//   fp32:     16500  20000  24999  26500  27000  30000  32768
//   256 x 26    136    156    190    198
//   512 x 16    152    167    197    203    208    225    233
//   256 x 32    153    172    205    212    217    230    241
#define CER_ROW_DISPATCH(T, N, LAUNCH)                  \
  do {                                                  \
    constexpr int V_ = 16 / sizeof(T);                  \
    if ((N) <= 64 * V_) LAUNCH(64, 1);                  \
    else if ((N) <= 256 * V_) LAUNCH(256, 1);           \
    else if ((N) <= 256 * 3 * V_) LAUNCH(256, 3);       \
    else if ((N) <= 256 * 8 * V_) LAUNCH(256, 8);       \
    else if ((N) <= 256 * 16 * V_) LAUNCH(256, 16);     \
    else if ((N) <= 256 * 26 * V_) LAUNCH(256, 26);     \
    else if ((N) <= 512 * 16 * V_) LAUNCH(512, 16);     \
    else LAUNCH(1024, 16);                              \
  } while (0)

static inline int row_threads(int N, int v) {       // of CER_ROW_DISPATCH and the slices
  return N <= 64 * v ? 64 : N <= 256 * 26 * v ? 256 : N <= 512 * 16 * v ? 512 : N <= 1024 * 16 * v ? 1024 : SL_TH;
}

template <typename T>
static bool dist_ok(const DistP& P) {
  return P.z && P.labels && cer_distill_ws(P.B, P.G, P.N, sizeof(T) == 2) >= 0 && P.K >= 0 && P.K <= KMAX && (P.K == 0 || (P.val && P.idx)) &&
         P.ldz >= (int64_t)P.G * P.N;
}

template <typename T>
static int launch_grad(DistP P, hipStream_t st) {
  const int64_t sl = slice_of<T>(P.N);
  P.slice = sl ? (int)sl : P.N;
  P.slices = (P.N + P.slice - 1) / P.slice;
  const dim3 grid(P.slices * P.B, P.G);
  if (sl) {
    distill_grad<T, SL_TH, SL_R><<<grid, SL_TH, 0, st>>>(P);
  } else {
#define CER_LG(TH, R) distill_grad<T, TH, R><<<grid, TH, 0, st>>>(P)
    CER_ROW_DISPATCH(T, P.N, CER_LG);
#undef CER_LG
  }
  return (int)hipGetLastError();
}

template <typename T>
static int dist_fwd(DistP P, float* loss, float* acc, int64_t ws_floats, float* ws,
                    hipStream_t st) {
  if (!dist_ok<T>(P) || !loss || !acc || !ws || !P.stats)
    return (int)hipErrorInvalidValue;
  const int64_t rows = (int64_t)P.G * P.B;
  const int64_t sl = slice_of<T>(P.N);
  P.slices = sl ? (int)((P.N + sl - 1) / sl) : 0;
  if (ws_floats < rows * (2 + 4 * (int64_t)P.slices)) return (int)hipErrorInvalidValue;
  P.rowloss = ws;
  P.rowhit = reinterpret_cast<int*>(ws + rows);
  P.part = ws + 2 * rows;
  if (sl) {
    P.slice = (int)sl;
    distill_stats<T><<<dim3(P.slices * P.B, P.G), SL_TH, 0, st>>>(P);
    distill_rows<T><<<dim3(P.B, P.G), SL_TH, 0, st>>>(P);
    if (P.dz) {
      const int rc = launch_grad<T>(P, st);
      if (rc) return rc;
    }
  } else {
    const dim3 grid(P.B, P.G);
#define CER_LR(TH, R) distill_row<T, TH, R><<<grid, TH, 0, st>>>(P)
    CER_ROW_DISPATCH(T, P.N, CER_LR);
#undef CER_LR
  }
  // one block a configuration: 4096 rows 8.8 us with 256 threads, 4.6 with 1024; 32
  // rows 1.9 us either way
  if (P.B > 512) distill_sum<1024><<<P.G, 1024, 0, st>>>(P.rowloss, P.rowhit, loss, acc, P.B);
  else distill_sum<256><<<P.G, 256, 0, st>>>(P.rowloss, P.rowhit, loss, acc, P.B);
  return (int)hipGetLastError();
}

static DistP dist_params(const void* z, int64_t ldz, const int* labels, const void* val,
                         int val_f32, int64_t val_gs, int64_t val_bs, const int* idx, int64_t idx_gs,
                         int64_t idx_bs, const float* alpha, float alpha0, const float* tau,
                         float tau0, const float* dloss, float* stats, void* dz, int B, int G, int N, int K) {
  DistP P = {};
  P.z = z; P.ldz = ldz; P.labels = labels;
  P.val = val; P.val_f32 = val_f32; P.val_gs = val_gs; P.val_bs = val_bs;
  P.idx = idx; P.idx_gs = idx_gs; P.idx_bs = idx_bs;
  P.alpha = alpha; P.alpha0 = alpha0; P.tau = tau; P.tau0 = tau0; P.dloss = dloss;
  P.stats = stats; P.dz = dz;
  P.B = B; P.G = G; P.N = N; P.K = K;
  return P;
}

// floats of workspace of a forward, -1 for sizes out of range
CER_API int64_t cer_distill_ws(int B, int G, int N, int is_bf16) {
  if (B <= 0 || G <= 0 || G > 65535 || N <= 0 || N >= 0x7ffffff0) return -1;
  const int64_t sl = is_bf16 ? slice_of<bf16_t>(N) : slice_of<float>(N);
  const int64_t slices = sl ? (N + sl - 1) / sl : 1;
  if (!grid_fits(slices * B, row_threads(N, is_bf16 ? 8 : 4))) return -1;
  return (int64_t)B * G * (2 + (sl ? 4 * ((N + sl - 1) / sl) : 0));
}

// fwd: loss [G], acc [G][4] +=, stats [G][B][4] for the backward; dz (or null): the
// gradient for dloss = 1.  bwd: dz from the forward's stats and dloss [G].
#define CER_DISTILL(T, F, B_)                                                                      \
  CER_API CER_DISTILL_FWD(F) {                                                                     \
    return dist_fwd<T>(dist_params(z, ldz, labels, val, val_f32, val_gs, val_bs, idx, idx_gs,      \
                                   idx_bs, alpha, alpha0, tau, tau0, nullptr, stats, dz, B, G, N,  \
                                   K),                                                             \
                       loss, acc, ws_floats, ws, st);                                              \
  }                                                                                                \
  CER_API CER_DISTILL_BWD(B_) {                                                                    \
    const DistP P = dist_params(z, ldz, labels, val, val_f32, val_gs, val_bs, idx, idx_gs, idx_bs, \
                                alpha, alpha0, tau, tau0, dloss, stats, dz, B, G, N, K);           \
    if (!dist_ok<T>(P) || !stats || !dz || !dloss) return (int)hipErrorInvalidValue;               \
    return launch_grad<T>(P, st);                                                                  \
  }
CER_DISTILL(bf16_t, cer_distill_fwd, cer_distill_bwd)
CER_DISTILL(float, cer_distill_fwd_f32, cer_distill_bwd_f32)
