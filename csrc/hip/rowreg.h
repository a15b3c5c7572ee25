// One row of logits in a block's registers: 16-B vectors from the first
// aligned address on, R per thread, and the up to 7 + 7 elements before and
// after them one per thread ("edge").  Rows start at any element.
#pragma once

#include "common.h"

template <typename T, int TH, int R>
struct RowRegs {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int CAP = TH * R * V;      // longest row that fits
  static_assert(TH >= 64, "edge slots");
  uint4 v[R];
  float edge;
  int head, nv, ej;      // elements before the vectors, vectors, this thread's edge element or -1

  // T's -inf: fills the slots past the row (exp gives 0, comparisons lose)
  static __device__ __forceinline__ uint32_t fill() {
    return sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  }

  __device__ __forceinline__ void load(const T* p, int n, int tid) {
    const int mis = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
    head = mis < n ? mis : n;
    nv = (n - head) / V;
    const int tail0 = head + nv * V, nt = n - tail0;
    const uint4* q = reinterpret_cast<const uint4*>(p + head);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = tid + r * TH;
      if (i < nv) v[r] = q[i];
      else v[r] = make_uint4(fill(), fill(), fill(), fill());
    }
    ej = tid < head ? tid : (tid >= 32 && tid - 32 < nt ? tail0 + tid - 32 : -1);
    edge = ej >= 0 ? ld1(p + ej) : -INFINITY;
  }

  // Unpacks the vectors of one pass over the row.  The shift and the mask are
  // opaque to the compiler, which would otherwise keep every bf16 of the row
  // unpacked, in twice the registers, from one pass to the next.
  struct Unpack {
    uint32_t shift, mask;
    __device__ __forceinline__ Unpack() {
      if constexpr (sizeof(T) == 2) {
        asm volatile("s_mov_b32 %0, 16" : "=s"(shift));
        asm volatile("s_mov_b32 %0, 0xffff0000" : "=s"(mask));
      }
    }
    __device__ __forceinline__ float operator()(const uint4& u, int e) const {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
      else return __uint_as_float((e & 1) ? (w[e >> 1] & mask) : (w[e >> 1] << shift));
    }
  };

  // f(element, value) over this thread's slots; slots past the row have value
  // -inf and an element number beyond every row's
  template <typename F>
  __device__ __forceinline__ void each(int tid, F f) const {
    vecs(tid, [&](int, int j, const float* z) {
#pragma unroll
      for (int e = 0; e < V; ++e) f(j + e, z[e]);
    });
    f(ej >= 0 ? ej : 0x7fffffff, edge);
  }

  // f(r, first element, V values) over this thread's vectors
  template <typename F>
  __device__ __forceinline__ void vecs(int tid, F f) const {
    const Unpack get;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r > 0 && r * TH >= nv) break;           // the same for all threads
      const int i = tid + r * TH;
      const int j = i < nv ? head + i * V : 0x7ffffff0;
      float z[V];
#pragma unroll
      for (int e = 0; e < V; ++e) z[e] = get(v[r], e);
      f(r, j, z);
    }
  }
};
