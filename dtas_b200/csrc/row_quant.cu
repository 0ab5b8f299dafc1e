// Rows on their way into a low-bit projection: the residual's addition with the RMS norm, and rows
// brought to 8 bits with one scale each (int8 or e4m3, symmetric).  No counterpart in the reference.
//
//   add_rms_norm : h = x + res (res optional), r = 1 / sqrt(mean(h^2) + eps), y = h * r * weight
//   quantize     : y = x
//   8-bit result : scale = max|y| / Q, q = round(y * Q / max|y|), ties to even, Q = 448 (e4m3) or 127 (int8)
//
// r is the same for the whole row, so it cancels out of q: with u = h * weight,
// q = round(u * Q / max|u|) and scale = r * max|u| / Q.  The sum of squares and max|u| are therefore
// taken in ONE pass and meet in one exchange between the row's warps, where the formula as written
// would need two (first r, then the maximum of what r scales).
//
// h is held in fp32 between the reduction and the result: the norm sees the exact sum of two fp16
// values, not the rounded one that is stored as the new residual.
//
// Design: blockDim.x threads own a row and blockDim.y rows share a CTA; a thread holds CH chunks of VEC
// consecutive elements, all loads in flight at once.  The threads per row are the row's chunks over CH,
// rounded up to whole warps and not to a power of two, so that 11008 columns take 352 threads x 4 chunks
// and none idles.  Bound: HBM; every element is read once and written once.
// Rows of a length that is no multiple of eight start anywhere inside a 16-byte vector, but at the same place in
// every operand (EDGE): chunks are cut where the flat index is a multiple of eight, loads take whole vectors, and of the
// results only the first and the last chunk of a row, which it shares with its neighbours, go element by element.
// Where the rows fill the device several times over, CTAs stay and take rows in turn (row_quant_stream_kernel).
// Measured (HBM 6.57 TB/s): add_rms_norm fp16 to e4m3 [8192, 4096] 39.1 us, 6.0 TB/s; fp32 [4096, 4096] 34.5 us, 6.3 TB/s;
// [1, 4096] 1.8 us; quantize to e4m3 [2048, 11008] 15.0 us, 4.5 TB/s; [8192, 4096] 17.6 us, 5.7 TB/s.
#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"

namespace dtas {
namespace {

enum { Q_NORM = 0, Q_QUANT = 1 };
constexpr int kMaxThreads = 1024;
// Threads a CTA may have: what leaves a thread the registers for its chunks, and one warp more than a row of 16384 elements
// needs, for the one that starts inside a vector.
constexpr int max_threads(int vec, int ch) { return vec * ch > 16 ? 544 : kMaxThreads; }

struct RowArgs {
  const void* x;
  const void* res;       // optional (norm)
  const __half* weight;  // norm
  void* y;
  void* res_out;         // optional (norm)
  float* scale;          // 8-bit results
  int64_t m;
  int64_t n_cols;
  float eps;
};

template <typename T>
struct OutTraits;
template <>
struct OutTraits<__half> {
  static constexpr float kQ = 0.f;
};
template <>
struct OutTraits<int8_t> {
  static constexpr float kQ = 127.f;
};
template <>
struct OutTraits<__nv_fp8_e4m3> {
  static constexpr float kQ = 448.f;
};

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

// VEC consecutive elements of a row; VEC = 8 needs 16-byte aligned rows (32-byte pairs for fp32).
template <int VEC>
__device__ __forceinline__ void store_vec(__half* p, const float* v) {
  if constexpr (VEC == 8) {
    __stcs(reinterpret_cast<uint4*>(p), epi_pack8(v));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = __float2half_rn(v[i]);
  }
}
template <int VEC>
__device__ __forceinline__ void store_vec(float* p, const float* v) {
  if constexpr (VEC == 8) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(v[4], v[5], v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = v[i];
  }
}
__device__ __forceinline__ uint32_t pack4(const float* v, int8_t) {
  const int a = __float2int_rn(v[0]), b = __float2int_rn(v[1]), c = __float2int_rn(v[2]), d = __float2int_rn(v[3]);
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t pack4(const float* v, __nv_fp8_e4m3) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// |v| <= Q: a quotient by the maximum, exact for the maximum itself.
template <int VEC, typename OutT>
__device__ __forceinline__ void store_q(OutT* p, const float* v) {
  if constexpr (VEC == 8) {
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack4(v, OutT{}), pack4(v + 4, OutT{})));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (sizeof(OutT) == 1 && OutTraits<OutT>::kQ == 127.f)
        p[i] = (int8_t)__float2int_rn(v[i]);
      else
        reinterpret_cast<__nv_fp8_storage_t*>(p)[i] = __nv_cvt_float_to_fp8(v[i], __NV_SATFINITE, __NV_E4M3);
    }
  }
}

// VEC weights as loaded.  They go through the read-only path: stores of the residual cannot alias them, so all of them are
// under way with the rows instead of one behind each store.  A row that starts `lead` elements inside a vector needs eight
// weights out of two vectors, moved together by whole words and then by half a word.
template <int VEC, bool EDGE>
struct Weights {
  static constexpr int kN = VEC == 8 ? 4 : VEC;
  uint32_t r[kN];
  // the vector of p's elements b .. b + 7 (b a multiple of eight), zeros for those that are not in 0 .. n - 1; `some`: the
  // warp has a vector that is partly there
  static __device__ __forceinline__ void vector_at(const __half* p, int b, int n, bool some, uint32_t* w) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (b >= 0 && b + 8 <= n) v = __ldg(reinterpret_cast<const uint4*>(p + b));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    if (some && b >= 0 && b < n && b + 8 > n) {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = b + 2 * i < n ? __ldg(u + b + 2 * i) : 0u, hi = b + 2 * i + 1 < n ? __ldg(u + b + 2 * i + 1) : 0u;
        w[i] = lo | (hi << 16);
      }
    }
  }
  __device__ __forceinline__ void load(const __half* p, int e, int lead, int n) {
    bool some = false;
    if constexpr (EDGE) some = __any_sync(0xffffffffu, e + lead - 8 < n && e + lead + 8 > n);
    if (e >= n) return;
    if constexpr (VEC == 8 && !EDGE) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p + e));
      r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
    } else if constexpr (VEC == 8) {
      uint32_t w[8];
      vector_at(p, lead ? e + lead - 8 : -8, n, some, w);
      vector_at(p, e + lead, n, some, w + 4);
      const int by = 8 - lead;
      if (by & 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = w[i + 4];
      }
      if (by & 4) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
      }
      if (by & 2) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = by & 1 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < VEC; ++i) r[i] = __ldg(u + e + i);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (VEC == 8) {
      const __half2 h = *reinterpret_cast<const __half2*>(&r[i >> 1]);
      return i & 1 ? __high2float(h) : __low2float(h);
    } else {
      return __half2float(__ushort_as_half((unsigned short)r[i]));
    }
  }
};

// max that keeps a NaN, so that a row with one is not taken for a finite row
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum and maximum over the threads of one row (blockDim.x, a multiple of 32).  One exchange through shared
// memory for both; `ex` holds two floats per warp of the CTA.  Rows of one warp need no exchange.
__device__ __forceinline__ void row_reduce(float& sum, float& top, float2* ex) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  const int nw = blockDim.x >> 5;
  if (nw == 1) return;
  const int lane = threadIdx.x & 31;
  if (lane == 0) ex[threadIdx.y * nw + (threadIdx.x >> 5)] = make_float2(sum, top);
  __syncthreads();
  const float2 e = lane < nw ? ex[threadIdx.y * nw + lane] : make_float2(0.f, 0.f);
  sum = e.x;
  top = e.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
}

// Sixteen-byte vectors of eight consecutive elements as loaded.
template <typename T>
struct Raw8 {
  uint4 r[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void get(float* v) const {
    const T* e = reinterpret_cast<const T*>(r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  }
};

// Which of a thread's chunks are partly outside the row (EDGE) for some thread of the warp, a bit each.  Two warps of a
// row have one; the others branch around all that such chunks need.
template <int VEC, int CH, bool EDGE>
__device__ __forceinline__ unsigned edge_chunks(const int* at, int n) {
  unsigned edges = 0;
  if constexpr (EDGE) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (__any_sync(0xffffffffu, at[c] < n && (at[c] < 0 || at[c] + VEC > n))) edges |= 1u << c;
  }
  return edges;
}

// A thread's chunks of a row, asked for at once and looked at later: nothing between the loads of a row and of its residual
// waits for either.  A vector that is partly the row's is read whole all the same, for the rest of it is the rows' before
// and behind, and only what the tensor ends in (`room` elements from the row's first) goes by its elements.
template <int VEC, int CH, bool EDGE, typename T>
struct RowChunks {
  Raw8<T> raw[CH];
  __device__ __forceinline__ void load(const T* row, const int* at, int n, int room) {
    if constexpr (VEC == 8) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (at[c] < n && (!EDGE || at[c] + 8 <= room)) raw[c].load(row + at[c]);
    }
  }
  // chunk c, zeros where it lies outside the row
  __device__ __forceinline__ void get(const T* row, int c, int at, int n, int room, unsigned edges, float* v) const {
    if constexpr (VEC == 8) {
      if (at < n) {
        raw[c].get(v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
      }
      if (EDGE && (edges >> c & 1)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (at + i < 0 || at + i >= n) v[i] = 0.f;
          else if (at + 8 > room) v[i] = to_f32(row[at + i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = at < n ? to_f32(row[at + i]) : 0.f;
    }
  }
};
// The chunk whose first element is e back into the row; edge: some thread's is partly outside.
template <int VEC, typename T>
__device__ __forceinline__ void store_chunk(T* row, int e, int n, bool edge, const float* v) {
  if (!edge) {
    if (e < n) {
      if constexpr (sizeof(T) == 1) store_q<VEC>(row + e, v);
      else store_vec<VEC>(row + e, v);
    }
  } else if (e >= 0 && e + VEC <= n) {
    if constexpr (sizeof(T) == 1) store_q<VEC>(row + e, v);
    else store_vec<VEC>(row + e, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (e + i >= 0 && e + i < n) {
        if constexpr (sizeof(T) == 1) store_q<1>(row + e + i, v + i);
        else store_vec<1>(row + e + i, v + i);
      }
  }
}

// Elements on their way to 8 bits: v * Q / top, exact where fp32 can hold it, so that a value halfway between two 8-bit
// ones is just that, and goes to the even one.  (With v times a rounded Q / top such values fall to either side, and rows
// of fp16 numbers have some: about one element in 10^4.)  Q / top is held as hi + lo to some 44 bits, and v hi + (v lo) in a
// fused multiply-add is rounded once but for an error far below its half step.  hi need not be the nearest number to
// Q / top, so an approximate reciprocal does: lo is what hi leaves, (Q - hi top) / top with the difference exact.  By
// pairs, two elements to an instruction, this takes no longer than the single product did ([8192, 4096] to e4m3 17.7 us
// both ways).  `pre`, a power of two, keeps the factors of very small and very large rows in range.  A row of
// zeros gets q = 0; a row that holds an infinity or a NaN gets a NaN scale, and so stands for NaN whatever its q.
struct QuantMul {
  float pre, hi, lo;
};
__device__ __forceinline__ QuantMul quant_mul(float top, float q) {
  if (!(top > 0.f && top < INFINITY)) return {0.f, 0.f, 0.f};
  const float pre = top < 0x1p-40f ? 0x1p100f : (top > 0x1p100f ? 0x1p-60f : 1.f);
  const float t = top * pre, inv = epi_rcp(t), hi = q * inv;
  return {pre, hi, fmaf(-hi, t, q) * inv};
}
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
// VEC elements in place.
template <int VEC>
__device__ __forceinline__ void quant_values(const QuantMul& m, float* v) {
  if (m.pre != 1.f) {      // the same for the whole row
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] *= m.pre;
  }
  if constexpr (VEC == 1) {
    v[0] = fmaf(v[0], m.hi, __fmul_rn(v[0], m.lo));
  } else {
    const uint64_t hi = pair(m.hi, m.hi), lo = pair(m.lo, m.lo);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      uint64_t r = pair(v[i], v[i + 1]);
      asm("{\n\t.reg .b64 t;\n\tmul.rn.f32x2 t, %0, %2;\n\tfma.rn.f32x2 %0, %0, %1, t;\n\t}" : "+l"(r) : "l"(hi), "l"(lo));
      asm("mov.b64 {%0, %1}, %2;" : "=f"(v[i]), "=f"(v[i + 1]) : "l"(r));
    }
  }
}
__device__ __forceinline__ float quant_scale(float top, float r, float q) {
  return top < INFINITY ? (top * r) / q : __int_as_float(0x7fc00000);
}

// A row whose elements - for the norm, their sums with the residual - are in registers: its results.
template <int OP, typename InT, typename OutT, int VEC, int CH, bool EDGE>
__device__ __forceinline__ void finish_row(const RowArgs& a, int64_t row, bool live, int n, const int* at,
                                           unsigned edges, float (*v)[VEC], const Weights<VEC, EDGE>* wt, float2* ex) {
  constexpr bool kNorm = OP == Q_NORM;
  constexpr bool k8 = sizeof(OutT) == 1;
  const int64_t off = row * a.n_cols;
  float sum = 0.f, top = 0.f;
  if constexpr (kNorm) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum = fmaf(v[c][i], v[c][i], sum);
      if (a.res_out != nullptr) store_chunk<VEC>(static_cast<InT*>(a.res_out) + off, at[c], n, edges >> c & 1, v[c]);
      if (at[c] < n) {
        if constexpr (k8) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[c][i] *= wt[c].get(i);
        }
      }
    }
  }
  if constexpr (k8) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < VEC; ++i) top = max_nan(top, fabsf(v[c][i]));
  }
  row_reduce(sum, top, ex);
  if (!live) return;
  float r = 1.f;
  if constexpr (kNorm) r = 1.0f / sqrtf(sum / (float)n + a.eps);
  OutT* y = static_cast<OutT*>(a.y) + off;
  if constexpr (k8) {
    const QuantMul qm = quant_mul(top, OutTraits<OutT>::kQ);
    if (threadIdx.x == 0) a.scale[row] = quant_scale(top, r, OutTraits<OutT>::kQ);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      quant_values<VEC>(qm, v[c]);
      store_chunk<VEC>(y, at[c], n, edges >> c & 1, v[c]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float o[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = __fmul_rn(__fmul_rn(v[c][i], r), wt[c].get(i));
      store_chunk<VEC>(reinterpret_cast<__half*>(y), at[c], n, edges >> c & 1, o);
    }
  }
}

template <int OP, typename InT, typename OutT, int VEC, int CH, bool EDGE>
__global__ void __launch_bounds__(max_threads(VEC, CH)) row_quant_kernel(const RowArgs a) {
  __shared__ float2 ex[kMaxThreads / 32];
  constexpr bool kNorm = OP == Q_NORM;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.m;
  const int n = live ? (int)a.n_cols : 0;
  const int64_t off = (live ? row : 0) * a.n_cols;
  const int lead = EDGE ? (int)(off & (VEC - 1)) : 0;      // elements of its first chunk that are not the row's
  const InT* x = static_cast<const InT*>(a.x) + off;
  int at[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) at[c] = (c * blockDim.x + threadIdx.x) * VEC - lead;

  pdl_wait();
  pdl_launch_dependents();
  const unsigned edges = edge_chunks<VEC, CH, EDGE>(at, n);
  const int64_t behind = a.m * a.n_cols - off;      // elements from the row's first to the tensor's last
  const int room = behind < (1 << 30) ? (int)behind : 1 << 30;
  const InT* res = kNorm && a.res != nullptr ? static_cast<const InT*>(a.res) + off : nullptr;
  RowChunks<VEC, CH, EDGE, InT> rx, rr;
  rx.load(x, at, n, room);
  if (res != nullptr) rr.load(res, at, n, room);
  Weights<VEC, EDGE> wt[CH];
  if constexpr (kNorm) {
#pragma unroll
    for (int c = 0; c < CH; ++c) wt[c].load(a.weight, at[c], lead, n);
  }
  float v[CH][VEC];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    rx.get(x, c, at[c], n, room, edges, v[c]);
    if (res != nullptr) {
      float t[VEC];
      rr.get(res, c, at[c], n, room, edges, t);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[c][i] += t[i];
    }
  }
  finish_row<OP, InT, OutT, VEC, CH, EDGE>(a, row, live, n, at, edges, v, wt, ex);
}

// Many rows: the CTAs that fit on the device take rows in turn, and a row's loads are under way while the one before
// it is reduced and stored.  The weights stay in registers, but for rows that start elsewhere inside a vector each time.
template <int OP, typename InT, typename OutT, int CH, bool EDGE>
__global__ void __launch_bounds__(EDGE ? max_threads(8, 4) : 512) row_quant_stream_kernel(const RowArgs a) {
  __shared__ float2 ex[2][kMaxThreads / 32];       // in turn: a row's exchange cannot meet the one before it
  constexpr bool kNorm = OP == Q_NORM;
  struct Place {
    int n, lead, room;
    int64_t off;
  };
  auto place = [&](int64_t row) {
    Place p;
    p.n = row < a.m ? (int)a.n_cols : 0;
    p.off = (row < a.m ? row : 0) * a.n_cols;
    p.lead = EDGE ? (int)(p.off & 7) : 0;
    const int64_t behind = a.m * a.n_cols - p.off;
    p.room = behind < (1 << 30) ? (int)behind : 1 << 30;
    return p;
  };
  auto at_of = [&](const Place& p, int* at) {
#pragma unroll
    for (int c = 0; c < CH; ++c) at[c] = (c * blockDim.x + threadIdx.x) * 8 - p.lead;
  };
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t first = (int64_t)blockIdx.x * blockDim.y;
  const InT *xs = static_cast<const InT*>(a.x), *rs = kNorm ? static_cast<const InT*>(a.res) : nullptr;

  pdl_wait();
  pdl_launch_dependents();
  RowChunks<8, CH, EDGE, InT> rx, rr;
  auto fetch = [&](const Place& p) {
    int at[CH];
    at_of(p, at);
    rx.load(xs + p.off, at, p.n, p.room);
    if (rs != nullptr) rr.load(rs + p.off, at, p.n, p.room);
  };
  Place p = place(first + threadIdx.y);
  fetch(p);
  int at[CH];
  Weights<8, EDGE> wt[CH];
  for (int turn = 0; first < a.m; first += step, turn ^= 1) {
    const int64_t row = first + threadIdx.y;
    at_of(p, at);
    if (kNorm && (EDGE || first == (int64_t)blockIdx.x * blockDim.y)) {
#pragma unroll
      for (int c = 0; c < CH; ++c) wt[c].load(a.weight, at[c], p.lead, (int)a.n_cols);
    }
    const unsigned edges = edge_chunks<8, CH, EDGE>(at, p.n);
    float v[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      rx.get(xs + p.off, c, at[c], p.n, p.room, edges, v[c]);
      if (rs != nullptr) {
        float t[8];
        rr.get(rs + p.off, c, at[c], p.n, p.room, edges, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] += t[i];
      }
    }
    const Place next = place(row + step);
    fetch(next);
    finish_row<OP, InT, OutT, 8, CH, EDGE>(a, row, row < a.m, p.n, at, edges, v, wt, ex[turn]);
    p = next;
  }
}

// Rows longer than the registers of a CTA hold: one CTA per row, which passes over it twice (the second
// time out of L2).  Every element of the results is written by the thread that has just read its inputs,
// behind the only reduction, so results in place of inputs are fine here too.
template <int OP, typename InT, typename OutT>
__global__ void __launch_bounds__(kMaxThreads) row_quant_long_kernel(const RowArgs a) {
  __shared__ float2 ex[kMaxThreads / 32];
  constexpr bool kNorm = OP == Q_NORM;
  constexpr bool k8 = sizeof(OutT) == 1;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t off = (int64_t)blockIdx.x * a.n_cols;
  const InT* x = static_cast<const InT*>(a.x) + off;
  const InT* res = kNorm && a.res != nullptr ? static_cast<const InT*>(a.res) + off : nullptr;
  float sum = 0.f, top = 0.f;
  for (int64_t i = threadIdx.x; i < a.n_cols; i += blockDim.x) {
    float h = to_f32(x[i]);
    if (kNorm && res != nullptr) h += to_f32(res[i]);
    if constexpr (kNorm) {
      sum = fmaf(h, h, sum);
      if constexpr (k8) h *= __half2float(a.weight[i]);
    }
    if constexpr (k8) top = max_nan(top, fabsf(h));
  }
  row_reduce(sum, top, ex);
  float r = 1.f;
  if constexpr (kNorm) r = 1.0f / sqrtf(sum / (float)a.n_cols + a.eps);
  const QuantMul qm = quant_mul(top, OutTraits<OutT>::kQ);
  if (k8 && threadIdx.x == 0) a.scale[blockIdx.x] = quant_scale(top, r, OutTraits<OutT>::kQ);
  OutT* y = static_cast<OutT*>(a.y) + off;
  for (int64_t i = threadIdx.x; i < a.n_cols; i += blockDim.x) {
    float h = to_f32(x[i]);
    if (kNorm && res != nullptr) h += to_f32(res[i]);
    const float w = kNorm ? __half2float(a.weight[i]) : 1.f;
    if constexpr (kNorm) {
      if (a.res_out != nullptr) store_vec<1>(static_cast<InT*>(a.res_out) + off + i, &h);
    }
    if constexpr (k8) {
      float q = kNorm ? h * w : h;
      quant_values<1>(qm, &q);
      store_q<1>(y + i, &q);
    } else {
      const float o = __fmul_rn(__fmul_rn(h, r), w);
      store_vec<1>(reinterpret_cast<__half*>(y) + i, &o);
    }
  }
}

// ---- dispatch ------------------------------------------------------------------
struct RowPlan {
  int vec;       // 8, or 1 where an address rules out 16-byte vectors; 0: the long kernel
  int ch;        // chunks per thread
  int tpr;       // threads per row
  int rows;      // rows per CTA
  bool edge;     // rows that start inside a vector
  bool stream;   // row_quant_stream_kernel
};

inline RowPlan row_plan(int64_t m, int64_t n_cols, bool aligned, bool norm, bool wide) {   // wide: fp32 inputs
  RowPlan p{0, 0, 0, 0, false, false};
  p.vec = aligned ? 8 : 1;
  p.edge = aligned && n_cols % 8 != 0;
  const int64_t chunks = (n_cols + p.vec - 1) / p.vec + (p.edge ? 1 : 0);
  const int64_t most = aligned ? 8 * max_threads(8, 8) : 16 * max_threads(1, 16);
  if (chunks > most) {
    p.vec = 0;
    p.edge = false;
    p.tpr = kMaxThreads;
    p.rows = 1;
    return p;
  }
  if (!aligned) {
    p.ch = chunks <= 256 * 4 ? 4 : 16;
  } else if (p.edge && norm) {
    // What rows that start inside a vector need besides leaves room for fewer threads, so a thread has two chunks or more
    // sooner ([8192, 4097] fp16 to int8: 163 us with one, 71 with two, 113 with four; [255, 2561] 3.8, 4.0 and 7.1); from
    // 4352 columns on fp16 rows go in turn ([8192, 8191] 149 us, a row per CTA 197; [1, 16383] 6.3 and 8.1) and fp32 rows
    // take four ([8192, 8191] 183 us, with two 215; [255, 8191] 10.4 with two).
    if (chunks <= 544) {
      p.ch = m > 592 || chunks > 512 ? 2 : 1;
    } else if (!wide && chunks <= 4 * 544) {
      p.stream = true;
      p.ch = chunks <= 2 * 544 ? 2 : 4;
    } else {
      p.ch = m > 592 ? 4 : 2;
    }
  } else if (p.edge) {
    // [8192, 1025] to int8: two chunks 11.6 us, four 13.5; [8192, 4097] 32.8 and 29.7; [255, 11009] 5.8 and 4.2
    p.ch = m <= 592 && chunks <= 1024 ? 1 : (chunks <= 160 ? 2 : 4);
  } else {
    p.ch = m <= 592 || norm ? 1 : (chunks <= 128 ? 2 : 4);
  }
  if (aligned)
    while (chunks > (int64_t)p.ch * max_threads(8, p.ch)) p.ch *= 2;
  // Rows in turn, four chunks to a thread (as many as leave it whole warps): fp16 norms of enough elements to fill the
  // device a few times over - [8192, 4096] to e4m3 49 us a row per CTA, 40 us in turn; [900, 4096] 8.0 and 7.5; [600, 16384]
  // 23.6 and 15.2; but [900, 1024] 3.3 and 3.6, and fp32 norms, whose rows in flight take twice the registers, 33 and 42
  // at [4096, 4096].  For quantize only short rows gain, by the launches of so many CTAs: [8192, 1024] 9.0 and 6.6 us,
  // [1500, 1024] 2.6 and 2.7, [8192, 4096] 17.8 and 18.0.
  if (aligned && !p.edge) {
    if (norm && !wide && m * n_cols > 2400000 && chunks <= 4 * 512) {
      p.stream = true;
      p.ch = chunks >= 128 ? 4 : (chunks >= 64 ? 2 : 1);
    } else if (!norm && m > 4096 && chunks <= 128) {
      p.stream = true;
      p.ch = 2;
    }
  }
  p.tpr = (int)((chunks + p.ch - 1) / p.ch + 31) / 32 * 32;
  p.rows = p.tpr >= 64 ? 1 : 64 / p.tpr;
  return p;
}

template <int OP, typename InT, typename OutT, int CH, bool EDGE>
int launch_stream(const RowPlan& p, const RowArgs& a, int sm_count, cudaStream_t st) {
  static std::atomic<int> per_sm[64][kMaxThreads / 32 + 1];      // [device]: CTAs of so many warps that an SM holds, once asked for
  const int threads = p.tpr * p.rows;
  int dev = 0;
  DTAS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64) DTAS_FAIL(DTAS_EINVAL, "row op: device ordinal %d out of range", dev);
  int fit = per_sm[dev][threads / 32].load(std::memory_order_relaxed);
  if (fit == 0) {
    DTAS_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, (row_quant_stream_kernel<OP, InT, OutT, CH, EDGE>), threads, 0));
    per_sm[dev][threads / 32].store(fit, std::memory_order_relaxed);
  }
  const int64_t groups = (a.m + p.rows - 1) / p.rows, most = (int64_t)sm_count * fit;
  launch_kernel((row_quant_stream_kernel<OP, InT, OutT, CH, EDGE>), (unsigned)(groups < most ? groups : most), dim3(p.tpr, p.rows), 0,
                st, a);
  return after_launch("row_quant_stream_kernel");
}

template <int OP, typename InT, typename OutT>
int launch_typed(const RowPlan& p, const RowArgs& a, int sm_count, cudaStream_t st) {
  const dim3 block(p.tpr, p.rows);
  const int64_t grid = (a.m + p.rows - 1) / p.rows;
  if (grid > 0x7fffffffLL) DTAS_FAIL(DTAS_EINVAL, "row op: too many rows (%lld)", (long long)a.m);
  if (p.vec == 0) {
    launch_kernel(row_quant_long_kernel<OP, InT, OutT>, (unsigned)grid, block, 0, st, a);
    return after_launch("row_quant_long_kernel");
  }
  if (p.stream) {
    if constexpr (OP == Q_NORM && sizeof(InT) == 2) {
      if (p.edge && p.ch == 2) return launch_stream<OP, InT, OutT, 2, true>(p, a, sm_count, st);
      if (p.edge) return launch_stream<OP, InT, OutT, 4, true>(p, a, sm_count, st);
      if (p.ch == 1) return launch_stream<OP, InT, OutT, 1, false>(p, a, sm_count, st);
      if (p.ch == 4) return launch_stream<OP, InT, OutT, 4, false>(p, a, sm_count, st);
    }
    if constexpr (OP == Q_QUANT || sizeof(InT) == 2) return launch_stream<OP, InT, OutT, 2, false>(p, a, sm_count, st);
  }
#define DTAS_ROWQ_CASE(V, C, E)                                                                    \
  if (p.vec == V && p.ch == C && p.edge == E) {                                                    \
    launch_kernel(row_quant_kernel<OP, InT, OutT, V, C, E>, (unsigned)grid, block, 0, st, a);      \
    return after_launch("row_quant_kernel");                                                       \
  }
  DTAS_ROWQ_CASE(8, 1, false) DTAS_ROWQ_CASE(8, 2, false) DTAS_ROWQ_CASE(8, 4, false) DTAS_ROWQ_CASE(8, 8, false)
  DTAS_ROWQ_CASE(8, 1, true) DTAS_ROWQ_CASE(8, 2, true) DTAS_ROWQ_CASE(8, 4, true) DTAS_ROWQ_CASE(8, 8, true)
  DTAS_ROWQ_CASE(1, 4, false) DTAS_ROWQ_CASE(1, 16, false)
#undef DTAS_ROWQ_CASE
  DTAS_FAIL(DTAS_EINVAL, "row op: no kernel for %d x %d", p.vec, p.ch);
}

template <int OP, typename InT>
int launch_out(const RowPlan& p, const RowArgs& a, int out_dtype, int sm_count, cudaStream_t st) {
  if (out_dtype == DTAS_E4M3) return launch_typed<OP, InT, __nv_fp8_e4m3>(p, a, sm_count, st);
  if (out_dtype == DTAS_I8) return launch_typed<OP, InT, int8_t>(p, a, sm_count, st);
  if constexpr (OP == Q_NORM) {
    if (out_dtype == DTAS_F16) return launch_typed<OP, InT, __half>(p, a, sm_count, st);
  }
  DTAS_FAIL(DTAS_EUNSUPPORTED, "row op: unsupported output dtype %d", out_dtype);
}

template <int OP>
int launch_in(const RowArgs& a, int in_dtype, int out_dtype, int sm_count, cudaStream_t st) {
  bool aligned = aligned16(a.x) && aligned16(a.res) && aligned16(a.res_out) && aligned16(a.weight);
  aligned = aligned && (reinterpret_cast<uintptr_t>(a.y) & (out_dtype == DTAS_F16 ? 15 : 7)) == 0;
  const RowPlan p = row_plan(a.m, a.n_cols, aligned, OP == Q_NORM, in_dtype == DTAS_F32);
  if (in_dtype == DTAS_F16) return launch_out<OP, __half>(p, a, out_dtype, sm_count, st);
  if (in_dtype == DTAS_F32) return launch_out<OP, float>(p, a, out_dtype, sm_count, st);
  DTAS_FAIL(DTAS_EUNSUPPORTED, "row op: unsupported input dtype %d", in_dtype);
}

}  // namespace

int launch_add_rms_norm(const void* x, const void* res, const void* weight, void* y, void* res_out, float* scale,
                        int64_t m, int64_t n_cols, float eps, int in_dtype, int out_dtype, const DeviceCtx* ctx, cudaStream_t st) {
  return launch_in<Q_NORM>(RowArgs{x, res, static_cast<const __half*>(weight), y, res_out, scale, m, n_cols, eps},
                           in_dtype, out_dtype, ctx->sm_count, st);
}

int launch_quantize(const void* x, void* q, float* scale, int64_t m, int64_t n_cols, int in_dtype, int out_dtype,
                    const DeviceCtx* ctx, cudaStream_t st) {
  return launch_in<Q_QUANT>(RowArgs{x, nullptr, nullptr, q, nullptr, scale, m, n_cols, 0.f}, in_dtype, out_dtype,
                            ctx->sm_count, st);
}

void row_quant_variant_name(const char* op, int64_t m, int64_t n_cols, char* buf, int len) {
  const RowPlan p = row_plan(m, n_cols, true, strcmp(op, "quantize") != 0, false);
  if (p.vec == 0)
    snprintf(buf, len, "%s_long_cta%d", op, p.tpr);
  else
    snprintf(buf, len, "%s_vec%d%s_tpr%d_ch%d%s", op, p.vec, p.edge ? "_edge" : "", p.tpr, p.ch, p.stream ? "_stream" : "");
}

}  // namespace dtas
