// Products of a few rows with 4-bit weights in groups (decoding one token, a batch of sequences, or a
// handful of drafted tokens).  No counterpart in the reference.
//
//   y[i, n] = tail( xs[i] * sum_g ws[n, g] * sum_{k in g} x[i, k] * (q[n, k] - z[n, g]) ),  i < m <= 16
//
// q: two codes to a byte, the even k in the low half; ws fp16 and z (a byte; 8 where there are no zero
// points) per row and group of G columns; x fp16, or int8 / e4m3 with one fp32 scale xs a row.
//
// The stream over q is the cost (N K / 2 bytes), and what stands in its way is arithmetic, not loads: at the
// HBM rate an SM takes in 46 codes per clock, and unpacking a code, widening it and a fused multiply-add
// for it are three instructions of the 128 an SM issues per clock.  So the products go to the tensor cores
// (mma.sync m16n8k16, fp32 accumulators: sixteen rows of q against up to eight rows of x at once, at
// a rate that these streams never reach), and a code only has to become an fp16 number:
// 0x6400 | code is 1024 + code, and one subtraction (for the codes in the high halves of a byte one fused
// multiply-add by 1/16) leaves code - z, exactly.  The order of k inside an MMA is free as long as both operands
// agree on it: the pairs that two masks cut out of a word are (k, k + 4), so x is paired the same way.
// A group's products are summed by themselves (in the accumulators of its MMAs) and enter the row's fp32
// sum with one multiply by the group's scale; x in 8 bits is widened to fp16, which holds it exactly.
//
// A CTA owns sixteen rows of q; its warps take blocks of 128 k in turn and add up through shared memory.
#include <cuda_fp8.h>

#include "common.cuh"

namespace dtas {
namespace {

constexpr int kRows = 16;          // rows of q per CTA = MMA M
constexpr int kStep = 32;          // k of one step: a word of eight codes per lane and row
static_assert(DTAS_W4_MAX_ROWS == 16, "two tiles of eight rows of x");

struct W4Args {
  const void* x;
  const float* x_scale;     // int8 / e4m3 rows
  const uint8_t* q;
  const __half* w_scale;
  const uint8_t* zero;      // optional
  void* y;
  Epilogue epi;
  int m, n, k, group;
};

__device__ __forceinline__ void mma_16816(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// Eight codes of a word as four pairs (k, k + 4), k = 0..3, of fp16 numbers code - z.
// zl = {1024 + z, 1024 + z}, zh = {-(64 + z), -(64 + z)}: both exact for any byte z.
__device__ __forceinline__ void widen(uint32_t w, __half2 zl, __half2 zh, uint32_t* p) {
  const __half2 sixteenth = __float2half2_rn(0.0625f);
  const uint32_t w8 = w >> 8;
  const uint32_t t0 = (w & 0x000f000fu) | 0x64006400u, t1 = (w & 0x00f000f0u) | 0x64006400u;
  const uint32_t t2 = (w8 & 0x000f000fu) | 0x64006400u, t3 = (w8 & 0x00f000f0u) | 0x64006400u;
  const __half2 h0 = __hsub2(*reinterpret_cast<const __half2*>(&t0), zl);
  const __half2 h1 = __hfma2(*reinterpret_cast<const __half2*>(&t1), sixteenth, zh);
  const __half2 h2 = __hsub2(*reinterpret_cast<const __half2*>(&t2), zl);
  const __half2 h3 = __hfma2(*reinterpret_cast<const __half2*>(&t3), sixteenth, zh);
  p[0] = *reinterpret_cast<const uint32_t*>(&h0);
  p[1] = *reinterpret_cast<const uint32_t*>(&h1);
  p[2] = *reinterpret_cast<const uint32_t*>(&h2);
  p[3] = *reinterpret_cast<const uint32_t*>(&h3);
}

// Eight consecutive elements of a row of x, as loaded, and as pairs (k, k + 4) of fp16 numbers.
template <typename XT>
struct XVec;
template <>
struct XVec<__half> {
  uint4 r;
  __device__ __forceinline__ void load(const __half* p) { r = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void clear() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void pairs(uint32_t* p) const {
    p[0] = __byte_perm(r.x, r.z, 0x5410);
    p[1] = __byte_perm(r.x, r.z, 0x7632);
    p[2] = __byte_perm(r.y, r.w, 0x5410);
    p[3] = __byte_perm(r.y, r.w, 0x7632);
  }
};
template <>
struct XVec<int8_t> {
  uint2 r;
  __device__ __forceinline__ void load(const int8_t* p) { r = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void clear() { r = make_uint2(0, 0); }
  __device__ __forceinline__ void pairs(uint32_t* p) const {
    const uint32_t a = r.x ^ 0x80808080u, b = r.y ^ 0x80808080u;      // x + 128 in 0..255
    const __half2 bias = __float2half2_rn(1152.f);                    // 1024 + 128
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t t = (__byte_perm(a, b, 0x0400 + 0x0101 * i) & 0x00ff00ffu) | 0x64006400u;
      const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&t), bias);
      p[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
template <>
struct XVec<__nv_fp8_e4m3> {
  uint2 r;
  __device__ __forceinline__ void load(const __nv_fp8_e4m3* p) { r = __ldg(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void clear() { r = make_uint2(0, 0); }
  __device__ __forceinline__ void pairs(uint32_t* p) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t t = __byte_perm(r.x, r.y, 0x0040 + 0x0011 * i);
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(t & 0xffffu), __NV_E4M3);
      p[i] = (uint32_t)h.x | ((uint32_t)h.y << 16);
    }
  }
};

// K % 32 == 0, group % 32 == 0, q 16-byte and x 16-byte (8-bit x: 8-byte) aligned.  NT tiles of eight rows of x.
// SPG steps (of 32 k) share a group's scale inside a block of four: 4 where the group is a multiple of 128.
template <typename XT, int NT, int SPG, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) gemv_w4_kernel(const W4Args a) {
  __shared__ float part[WARPS][kRows][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kRows;
  const int r0 = min(n0 + g, a.n - 1), r1 = min(n0 + g + 8, a.n - 1);
  const int steps = a.k / kStep;
  const int groups = a.k / a.group, steps_per_group = a.group / kStep;
  const int64_t row_words = a.k >> 3;
  const uint32_t* q0 = reinterpret_cast<const uint32_t*>(a.q) + r0 * row_words + t;
  const uint32_t* q1 = reinterpret_cast<const uint32_t*>(a.q) + r1 * row_words + t;
  const XT* x = static_cast<const XT*>(a.x) + 8 * t;

  pdl_wait();
  pdl_launch_dependents();

  float acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;

  for (int s0 = warp * 4; s0 < steps; s0 += WARPS * 4) {
    uint32_t w0[4], w1[4];
    XVec<XT> xv[4][NT];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bool on = s0 + s < steps;
      w0[s] = on ? __ldg(q0 + (s0 + s) * 4) : 0u;
      w1[s] = on ? __ldg(q1 + (s0 + s) * 4) : 0u;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (on && j * 8 + g < a.m) xv[s][j].load(x + (int64_t)(j * 8 + g) * a.k + (s0 + s) * kStep);
        else xv[s][j].clear();
      }
    }
    float grp[NT][4];
    __half2 zl0, zh0, zl1, zh1;
    float sc0 = 0.f, sc1 = 0.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s0 + s < steps) {
        if (s % SPG == 0) {
          const int gi = (s0 + s) / steps_per_group;
          sc0 = __half2float(a.w_scale[(int64_t)r0 * groups + gi]);
          sc1 = __half2float(a.w_scale[(int64_t)r1 * groups + gi]);
          const float z0 = a.zero != nullptr ? (float)a.zero[(int64_t)r0 * groups + gi] : 8.f;
          const float z1 = a.zero != nullptr ? (float)a.zero[(int64_t)r1 * groups + gi] : 8.f;
          zl0 = __float2half2_rn(1024.f + z0);
          zh0 = __float2half2_rn(-(64.f + z0));
          zl1 = __float2half2_rn(1024.f + z1);
          zh1 = __float2half2_rn(-(64.f + z1));
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) grp[j][i] = 0.f;
        }
        uint32_t p0[4], p1[4];
        widen(w0[s], zl0, zh0, p0);
        widen(w1[s], zl1, zh1, p1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t b[4];
          xv[s][j].pairs(b);
          const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]};
          const uint32_t a1[4] = {p0[2], p1[2], p0[3], p1[3]};
          mma_16816(grp[j], a0, b);
          mma_16816(grp[j], a1, b + 2);
        }
        if (s % SPG == SPG - 1 || s0 + s + 1 == steps) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            acc[j][0] = fmaf(sc0, grp[j][0], acc[j][0]);
            acc[j][1] = fmaf(sc0, grp[j][1], acc[j][1]);
            acc[j][2] = fmaf(sc1, grp[j][2], acc[j][2]);
            acc[j][3] = fmaf(sc1, grp[j][3], acc[j][3]);
          }
        }
      }
    }
  }

#pragma unroll
  for (int j = 0; j < NT; ++j) {
    part[warp][g][j * 8 + 2 * t] = acc[j][0];
    part[warp][g][j * 8 + 2 * t + 1] = acc[j][1];
    part[warp][g + 8][j * 8 + 2 * t] = acc[j][2];
    part[warp][g + 8][j * 8 + 2 * t + 1] = acc[j][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kRows * a.m; e += WARPS * 32) {
    const int r = e % kRows, i = e / kRows;       // neighbouring threads: neighbouring columns of y
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += part[w][r][i];
    const int col = n0 + r;
    if (col < a.n) {
      if (a.x_scale != nullptr) sum *= a.x_scale[i];
      epi_store(a.epi, a.y, a.n, i, col, epi_value(a.epi, sum, i, col));
    }
  }
}

// Any even K, any group that divides it, any alignment: one warp per element of y.
template <typename XT>
__global__ void __launch_bounds__(256) gemv_w4_scalar_kernel(const W4Args a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = blockIdx.x * 8 + warp, i = blockIdx.y;
  pdl_wait();
  pdl_launch_dependents();
  if (n >= a.n) return;
  const uint8_t* q = a.q + (int64_t)n * (a.k >> 1);
  const XT* x = static_cast<const XT*>(a.x) + (int64_t)i * a.k;
  const int groups = a.k / a.group;
  float sum = 0.f;
  for (int k = lane; k < a.k; k += 32) {
    const int gi = k / a.group;
    const int code = (q[k >> 1] >> (4 * (k & 1))) & 15;
    const float z = a.zero != nullptr ? (float)a.zero[(int64_t)n * groups + gi] : 8.f;
    const float w = __half2float(a.w_scale[(int64_t)n * groups + gi]) * ((float)code - z);
    sum = fmaf(w, (float)x[k], sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    if (a.x_scale != nullptr) sum *= a.x_scale[i];
    epi_store(a.epi, a.y, a.n, i, n, epi_value(a.epi, sum, i, n));
  }
}

constexpr int kWarpsW4 = 8;

template <typename XT, int NT>
int launch_nt(const W4Args& a, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.n + kRows - 1) / kRows);
  if (a.group % 128 == 0)
    launch_kernel(gemv_w4_kernel<XT, NT, 4, kWarpsW4>, grid, kWarpsW4 * 32, 0, st, a);
  else if (a.group % 64 == 0)
    launch_kernel(gemv_w4_kernel<XT, NT, 2, kWarpsW4>, grid, kWarpsW4 * 32, 0, st, a);
  else
    launch_kernel(gemv_w4_kernel<XT, NT, 1, kWarpsW4>, grid, kWarpsW4 * 32, 0, st, a);
  return after_launch("gemv_w4_kernel");
}

template <typename XT>
int launch_x(const W4Args& a, cudaStream_t st) {
  const bool vec = a.k % kStep == 0 && a.group % kStep == 0 && aligned16(a.q) &&
                   (reinterpret_cast<uintptr_t>(a.x) & (8 * sizeof(XT) - 1)) == 0;
  if (!vec) {
    launch_kernel(gemv_w4_scalar_kernel<XT>, dim3((unsigned)((a.n + 7) / 8), (unsigned)a.m), 256, 0, st, a);
    return after_launch("gemv_w4_scalar_kernel");
  }
  return a.m <= 8 ? launch_nt<XT, 1>(a, st) : launch_nt<XT, 2>(a, st);
}

}  // namespace

void gemv_w4_variant_name(int64_t m, int64_t n, int64_t k, char* buf, int len) {
  (void)n;
  if (k % kStep != 0) snprintf(buf, len, "gemv_w4_scalar_warp_per_element");
  else snprintf(buf, len, "gemv_w4_mma_m%d_warps%d", m <= 8 ? 8 : 16, kWarpsW4);
}

int launch_gemv_w4(const void* x, const float* x_scale, const void* w, const void* w_scale, const void* w_zero,
                   const Epilogue& epi, void* y, int64_t m, int64_t n, int64_t k, int64_t group, int x_dtype,
                   cudaStream_t st) {
  W4Args a;
  a.x = x;
  a.x_scale = x_scale;
  a.q = static_cast<const uint8_t*>(w);
  a.w_scale = static_cast<const __half*>(w_scale);
  a.zero = static_cast<const uint8_t*>(w_zero);
  a.y = y;
  a.epi = epi;
  a.m = (int)m;
  a.n = (int)n;
  a.k = (int)k;
  a.group = (int)group;
  if (x_dtype == DTAS_I8) return launch_x<int8_t>(a, st);
  if (x_dtype == DTAS_E4M3) return launch_x<__nv_fp8_e4m3>(a, st);
  return launch_x<__half>(a, st);
}

}  // namespace dtas
