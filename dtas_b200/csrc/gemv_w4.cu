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
#include <cuda_fp8.h>

#include "common.cuh"

namespace dtas {
namespace {

constexpr int kRows = 32;          // rows of q per tile: two MMAs of sixteen
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

// (w & mask) | 0x64006400 as one instruction.
__device__ __forceinline__ __half2 pick(uint32_t w, uint32_t mask) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(0x64006400u));
  return *reinterpret_cast<const __half2*>(&r);
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
// Eight codes of a word as four pairs (k, k + 4), k = 0..3, of fp16 numbers code - z.
// zl = {1024 + z, 1024 + z}, zh = {-(64 + z), -(64 + z)}: both exact for any byte z.
__device__ __forceinline__ void widen(uint32_t w, __half2 zl, __half2 zh, uint32_t* p) {
  const __half2 sixteenth = __float2half2_rn(0.0625f);
  const uint32_t w8 = w >> 8;
  p[0] = as_u32(__hsub2(pick(w, 0x000f000fu), zl));
  p[1] = as_u32(__hfma2(pick(w, 0x00f000f0u), sixteenth, zh));
  p[2] = as_u32(__hsub2(pick(w8, 0x000f000fu), zl));
  p[3] = as_u32(__hfma2(pick(w8, 0x00f000f0u), sixteenth, zh));
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

__device__ __forceinline__ void mma_16816_first(float* c, const uint32_t* a, const uint32_t* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}
// 16 bytes from global to shared memory behind the thread's back; `bytes` (0 or 16) of them are read, the rest is zero.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The fast kernel: K % 32 == 0, group % 32 == 0, q and x 16-byte aligned.
//
// An item is a tile of 32 rows of q by 256 k: 4 KB that a warp copies into its own ring of shared memory with
// cp.async (a row of an item is one 128-byte line), kStages - 1 items ahead, across the borders of tiles.
// kw warps share a tile, each taking every kw-th item of it; behind a tile they add up through shared
// memory in the order of the warps, with one barrier (of these kw warps) a tile: the sums of consecutive tiles
// go to two areas in turn.  CTAs are persistent, so the copies never run dry between tiles.
// The 16-byte chunk c of row r of an item lies at chunk c ^ (r / 2 % 4) ^ (r % 2 * 4) of its line: a word each of
// eight rows by four lanes, and 16 bytes each of two rows by four lanes, are then in different banks.
// x waits in shared memory as the pairs that the MMAs take (XS); where it does not fit there it is read from
// global memory (L1) and paired at each use.
constexpr int kCtaWarps = 8;
constexpr int kItemK = 256;
constexpr int kItemSteps = kItemK / kStep;
constexpr int kStages = 2;
constexpr int kRowBytes = kItemK / 2;
constexpr int kItemBytes = kRows * kRowBytes;
constexpr int kRingBytes = kCtaWarps * kStages * kItemBytes;

// Scales (and zero points) of an item for the four rows g + 8 i of a lane, two rows to a register.  GS steps share a
// group; lane t of four holds groups t (GS = 2), t & 1 (GS = 4), 2t and 2t + 1 (GS = 1), and the others get
// them by a shuffle.
template <int GS>
struct GroupRegs {
  static constexpr int kN = GS == 1 ? 2 : 1;
  uint32_t v[kN][2];
  template <typename T>
  __device__ __forceinline__ void load(const T* const* row, int item, int t, int groups, int spg) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int block = GS == 1 ? 2 * t + i : (GS == 2 ? t : (GS == 4 ? (t & 1) : 0));
      // a group of exactly GS steps (32, 64, 128 or 256 k) needs no division
      int gi = spg == GS ? item * (kItemSteps / GS) + block : (item * kItemSteps + block * GS) / spg;
      gi = min(gi, groups - 1);
      v[i][0] = (uint32_t)__ldg(row[0] + gi) | ((uint32_t)__ldg(row[1] + gi) << 16);
      v[i][1] = (uint32_t)__ldg(row[2] + gi) | ((uint32_t)__ldg(row[3] + gi) << 16);
    }
  }
  __device__ __forceinline__ uint32_t get(int block, int half) const {
    if constexpr (GS == 8) return v[0][half];
    if constexpr (GS == 1) return __shfl_sync(0xffffffffu, v[block & 1][half], block >> 1, 4);
    return __shfl_sync(0xffffffffu, v[0][half], block, 4);
  }
};

template <typename XT, int NT, int GS, bool ZERO, bool XS>
__global__ void __launch_bounds__(kCtaWarps * 32, 2) gemv_w4_kernel(const W4Args a, const int kw, const int n_tiles) {
  extern __shared__ __align__(128) uint8_t w4_smem[];
  // With groups of 128 k and more, lane t takes the codes 32 t .. 32 t + 31 of 128 (one 16-byte read a row), a
  // word of them per step; with smaller ones a step has to stay inside a group: the words of 32 k.
  constexpr bool kWide = GS >= 4;
  uint8_t* ring = w4_smem;
  float* part = reinterpret_cast<float*>(w4_smem + kRingBytes);                    // [2][warp][row of x][row of q]
  uint4* xs = reinterpret_cast<uint4*>(part + 2 * kCtaWarps * a.m * kRows);        // [step][row of x][t]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int slots = kCtaWarps / kw, slot = warp / kw, kpos = warp - slot * kw;
  const int steps = a.k / kStep, items = (steps + kItemSteps - 1) / kItemSteps;
  const int groups = a.k / a.group, spg = a.group / kStep;
  const int tile0 = blockIdx.x * slots + slot, tile_step = gridDim.x * slots;
  const int64_t row_bytes = a.k >> 1;

  pdl_wait();
  pdl_launch_dependents();

  // ---- copies: item (ptile, pitem) is the next one to be asked for
  uint8_t* my_ring = ring + warp * kStages * kItemBytes;
  int ptile = tile0, pitem = kpos;
  // a copy instruction: four rows of 128 bytes; the rows of a lane are crow + 4 i, so only bit 2 of crow + 4 i changes
  // the chunk's place: by 2
  const int crow = lane >> 3, chunk = lane & 7;
  const int swz = chunk ^ (crow >> 1) ^ ((crow & 1) << 2);
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(my_ring) + crow * kRowBytes;
  const uint32_t even = swz * 16, odd = (swz ^ 2) * 16;
  uint32_t stage_off = 0;
  const uint8_t* const src0 = a.q + crow * row_bytes + kpos * (kItemK / 2) + chunk * 16;
  const uint8_t* src = src0 + (int64_t)ptile * kRows * row_bytes;
  const int64_t four_rows = 4 * row_bytes;
  auto ask = [&]() {
    if (ptile < n_tiles) {
      const uint32_t dst = ring_s + stage_off;
      if ((ptile + 1) * kRows <= a.n && (pitem + 1) * kItemSteps <= steps) {
#pragma unroll
        for (int i = 0; i < kRows / 4; ++i)
          cp_async16(dst + 4 * i * kRowBytes + (i & 1 ? odd : even), src + i * four_rows, 16u);
      } else {                                              // rows beyond N and k beyond K arrive as zeros
        const bool in = (int64_t)pitem * (kItemK / 2) + chunk * 16 < row_bytes;
#pragma unroll
        for (int i = 0; i < kRows / 4; ++i) {
          const bool on = in && ptile * kRows + crow + 4 * i < a.n;
          cp_async16(dst + 4 * i * kRowBytes + (i & 1 ? odd : even), on ? src + i * four_rows : a.q, on ? 16u : 0u);
        }
      }
      pitem += kw;
      src += kw * (kItemK / 2);
      if (pitem >= items) {
        pitem = kpos;
        ptile += tile_step;
        src = src0 + (int64_t)ptile * kRows * row_bytes;
      }
    }
    stage_off = stage_off == (kStages - 1) * kItemBytes ? 0 : stage_off + kItemBytes;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) ask();

  const XT* x = static_cast<const XT*>(a.x);
  if constexpr (XS) {
    const int chunks = a.k >> 3;
    int i = 0, c = threadIdx.x;
    auto settle = [&]() {
      while (c >= chunks && i < a.m) {
        c -= chunks;
        ++i;
      }
    };
    settle();
    while (i < a.m) {
      constexpr int kBatch = 8;
      XVec<XT> v[kBatch];
      int to[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int j = kWide ? c & 3 : (c >> 2) & 3, tt = kWide ? (c >> 2) & 3 : c & 3;
        to[u] = i < a.m ? (((c >> 4) * 4 + j) * a.m + i) * 4 + tt : -1;
        if (i < a.m) v[u].load(x + (int64_t)i * a.k + 8 * c);
        c += kCtaWarps * 32;
        settle();
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (to[u] >= 0) {
          uint32_t p[4];
          v[u].pairs(p);
          xs[to[u]] = make_uint4(p[0], p[1], p[2], p[3]);
        }
      }
    }
    __syncthreads();
  }
  // Columns at or beyond m of an MMA read the last row of x again: nothing looks at their sums.
  const uint4* x_lane[NT];
  const XT* x_row[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int col = min(j * 8 + g, a.m - 1);
    x_lane[j] = xs + col * 4 + t;
    x_row[j] = x + (int64_t)col * a.k + 8 * t * (kWide ? 4 : 1);
  }
  const int x_step = a.m * 4;
  const int wswz = ((g >> 1) ^ ((g & 1) << 2)) * 16;      // the same for the rows g + 8 i
  const uint8_t* codes = my_ring + g * kRowBytes;
  const uint8_t* const codes_end = codes + kStages * kItemBytes;
  int buf = 0;
  for (int tile = tile0; tile < n_tiles; tile += tile_step) {
    const int n0 = tile * kRows;
    const unsigned short* ws[4];
    const uint8_t* wz[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t o = (int64_t)min(n0 + g + 8 * i, a.n - 1) * groups;
      ws[i] = reinterpret_cast<const unsigned short*>(a.w_scale) + o;
      wz[i] = ZERO ? a.zero + o : nullptr;
    }
    float acc[NT][2][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[j][i >> 2][i & 3] = 0.f;
    GroupRegs<GS> next_s, next_z;
    next_s.load(ws, kpos, t, groups, spg);
    if constexpr (ZERO) next_z.load(wz, kpos, t, groups, spg);
    for (int item = kpos; item < items; item += kw) {
      const GroupRegs<GS> gs = next_s, gz = next_z;
      if (item + kw < items) {
        next_s.load(ws, item + kw, t, groups, spg);
        if constexpr (ZERO) next_z.load(wz, item + kw, t, groups, spg);
      }
      ask();
      cp_async_wait<kStages - 1>();
      __syncwarp();            // every lane's copies of this item have landed
      const int x_item = item * kItemSteps * x_step;
      uint32_t w[4][4];        // [row g + 8 i][step of the block of 128 k]
      float grp[NT][2][4];
      __half2 zl[4], zh[4];
      float2 sf[2];
      auto load_words = [&](int h) {
        if constexpr (kWide) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(codes + 8 * i * kRowBytes + ((64 * h + 16 * t) ^ wswz));
            w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
          }
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i][u] = *reinterpret_cast<const uint32_t*>(codes + 8 * i * kRowBytes + ((64 * h + 16 * u) ^ wswz) + 4 * t);
        }
      };
      auto open_group = [&](int b) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t sc = gs.get(b, r);
          sf[r] = __half22float2(*reinterpret_cast<const __half2*>(&sc));
          if constexpr (ZERO) {
            const uint32_t z = gz.get(b, r) | 0x64006400u;
            const uint32_t z0 = __byte_perm(z, z, 0x1010), z1 = __byte_perm(z, z, 0x3232);
            zl[2 * r] = *reinterpret_cast<const __half2*>(&z0);
            zl[2 * r + 1] = *reinterpret_cast<const __half2*>(&z1);
            zh[2 * r] = __hsub2(__float2half2_rn(960.f), zl[2 * r]);
            zh[2 * r + 1] = __hsub2(__float2half2_rn(960.f), zl[2 * r + 1]);
          } else {
            zl[2 * r] = zl[2 * r + 1] = __float2half2_rn(1032.f);
            zh[2 * r] = zh[2 * r + 1] = __float2half2_rn(-72.f);
          }
        }
      };
      auto step = [&](int s, bool first) {
        uint32_t p[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) widen(w[i][s & 3], zl[i], zh[i], p[i]);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t bx[4];
          if constexpr (XS) {
            const uint4 v = x_lane[j][x_item + s * x_step];
            bx[0] = v.x; bx[1] = v.y; bx[2] = v.z; bx[3] = v.w;
          } else {
            XVec<XT> v;
            v.load(x_row[j] + item * kItemK + (kWide ? 128 * (s >> 2) + 8 * (s & 3) : 32 * s));
            v.pairs(bx);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t a0[4] = {p[2 * r][0], p[2 * r + 1][0], p[2 * r][1], p[2 * r + 1][1]};
            const uint32_t a1[4] = {p[2 * r][2], p[2 * r + 1][2], p[2 * r][3], p[2 * r + 1][3]};
            if (first) mma_16816_first(grp[j][r], a0, bx);
            else mma_16816(grp[j][r], a0, bx);
            mma_16816(grp[j][r], a1, bx + 2);
          }
        }
      };
      auto close_group = [&]() {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            acc[j][r][0] = fmaf(sf[r].x, grp[j][r][0], acc[j][r][0]);
            acc[j][r][1] = fmaf(sf[r].x, grp[j][r][1], acc[j][r][1]);
            acc[j][r][2] = fmaf(sf[r].y, grp[j][r][2], acc[j][r][2]);
            acc[j][r][3] = fmaf(sf[r].y, grp[j][r][3], acc[j][r][3]);
          }
      };
      const int live = steps - item * kItemSteps;             // steps of this item; K ends on the border of a group
      if (live >= kItemSteps) {                               // a whole item without a branch inside: its steps interleave
#pragma unroll
        for (int s = 0; s < kItemSteps; ++s) {
          if (s % 4 == 0) load_words(s / 4);
          if (s % GS == 0) open_group(s / GS);
          step(s, s % GS == 0);
          if (s % GS == GS - 1) close_group();
        }
      } else {
#pragma unroll
        for (int s = 0; s < kItemSteps; ++s) {
          if (s < live) {
            if (s % 4 == 0) load_words(s / 4);
            if (s % GS == 0) open_group(s / GS);
            step(s, s % GS == 0);
            if (s % GS == GS - 1) close_group();
          }
        }
      }
      __syncwarp();            // the item is read: its place may be asked for
      codes = codes + kItemBytes == codes_end ? codes_end - kStages * kItemBytes : codes + kItemBytes;
    }
    float* mine = part + (buf * kCtaWarps + warp) * (a.m * kRows);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int c = j * 8 + 2 * t + e;
        if (c < a.m) {
#pragma unroll
          for (int i = 0; i < 4; ++i) mine[c * kRows + g + 8 * i] = acc[j][i >> 1][(i & 1) * 2 + e];
        }
      }
    if (kw == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(kw * 32) : "memory");
    const float* all = part + (buf * kCtaWarps + slot * kw) * (a.m * kRows) + lane;
    const int col = n0 + lane;
    for (int i = kpos; i < a.m; i += kw) {        // a warp finishes whole rows of x
      float sum = 0.f;
      for (int v = 0; v < kw; ++v) sum += all[(v * a.m + i) * kRows];
      if (col < a.n) {
        if (a.x_scale != nullptr) sum *= a.x_scale[i];
        epi_store(a.epi, a.y, a.n, i, col, epi_value(a.epi, sum, i, col));
      }
    }
    buf ^= 1;
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

// Shared memory of a CTA, and how many share an SM: two where it leaves room for two.
constexpr int kSmemSm = 226 * 1024, kSmemTwo = 112 * 1024;
inline int64_t smem_bytes(int64_t m, int64_t x_bytes) { return kRingBytes + 2 * kCtaWarps * m * kRows * 4 + x_bytes; }
// x in shared memory: m rows of k fp16 numbers, whatever x's type.
inline bool x_in_smem(int64_t m, int64_t k) { return smem_bytes(m, 2 * m * k) <= kSmemSm; }
// Warps that share a row tile: as many as have an item of it each, up to the whole CTA; half as many where
// there are tiles enough to keep every CTA busy for several rounds all the same (a tile costs its warps a
// barrier and a sum, whatever its length).
inline int tile_warps(int64_t n, int64_t k, int sm_count) {
  const int64_t items = (k + kItemK - 1) / kItemK, tiles = (n + kRows - 1) / kRows;
  int kw = 1;
  while (kw < kCtaWarps && 2 * kw <= items) kw *= 2;
  while (kw > 2 && tiles * kw / kCtaWarps >= 6 * 2 * sm_count) kw /= 2;
  return kw;
}

template <typename XT, int NT, int GS, bool ZERO, bool XS>
int launch_one(const W4Args& a, int sm_count, cudaStream_t st) {
  const size_t smem = (size_t)smem_bytes(a.m, XS ? (int64_t)2 * a.m * a.k : 0);
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  DTAS_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
    DTAS_CUDA(cudaFuncSetAttribute((gemv_w4_kernel<XT, NT, GS, ZERO, XS>), cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemSm));
    if (dev < 64) attr_set[dev].store(true, std::memory_order_release);
  }
  const int kw = tile_warps(a.n, a.k, sm_count), n_tiles = (a.n + kRows - 1) / kRows, slots = kCtaWarps / kw;
  const int want = (n_tiles + slots - 1) / slots, most = sm_count * (smem <= kSmemTwo ? 2 : 1);
  launch_kernel(gemv_w4_kernel<XT, NT, GS, ZERO, XS>, (unsigned)(want < most ? want : most), kCtaWarps * 32, smem, st, a, kw, n_tiles);
  return after_launch("gemv_w4_kernel");
}

template <typename XT, int NT, int GS, bool ZERO>
int launch_xs(const W4Args& a, int sm_count, cudaStream_t st) {
  return x_in_smem(a.m, a.k) ? launch_one<XT, NT, GS, ZERO, true>(a, sm_count, st) : launch_one<XT, NT, GS, ZERO, false>(a, sm_count, st);
}
template <typename XT, int NT, int GS>
int launch_gs(const W4Args& a, int sm_count, cudaStream_t st) {
  return a.zero != nullptr ? launch_xs<XT, NT, GS, true>(a, sm_count, st) : launch_xs<XT, NT, GS, false>(a, sm_count, st);
}
// Steps of 32 k that share a scale inside an item: the largest power of two that divides the group.
template <typename XT, int NT>
int launch_nt(const W4Args& a, int sm_count, cudaStream_t st) {
  if (a.group % 256 == 0) return launch_gs<XT, NT, 8>(a, sm_count, st);
  if (a.group % 128 == 0) return launch_gs<XT, NT, 4>(a, sm_count, st);
  if (a.group % 64 == 0) return launch_gs<XT, NT, 2>(a, sm_count, st);
  return launch_gs<XT, NT, 1>(a, sm_count, st);
}

template <typename XT>
int launch_x(const W4Args& a, int sm_count, cudaStream_t st) {
  const bool vec = a.k % kStep == 0 && a.group % kStep == 0 && aligned16(a.q) &&
                   aligned16(a.x);
  if (!vec) {
    launch_kernel(gemv_w4_scalar_kernel<XT>, dim3((unsigned)((a.n + 7) / 8), (unsigned)a.m), 256, 0, st, a);
    return after_launch("gemv_w4_scalar_kernel");
  }
  return a.m <= 8 ? launch_nt<XT, 1>(a, sm_count, st) : launch_nt<XT, 2>(a, sm_count, st);
}

}  // namespace

void gemv_w4_variant_name(int64_t m, int64_t n, int64_t k, char* buf, int len) {
  if (k % kStep != 0) snprintf(buf, len, "gemv_w4_scalar_warp_per_element");
  else snprintf(buf, len, "gemv_w4_mma_m%d_kw%d_x%s", m <= 8 ? 8 : 16, tile_warps(n, k, 148), x_in_smem(m, k) ? "smem" : "l1");
}

int launch_gemv_w4(const void* x, const float* x_scale, const void* w, const void* w_scale, const void* w_zero,
                   const Epilogue& epi, void* y, int64_t m, int64_t n, int64_t k, int64_t group, int x_dtype,
                   const DeviceCtx* ctx, cudaStream_t st) {
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
  if (x_dtype == DTAS_I8) return launch_x<int8_t>(a, ctx->sm_count, st);
  if (x_dtype == DTAS_E4M3) return launch_x<__nv_fp8_e4m3>(a, ctx->sm_count, st);
  return launch_x<__half>(a, ctx->sm_count, st);
}

}  // namespace dtas
