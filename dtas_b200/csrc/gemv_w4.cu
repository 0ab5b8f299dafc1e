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
// a rate that these streams never reach), and a code has to become an fp16 number for them - for which it
// is enough to cut it out: sixteen bits that hold a code in the lowest four and zeros above are the
// subnormal fp16 number code * 2^-24, and a code four bits higher is code * 2^-20.  One AND per two codes and one
// shift per eight; no conversion, no subtraction.  Low and high codes go to accumulators of their own, and
//   sum_k x (q - z) = sum_k x q - z sum_k x,
// where the sums of x over the groups are taken once per CTA (in fp32) and -z times them is what the
// accumulators of a group start from.  The order of k inside an MMA is free as long as both operands agree on it:
// the pairs that the masks cut out of a word are (k, k + 4), so x is paired the same way.  A group's sums enter the
// row's fp32 sum with one multiply by the group's scale; x in 8 bits is widened to fp16, which holds it exactly.
//
// Measured, HBM 6.57 TB/s: one row by [22016, 4096] in groups of 32, bias and GELU 15.7 us (3.2 TB/s; its bytes take 7.7), by
// [4096, 4096] 5.8 us; sixteen rows by [4096, 11008] with zero points 19.0 us; four e4m3 or int8 rows by [50280, 2560] in groups of
// 64 17.6 us (3.9 TB/s).  Neither loads nor a pipe are at their limit, and with the codes in L2 it takes as long: three warps a
// scheduler take half of the issue slots between the preparation of x and the exchange of the sums.
#include <cuda.h>
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

__device__ __forceinline__ void mma_16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight consecutive elements of a row of x, as loaded, and as pairs (k, k + 4) of fp16 numbers.  Ordinary loads, not those
// of the read-only path: the kernel before this one may be writing x still when this one begins (pdl_wait).
template <typename XT>
struct XVec;
template <>
struct XVec<__half> {
  uint4 r;
  __device__ __forceinline__ void load(const __half* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void pairs(uint32_t* p) const {      // (0, 4), (1, 5), (2, 6), (3, 7)
    p[0] = __byte_perm(r.x, r.z, 0x5410);
    p[1] = __byte_perm(r.x, r.z, 0x7632);
    p[2] = __byte_perm(r.y, r.w, 0x5410);
    p[3] = __byte_perm(r.y, r.w, 0x7632);
  }
};
template <>
struct XVec<int8_t> {
  uint2 r;
  __device__ __forceinline__ void load(const int8_t* p) { r = *reinterpret_cast<const uint2*>(p); }
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
  __device__ __forceinline__ void load(const __nv_fp8_e4m3* p) { r = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void pairs(uint32_t* p) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t t = __byte_perm(r.x, r.y, 0x0040 + 0x0011 * i);
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(t & 0xffffu), __NV_E4M3);
      p[i] = (uint32_t)h.x | ((uint32_t)h.y << 16);
    }
  }
};

// The same from given accumulators: c0, c1 for the row g, c2, c3 for g + 8.
__device__ __forceinline__ void mma_16816_from(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, float c0, float c1,
                                               float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t w4_smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void w4_mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void w4_mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool w4_mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(20000u)      // may sleep for that many ns: a warp that polls takes issue slots from the others
      : "memory");
  return done != 0;
}
// Waits for a copy, for about a second; then records `code` and returns false.
__device__ __noinline__ bool w4_wait_slow(uint32_t bar, uint32_t parity, int* status, int code) {
  uint64_t t0, t1;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (;;) {
    for (int i = 0; i < 64; ++i)
      if (w4_mbar_try(bar, parity)) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
    if (t1 - t0 > 1000000000ull) {
      atomicExch(status, code);
      return false;
    }
  }
}
// Called by whole warps; the answer is the same for all lanes.
__device__ __forceinline__ bool w4_wait(uint32_t bar, uint32_t parity, int* status, int code) {
  bool done = w4_mbar_try(bar, parity);
  if (!done) done = w4_wait_slow(bar, parity, status, code);
  return __all_sync(0xffffffffu, done);
}
constexpr int ERR_W4_CODES = 0x301;

template <int BYTES>
__device__ __forceinline__ void w4_cp_async(uint32_t dst, const void* src, uint32_t bytes) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}

// The fast kernel: K % 32 == 0, groups of 32, 64 or a multiple of 128; x, q, scales and zero points 16-byte aligned.
//
// An item is a tile of 32 rows of q by IK k.  A CTA (one per SM) owns a band of tiles, and its twelve warps equal
// runs of the band's items, whatever tiles those fall into: a warp's sums of a tile that others share wait in
// shared memory, and one barrier at the end lets them be added up, in the order of the warps.  Items come into
// a ring of shared memory of the warp's own - the codes by one TMA load, scales and zero points by one cp.async of a
// lane per row - as far ahead as there is room.  Items of 256 k halve what an item costs beside its codes; items
// of 128 k take less room, and their place is asked for again as soon as their words are in registers.
// x waits in shared memory, as the pairs that the MMAs take, with the sums of its groups.  Where it does not fit
// there the CTAs of a cluster share out K (items [rank * share, ...)); a batch of tiles at a time they hand their sums to
// the CTA that finishes the row of x (row % CTAs), through distributed shared memory.
//
// TMA's 128-byte swizzle puts chunk c of row r at chunk c ^ (r % 8), its 64-byte swizzle (IK = 128) at c ^ (r / 2 % 4).
// MMA row g of a lane is row rho of the tile, chosen so that a word each of eight rows by four lanes, and 16
// bytes each of the two rows that a quarter warp reads, are in different banks.
constexpr int kWarps = 12;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxStages = 4;

template <int IK, int GS, bool ZERO>
struct Item {
  static constexpr int kSteps = IK / kStep;
  static constexpr int kGroups = kSteps / GS;
  static constexpr int kRowBytes = IK / 2;
  static constexpr int kCodes = kRows * kRowBytes;
  static constexpr int kSRow = kGroups == 1 ? 4 : 2 * kGroups;            // bytes of a row's scales as copied
  static constexpr int kZRow = !ZERO ? 0 : (kGroups < 4 ? 4 : kGroups);
  static constexpr int kParams = kRows * (kSRow + kZRow);
};

struct W4Shape {
  int n_tiles;
  int items;     // of a whole row
  int share;     // items of a CTA (all of them without a cluster)
  int stages;    // items a warp's ring holds
  int batch;     // tiles whose sums a cluster exchanges at a time
  int vec;       // an item's scales of a row can be copied as they lie
  int x_dtype;
  int* status;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A CTA's part of x, as pairs and as sums over the groups (times -8 or -1, in units of 2^-24).
// `meanwhile` runs while the first loads are under way.
template <typename XT, int GS, bool ZERO, typename F>
__device__ __forceinline__ void fill_x(const XT* x, int64_t k, int m, int chunks, int x_stride, int cols, uint4* xs, float* xsum,
                                       F meanwhile) {
  constexpr bool kWide = GS == 4;
  constexpr int kLoads = 8;
  const int total = chunks * m;
  int i = 0, c = threadIdx.x;
  for (int base = 0; base < total; base += kLoads * kThreads) {
    XVec<XT> v[kLoads];
    int row[kLoads], at[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      while (c >= chunks && i < m) {
        c -= chunks;
        ++i;
      }
      row[u] = i;
      at[u] = c;
      if (base + u * kThreads < total) v[u].load(i < m ? x + (int64_t)i * k + 8 * c : x);
      c += kThreads;
    }
    if (base == 0) meanwhile();
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      if (base + u * kThreads >= total) break;        // the same for the whole CTA
      uint32_t p[4];
      v[u].pairs(p);
      float2 s2 = __half22float2(*reinterpret_cast<const __half2*>(&p[0]));
#pragma unroll
      for (int e = 1; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[e]));
        s2.x += f.x;
        s2.y += f.y;
      }
      float sum = s2.x + s2.y;
      // the 4 GS chunks of a group are in neighbouring lanes: rows of this part are whole groups
#pragma unroll
      for (int o = 1; o < 4 * GS; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (row[u] < m) {
        const int j = kWide ? at[u] & 3 : (at[u] >> 2) & 3, tt = kWide ? (at[u] >> 2) & 3 : at[u] & 3;
        xs[row[u] * x_stride + ((at[u] >> 4) * 4 + j) * 4 + tt] = make_uint4(p[0], p[2], p[1], p[3]);      // low codes, high codes
        if (at[u] % (4 * GS) == 0) {      // {row 2t, 2t + 1, 2t, 2t + 1}: an MMA's accumulators as they start
          float* to = xsum + at[u] / (4 * GS) * (2 * cols) + (row[u] >> 1) * 4 + (row[u] & 1);
          to[0] = to[2] = sum * (ZERO ? -0x1p-24f : -0x1p-21f);
        }
      }
    }
  }
  if (total == 0) meanwhile();
}

// An element of y whose sum on the tensor cores, v, is not finite.  There an infinite x meets -z sum x and the code
// apart, which makes a NaN of what may be an infinity (so does an infinite scale).  Beside such terms the finite ones do not
// matter: one thread looks for them - at k whose x, and in groups whose scale is not finite - and adds up those alone,
// until they make a NaN.
template <typename XT>
__device__ __forceinline__ float w4_not_finite(const W4Args& a, int i, int n, float v) {
  const XT* x = static_cast<const XT*>(a.x) + (int64_t)i * a.k;
  const int groups = a.k / a.group;
  const __half* scales = a.w_scale + (int64_t)n * groups;
  float sum = 0.f;
  bool found = false;
  auto add = [&](int k) {
    const int code = (a.q[(int64_t)n * (a.k >> 1) + (k >> 1)] >> (4 * (k & 1))) & 15;
    const float z = a.zero != nullptr ? (float)a.zero[(int64_t)n * groups + k / a.group] : 8.f;
    sum = fmaf(__half2float(scales[k / a.group]) * ((float)code - z), (float)x[k], sum);
    found = true;
  };
#pragma unroll 1
  for (int k = 0; k < a.k && sum == sum; k += 8) {
    XVec<XT> c;
    uint32_t p[4];
    c.load(x + k);
    c.pairs(p);
    bool any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) any = any || (p[j] & 0x7c00u) == 0x7c00u || (p[j] & 0x7c000000u) == 0x7c000000u;
    if (any)
#pragma unroll 1
      for (int j = k; j < k + 8; ++j)
        if (!(fabsf((float)x[j]) < INFINITY)) add(j);
  }
#pragma unroll 1
  for (int gi = 0; gi < groups && sum == sum; ++gi)
    if (!(fabsf(__half2float(scales[gi])) < INFINITY))
      for (int k = gi * a.group; k < (gi + 1) * a.group; ++k) add(k);
  return found ? sum * 0x1p-24f : v;
}
__device__ __noinline__ float w4_not_finite(const W4Args& a, int x_dtype, int i, int n, float v) {
  if (x_dtype == DTAS_F16) return w4_not_finite<__half>(a, i, n, v);
  if (x_dtype == DTAS_I8) return w4_not_finite<int8_t>(a, i, n, v);
  return w4_not_finite<__nv_fp8_e4m3>(a, i, n, v);
}

// GS steps share a scale: 1, 2, or 4 (groups of 128 and more).
template <int IK, int NT, int GS, bool ZERO>
__global__ void __launch_bounds__(kThreads, 1)
    gemv_w4_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ W4Args a, const W4Shape sh) {
  using It = Item<IK, GS, ZERO>;
  extern __shared__ uint8_t w4_smem_raw[];
  // With groups of 128 k and more, lane t takes the codes 32 t .. 32 t + 31 of 128 (one 16-byte read a row), a word of
  // them per step; with smaller ones a step has to stay inside a group: the words of 32 k.
  constexpr bool kWide = GS == 4;
  constexpr int kGroups = It::kGroups, kCols = 8 * NT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rho = IK == 256 ? (g >> 1) | ((g & 1) << 2) : g;
  const int steps = a.k / kStep;
  const int cs = (int)cluster_size(), rank = (int)cluster_rank();
  const int item0 = rank * sh.share, n_items = max(0, min(sh.share, sh.items - item0));      // none, perhaps, at the end
  const int cluster = blockIdx.x / cs, n_clusters = gridDim.x / cs;
  const int band0 = (int)((int64_t)cluster * sh.n_tiles / n_clusters), band1 = (int)((int64_t)(cluster + 1) * sh.n_tiles / n_clusters);
  const int batch_tiles = cs == 1 ? band1 - band0 : sh.batch;
  const int groups = a.k / a.group;
  const int wide_group = a.group >> 7;              // > 1: items that share a scale

  uint8_t* ring = w4_smem_raw + ((1024u - (w4_smem_u32(w4_smem_raw) & 1023u)) & 1023u);      // [warp][stage]
  uint8_t* params = ring + kWarps * sh.stages * It::kCodes;                              // [warp][stage]: scales, zero points
  uint64_t* bars = reinterpret_cast<uint64_t*>(params + kWarps * sh.stages * It::kParams);        // [warp][stage]
  float* part = reinterpret_cast<float*>(bars + kWarps * kMaxStages);                     // [warp][2][row of x][row of q]
  float* xpart = part + kWarps * 2 * a.m * kRows;                                         // [tile][CTA][row of x / CTAs][row of q]
  const int xrows = (a.m + cs - 1) / cs;
  float* xsum = xpart + (cs > 1 ? sh.batch * cs * xrows * kRows : 0);                         // [group][pair of rows of x][4]
  const int x_stride = ((sh.share * It::kSteps) | 1) * 4;                                     // odd: rows of x in turn in both halves of the banks
  uint4* xs = reinterpret_cast<uint4*>(xsum + sh.share * kGroups * 2 * kCols);                // [row of x][step][t]

  const uint32_t full0 = w4_smem_u32(bars) + 8 * warp * kMaxStages;
  if (lane < sh.stages) {
    w4_mbar_init(full0 + 8 * lane, 1 + 32);       // the TMA load, and every lane's scales
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (threadIdx.x == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap)) : "memory");
  __syncwarp();
  if (cs > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // waited for before the first store to another CTA
  pdl_wait();
  pdl_launch_dependents();

  // A warp's run of the items of a batch of tiles that begins with tile `first`: this many, the last ones perhaps fewer.
  auto run_length = [&](int first) { return (min(batch_tiles, band1 - first) * n_items + kWarps - 1) / kWarps; };
  bool ok = true;

  // ---- copies.  The next item to be asked for, and how many of its run remain.
  const uint32_t my_ring = w4_smem_u32(ring) + warp * sh.stages * It::kCodes;
  const uint32_t my_scales = w4_smem_u32(params) + warp * sh.stages * It::kParams + lane * It::kSRow;      // lane = row of the tile
  const uint32_t my_zeros = w4_smem_u32(params) + warp * sh.stages * It::kParams + kRows * It::kSRow + lane * It::kZRow;
  int ask_first = band0, ask_tile = 0, ask_item = 0, ask_left = 0;
  const int64_t n_scales = (int64_t)a.n * groups;
  int64_t ask_o = 0;                        // first scale of the item in the lane's row
  auto ask_row = [&]() { ask_o = (int64_t)min(ask_tile * kRows + lane, a.n - 1) * groups + (int64_t)(item0 + ask_item) * kGroups; };
  auto ask_run = [&]() {                    // sets out for the run of batch ask_first, or of the next one that has any
    while (ask_left == 0 && ask_first < band1) {
      const int total = min(batch_tiles, band1 - ask_first) * n_items, per = run_length(ask_first), u = min(warp * per, total);
      ask_left = min(u + per, total) - u;
      if (ask_left > 0) {
        ask_tile = ask_first + u / n_items;
        ask_item = u % n_items;
        ask_row();
      }
      ask_first += batch_tiles;
    }
  };
  auto ask = [&](int stage) {
    if (ask_left == 0) return;
    const uint32_t bar = full0 + 8 * stage;
    if (lane == 0) {
      w4_mbar_expect(bar, It::kCodes);
      asm volatile(
          "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
              my_ring + stage * It::kCodes),
          "l"(reinterpret_cast<uint64_t>(&tmap)), "r"((item0 + ask_item) * It::kRowBytes), "r"(ask_tile * kRows), "r"(bar)
          : "memory");
    }
    const uint32_t sd = my_scales + stage * It::kParams, zd = my_zeros + stage * It::kParams;
    if (sh.vec) {
      if constexpr (kGroups == 1) {                  // the word that holds the scale; cut behind the last one
        const int64_t at = ask_o & ~(int64_t)1;
        w4_cp_async<4>(sd, a.w_scale + at, n_scales - at >= 2 ? 4u : 2u);
      } else {
        w4_cp_async<It::kSRow>(sd, a.w_scale + ask_o, It::kSRow);
      }
      if constexpr (ZERO) {
        if constexpr (kGroups < 4) {
          const int64_t at = ask_o & ~(int64_t)3;
          w4_cp_async<4>(zd, a.zero + at, n_scales - at >= 4 ? 4u : (uint32_t)(n_scales - at));
        } else {
          w4_cp_async<kGroups>(zd, a.zero + ask_o, kGroups);
        }
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    } else {
      const int64_t row = (int64_t)min(ask_tile * kRows + lane, a.n - 1) * groups;
#pragma unroll
      for (int e = 0; e < kGroups; ++e) {
        const int gi = (item0 + ask_item) * kGroups + e;
        const int64_t o = row + min(kWide ? gi / wide_group : gi, groups - 1);
        asm volatile("st.shared.b16 [%0], %1;" ::"r"(sd + 2 * e), "h"(__half_as_ushort(a.w_scale[o])) : "memory");
        if constexpr (ZERO) asm volatile("st.shared.b8 [%0], %1;" ::"r"(zd + e), "r"((uint32_t)a.zero[o]) : "memory");
      }
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
    }
    ask_o += kGroups;
    if (++ask_item == n_items) {
      ask_item = 0;
      ++ask_tile;
      ask_row();
    }
    if (--ask_left == 0) ask_run();
  };
  {
    auto ask_first_item = [&]() {
      ask_run();
      ask(0);
    };
    const int64_t first = (int64_t)item0 * IK;
    const int chunks = n_items > 0 ? (min((item0 + n_items) * IK, a.k) - (int)first) >> 3 : 0;      // of this CTA's part of a row
    if (sh.x_dtype == DTAS_F16)
      fill_x<__half, GS, ZERO>(static_cast<const __half*>(a.x) + first, a.k, a.m, chunks, x_stride, kCols, xs, xsum, ask_first_item);
    else if (sh.x_dtype == DTAS_I8)
      fill_x<int8_t, GS, ZERO>(static_cast<const int8_t*>(a.x) + first, a.k, a.m, chunks, x_stride, kCols, xs, xsum, ask_first_item);
    else
      fill_x<__nv_fp8_e4m3, GS, ZERO>(static_cast<const __nv_fp8_e4m3*>(a.x) + first, a.k, a.m, chunks, x_stride, kCols, xs, xsum, ask_first_item);
    for (int i = 1; i < sh.stages; ++i) ask(i);      // behind the first items of all warps, which are wanted first
    __syncthreads();
  }

  // Columns at or beyond m of an MMA read the last row of x again: nothing looks at their sums.
  const uint4* x_lane[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) x_lane[j] = xs + min(j * 8 + g, a.m - 1) * x_stride + t;
  const float4* const s_lane = reinterpret_cast<const float4*>(xsum) + t;
  const uint8_t* const codes0 = ring + warp * sh.stages * It::kCodes + rho * It::kRowBytes;
  const uint8_t* const scales0 = params + warp * sh.stages * It::kParams + rho * It::kSRow;
  const uint8_t* const zeros0 = params + warp * sh.stages * It::kParams + kRows * It::kSRow + rho * It::kZRow;
  const int swz = (IK == 256 ? rho : (rho >> 1) & 3) * 16;                   // the same for the rows rho + 8 i
  int code_off[4];                                       // of the words of a step of the first 128 k, or (kWide) of the lane's 16 bytes
#pragma unroll
  for (int v = 0; v < 4; ++v) code_off[v] = kWide ? (16 * t) ^ swz : ((16 * v) ^ swz) + 4 * t;
  // Sums are handled four columns to a lane: eight lanes a row of x, four rows a warp.
  const int quad = (lane & 7) * 4, row4 = lane >> 3;
  auto finish = [&](int i, int col, float4 sum) {
    float v[4] = {sum.x, sum.y, sum.z, sum.w};
    if (!(fabsf(v[0]) + fabsf(v[1]) + fabsf(v[2]) + fabsf(v[3]) < INFINITY)) {
#pragma unroll 1
      for (int e = 0; e < 4; ++e)
        if (col + e < a.n && !(fabsf(v[e]) < INFINITY)) v[e] = w4_not_finite(a, sh.x_dtype, i, col + e, v[e]);
    }
    const float scale = a.x_scale != nullptr ? a.x_scale[i] : 1.f;
    if (col + 4 <= a.n && !a.epi.out_f32 && (reinterpret_cast<uintptr_t>(a.y) & 7) == 0 && (a.n & 3) == 0) {
      __half h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = __float2half_rn(epi_value(a.epi, v[e] * 0x1p24f * scale, i, col + e));
      *reinterpret_cast<uint2*>(static_cast<__half*>(a.y) + (int64_t)i * a.n + col) = *reinterpret_cast<const uint2*>(h);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < a.n) epi_store(a.epi, a.y, a.n, i, col + e, epi_value(a.epi, v[e] * 0x1p24f * scale, i, col + e));
    }
  };
  // This CTA's sums of tile `tl` of a batch for row i of x: the result, or what the CTA that finishes the row is sent.
  auto tile_sum = [&](int tl, int first, int i, float4 sum) {
    if (cs == 1) {
      finish(i, (first + tl) * kRows + quad, sum);
    } else {
      const uint32_t local = w4_smem_u32(xpart + ((tl * cs + rank) * xrows + i / cs) * kRows + quad);
      uint32_t remote;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(i % cs));
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(sum.x), "f"(sum.y), "f"(sum.z), "f"(sum.w)
                   : "memory");
    }
  };
  auto add4 = [](float4& to, const float* from) {
    const float4 v = *reinterpret_cast<const float4*>(from);
    to.x += v.x; to.y += v.y; to.z += v.z; to.w += v.w;
  };
  bool joined = cs == 1;
  auto join = [&]() {        // once, before the first store to another CTA: by then it has long begun to run
    if (!joined) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    joined = true;
  };
  int stage = 0;
  uint32_t phase = 0;
  for (int first = band0; first < band1; first += batch_tiles) {
    const int tiles = min(batch_tiles, band1 - first), total = tiles * n_items, per = run_length(first);
    int u = min(warp * per, total);
    const int run_end = min(u + per, total);
    while (u < run_end) {
      const int tl = u / n_items, begin = u - tl * n_items, end = min(n_items, begin + run_end - u);      // items of this tile
      u += end - begin;
      const int n0 = (first + tl) * kRows;
      float acc[NT][2][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j][i >> 2][i & 3] = 0.f;
      for (int local = begin; local < end && ok; ++local) {
        ok = w4_wait(full0 + 8 * stage, phase, sh.status, ERR_W4_CODES);
        if (!ok) break;
        const int item = item0 + local;
        // scales and zero points of the rows rho + 8 i, in pairs of groups and in bytes
        uint32_t sc[4][(kGroups + 1) / 2], zp[4][kGroups > 4 ? 2 : 1];
        {
          const uint8_t* sp = scales0 + stage * It::kParams;
          const uint8_t* zq = zeros0 + stage * It::kParams;
          // where a scale or its zero points lie in a word depends on the row's parity; 8 rows on it is the same
          const uint32_t o = sh.vec ? (uint32_t)(n0 + rho) * (uint32_t)groups + (uint32_t)(item * kGroups) : 0u;
          const bool last_rows = n0 + kRows > a.n;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t oi = last_rows && sh.vec ? (uint32_t)min(n0 + rho + 8 * i, a.n - 1) * (uint32_t)groups + (uint32_t)(item * kGroups) : o;
            if constexpr (kGroups == 8) {
              const uint4 v = *reinterpret_cast<const uint4*>(sp + 8 * i * It::kSRow);
              sc[i][0] = v.x; sc[i][1] = v.y; sc[i][2] = v.z; sc[i][3] = v.w;
            } else if constexpr (kGroups == 4) {
              const uint2 v = *reinterpret_cast<const uint2*>(sp + 8 * i * It::kSRow);
              sc[i][0] = v.x; sc[i][1] = v.y;
            } else if constexpr (kGroups == 2) {
              sc[i][0] = *reinterpret_cast<const uint32_t*>(sp + 8 * i * It::kSRow);
            } else {
              sc[i][0] = *reinterpret_cast<const uint32_t*>(sp + 8 * i * It::kSRow) >> (16 * (oi & 1));
            }
            if constexpr (ZERO) {
              if constexpr (kGroups == 8) {
                const uint2 v = *reinterpret_cast<const uint2*>(zq + 8 * i * It::kZRow);
                zp[i][0] = v.x; zp[i][1] = v.y;
              } else if constexpr (kGroups == 4) {
                zp[i][0] = *reinterpret_cast<const uint32_t*>(zq + 8 * i * It::kZRow);
              } else {
                zp[i][0] = *reinterpret_cast<const uint32_t*>(zq + 8 * i * It::kZRow) >> (8 * (oi & 3));
              }
            }
          }
        }
        const int x_item = local * (It::kSteps * 4), s_item = local * (kGroups * kCols / 2);
        const uint8_t* codes = codes0 + stage * It::kCodes;
        uint32_t w[4][4];        // [row rho + 8 i][step of 128 k]
        auto load_words = [&](int h) {
          if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(codes + 8 * i * It::kRowBytes + (code_off[0] ^ (64 * h)));
              w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
            }
          } else {
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i][v] = *reinterpret_cast<const uint32_t*>(codes + 8 * i * It::kRowBytes + (code_off[v] ^ (64 * h)));
          }
        };
        auto release = [&]() {
          // Every lane has read the item: its place may be filled again.  The copies write through the asynchronous
          // proxy, which only this fence orders behind the lanes' reads - without it some reads were seen to
          // return the next item's bytes.
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          ask(stage);
          if (++stage == sh.stages) {
            stage = 0;
            phase ^= 1u;
          }
        };
        load_words(0);
        if constexpr (IK == 128) release();
        float lo[NT][2][4], hi[NT][2][4];      // sums of the low and the high codes of a group, in units of 2^-24 and 2^-20
        auto step = [&](int s) {
          const int b = s / GS;
          uint32_t p[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w8 = w[i][s & 3] >> 8;
            p[i][0] = w[i][s & 3] & 0x000f000fu;
            p[i][1] = w[i][s & 3] & 0x00f000f0u;
            p[i][2] = w8 & 0x000f000fu;
            p[i][3] = w8 & 0x00f000f0u;
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint4 x = x_lane[j][x_item + s * 4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint32_t al[4] = {p[2 * r][0], p[2 * r + 1][0], p[2 * r][2], p[2 * r + 1][2]};
              const uint32_t ah[4] = {p[2 * r][1], p[2 * r + 1][1], p[2 * r][3], p[2 * r + 1][3]};
              if (s % GS == 0) {
                const float4 v = s_lane[s_item + b * (kCols / 2) + j * 4];
                if constexpr (ZERO) {
                  const float f0 = (float)((zp[2 * r][b / 4] >> (8 * (b & 3))) & 0xffu);
                  const float f1 = (float)((zp[2 * r + 1][b / 4] >> (8 * (b & 3))) & 0xffu);
                  mma_16816_from(lo[j][r], al, x.x, x.y, f0 * v.x, f0 * v.y, f1 * v.z, f1 * v.w);
                } else {
                  mma_16816_from(lo[j][r], al, x.x, x.y, v.x, v.y, v.z, v.w);
                }
                mma_16816_from(hi[j][r], ah, x.z, x.w, 0.f, 0.f, 0.f, 0.f);
              } else {
                mma_16816(lo[j][r], al, x.x, x.y);
                mma_16816(hi[j][r], ah, x.z, x.w);
              }
            }
          }
          if (s % GS == GS - 1) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float sf[2], sf16[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t v = sc[2 * r + i][b / 2];
                const __half2 h = *reinterpret_cast<const __half2*>(&v);
                sf[i] = (b & 1) ? __high2float(h) : __low2float(h);
                sf16[i] = sf[i] * 0.0625f;
              }
#pragma unroll
              for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  acc[j][r][e] = fmaf(sf[e >> 1], lo[j][r][e], acc[j][r][e]);
                  acc[j][r][e] = fmaf(sf16[e >> 1], hi[j][r][e], acc[j][r][e]);
                }
            }
          }
        };
        const int live = steps - item * It::kSteps;             // steps of this item; K ends on the border of a group
        if (live >= It::kSteps) {                               // a whole item without a branch inside: its steps interleave
#pragma unroll
          for (int s = 0; s < It::kSteps; ++s) {
            if (s == 4) load_words(1);
            step(s);
          }
        } else {
#pragma unroll
          for (int s = 0; s < It::kSteps; ++s) {
            if (s < live) {
              if (s == 4) load_words(1);
              step(s);
            }
          }
        }
        if constexpr (IK == 256) release();
      }
      join();
      // ---- this warp's sums of the tile: area 0 where the run begins inside it, else area 1
      float* mine = part + (warp * 2 + (begin == 0 ? 1 : 0)) * (a.m * kRows);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = j * 8 + 2 * t + e;
          if (c < a.m) {
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[c * kRows + rho + 8 * i] = acc[j][i >> 1][(i & 1) * 2 + e];
          }
        }
      if (begin == 0 && end == n_items) {            // no other warp has a part in it
        __syncwarp();
        for (int i = row4; i < a.m; i += 4) tile_sum(tl, first, i, *reinterpret_cast<const float4*>(mine + i * kRows + quad));
        __syncwarp();
      }
    }
    // ---- tiles that several warps share
    join();
    __syncthreads();
    const int m4 = (a.m + 3) >> 2;
    for (int e = warp; e < m4 * tiles; e += kWarps) {
      const int tl = e / m4, i = (e - tl * m4) * 4 + row4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (n_items > 0) {
        const int u0 = tl * n_items, w0 = u0 / per, w1 = (u0 + n_items - 1) / per;
        if (w0 == w1) continue;             // that warp has done it
        if (i < a.m) {                      // area 1 of the warp whose run holds the tile's first item; area 0 of the others
          const float* from = part + i * kRows + quad;
          add4(sum, from + (2 * w0 + 1) * (a.m * kRows));
          for (int w = w0 + 1; w <= w1; ++w) add4(sum, from + 2 * w * (a.m * kRows));
        }
      }
      if (i < a.m) tile_sum(tl, first, i, sum);
    }
    if (cs > 1) {
      cluster_barrier();
      const int x4 = (xrows + 3) >> 2;
      for (int e = warp; e < tiles * x4; e += kWarps) {
        const int tl = e / x4, q = (e - tl * x4) * 4 + row4, i = q * cs + rank;
        if (q < xrows && i < a.m) {
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int v = 0; v < cs; ++v) add4(sum, xpart + ((tl * cs + v) * xrows + q) * kRows + quad);      // rank order = K order
          finish(i, (first + tl) * kRows + quad, sum);
        }
      }
      if (first + batch_tiles < band1) cluster_barrier();
    }
  }
  // A wait that gave up leaves copies on their way into this CTA's shared memory: give them time to land.
  if (!ok) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    uint64_t t0, t1;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    do {
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
    } while (t1 - t0 < 100000000ull);
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

// ---- dispatch ------------------------------------------------------------------
constexpr int64_t kSmemMax = 227 * 1024;
constexpr int kMaxCluster = 8;

struct W4Plan {
  W4Shape sh;
  int item_k;       // 256, or 128
  int cluster;      // CTAs that share out K; 0: the shape does not fit eight CTAs
  int grid;
  int64_t smem;
};

// Clusters of c CTAs that the device holds at once: they do not pack every SM of its GPCs.  As the driver answers for one CTA
// per SM (any instantiation: one fills an SM); before the first launch on a device the figures of a B200 are assumed.
constexpr int kMaxDevices = 64;
std::atomic<int> w4_max_clusters[kMaxDevices][3];      // of 2, 4 and 8 CTAs; 0: not asked yet
inline int w4_clusters(int c, int sm_count, int device) {
  if (c == 1) return sm_count;
  const int slot = c == 2 ? 0 : (c == 4 ? 1 : 2);
  static const int assumed[3] = {74, 33, 15};
  const int n = device >= 0 && device < kMaxDevices ? w4_max_clusters[device][slot].load(std::memory_order_relaxed) : 0;
  return n > 0 ? n : assumed[slot];
}

// A CTA takes a whole row's K where m rows of x fit beside its rings, else as many CTAs as it takes for a part of them to
// fit share it out, with the sums of all their tiles exchanged at once; only where eight CTAs leave no room for that,
// in batches (every batch ends in two barriers of the cluster, and its few items leave the warps with little to do:
// sixteen rows, [4096, 11008], 21 us in four batches).  Items of 256 k, two to a ring, where there is room for them; else
// of 128 k, two to four.  Deeper rings only let the first items of some warps queue behind later items of others
// ([12288, 4096], one token: 10.7 us with two items of 256 k, 13.7 with three).
inline W4Plan w4_plan(int64_t m, int64_t n, int64_t k, int64_t group, bool zero, int sm_count, int device) {
  W4Plan p{};
  const int64_t groups = k / group, cols = m <= 8 ? 8 : 16;
  p.sh.n_tiles = (int)((n + kRows - 1) / kRows);
  for (int c = 1; c <= kMaxCluster; c *= 2) {
    const int most = w4_clusters(c, sm_count, device), n_clusters = p.sh.n_tiles < most ? p.sh.n_tiles : most;
    const int band = (p.sh.n_tiles + n_clusters - 1) / n_clusters;
    const int64_t xrows = (m + c - 1) / c;
    for (int ik = m <= 8 && c == 1 ? 256 : 128; ik >= 128; ik /= 2) {
      const int64_t per_item = ik / (group < 128 ? group : 128);
      const int64_t params = kRows * ((per_item == 1 ? 4 : 2 * per_item) + (!zero ? 0 : (per_item < 4 ? 4 : per_item)));
      const int64_t stage_bytes = kWarps * (kRows * ik / 2 + params), tile_bytes = c > 1 ? 4 * c * xrows * kRows : 0;
      p.sh.items = (int)((k + ik - 1) / ik);
      p.sh.share = (p.sh.items + c - 1) / c;
      p.sh.vec = group <= 128 && groups % per_item == 0 ? 1 : 0;
      p.item_k = ik;
      const int64_t left = kSmemMax - 1024 - 8 * kWarps * kMaxStages - 4 * (kWarps * 2 * m * kRows + p.sh.share * per_item * 2 * cols) -
                           (((int64_t)p.sh.share * ik / kStep) | 1) * 64 * m;
      int64_t batch = band;
      if (left < 2 * stage_bytes + band * tile_bytes) {
        if (c < kMaxCluster || left < 2 * stage_bytes + tile_bytes) continue;
        const int64_t fit = (left - 2 * stage_bytes) / tile_bytes, parts = (band + fit - 1) / fit;
        batch = (band + parts - 1) / parts;
      }
      const int64_t deep = (left - batch * tile_bytes) / stage_bytes, most_stages = ik == 256 ? 2 : kMaxStages;
      p.sh.batch = (int)batch;
      p.sh.stages = (int)(deep < most_stages ? deep : most_stages);
      p.smem = kSmemMax - left + p.sh.stages * stage_bytes + batch * tile_bytes;
      p.cluster = c;
      p.grid = n_clusters * c;
      return p;
    }
  }
  return p;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn w4_encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

template <int IK, int NT, int GS, bool ZERO>
int launch_one(const W4Args& a, int x_dtype, const DeviceCtx* ctx, cudaStream_t st) {
  static std::atomic<bool> ready[kMaxDevices];
  int dev = 0;
  DTAS_CUDA(cudaGetDevice(&dev));
  if (dev >= kMaxDevices) DTAS_FAIL(DTAS_EINVAL, "gemv_w4: device ordinal %d out of range", dev);
  if (!ready[dev].load(std::memory_order_acquire)) {
    DTAS_CUDA(cudaFuncSetAttribute((gemv_w4_kernel<IK, NT, GS, ZERO>), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
    for (int i = 0; i < 3; ++i) {
      if (w4_max_clusters[dev][i].load(std::memory_order_relaxed) != 0) continue;
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr;
      cfg.gridDim = dim3((unsigned)(2 << i));
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = (size_t)kSmemMax;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = (unsigned)(2 << i);
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, gemv_w4_kernel<IK, NT, GS, ZERO>, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        n = 0;
      }
      w4_max_clusters[dev][i].store(n, std::memory_order_relaxed);
    }
    ready[dev].store(true, std::memory_order_release);
  }
  const W4Plan p = w4_plan(a.m, a.n, a.k, a.group, ZERO, ctx->sm_count, dev);
  if (p.cluster == 0 || p.item_k != IK) DTAS_FAIL(DTAS_EUNSUPPORTED, "gemv_w4: no plan");      // the caller has asked
  // q as bytes [n, k / 2], boxes of 32 rows by IK / 2 bytes; what lies outside arrives as zeros
  const EncodeTiledFn encode = w4_encode_fn();
  if (encode == nullptr) DTAS_FAIL(DTAS_ECUDA, "gemv_w4: cuTensorMapEncodeTiled is not available from the driver");
  CUtensorMap map;
  const cuuint64_t dims[2] = {(cuuint64_t)a.k / 2, (cuuint64_t)a.n}, strides[1] = {(cuuint64_t)a.k / 2};
  const cuuint32_t box[2] = {IK / 2, kRows}, ones[2] = {1, 1};
  const CUresult r = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(a.q), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, IK == 256 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) DTAS_FAIL(DTAS_ECUDA, "gemv_w4: cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)p.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  W4Shape sh = p.sh;
  sh.status = ctx->status;
  sh.x_dtype = x_dtype;
  (void)cudaLaunchKernelEx(&cfg, gemv_w4_kernel<IK, NT, GS, ZERO>, map, a, sh);
  return after_launch("gemv_w4_kernel");
}

template <typename XT>
int launch_scalar(const W4Args& a, cudaStream_t st) {
  launch_kernel(gemv_w4_scalar_kernel<XT>, dim3((unsigned)((a.n + 7) / 8), (unsigned)a.m), 256, 0, st, a);
  return after_launch("gemv_w4_scalar_kernel");
}

template <int GS, bool ZERO>
int launch_gs(const W4Args& a, int item_k, int x_dtype, const DeviceCtx* ctx, cudaStream_t st) {
  if (a.m > 8) return launch_one<128, 2, GS, ZERO>(a, x_dtype, ctx, st);
  return item_k == 256 ? launch_one<256, 1, GS, ZERO>(a, x_dtype, ctx, st) : launch_one<128, 1, GS, ZERO>(a, x_dtype, ctx, st);
}
template <int GS>
int launch_zero(const W4Args& a, int item_k, int x_dtype, const DeviceCtx* ctx, cudaStream_t st) {
  return a.zero != nullptr ? launch_gs<GS, true>(a, item_k, x_dtype, ctx, st) : launch_gs<GS, false>(a, item_k, x_dtype, ctx, st);
}

inline bool w4_fast_shape(int64_t k, int64_t group) {
  return k % kStep == 0 && (group == 32 || group == 64 || group % 128 == 0);
}

template <typename XT>
int launch_x(const W4Args& a, int x_dtype, const DeviceCtx* ctx, cudaStream_t st) {
  const bool fast = w4_fast_shape(a.k, a.group) && aligned16(a.q) && aligned16(a.x) && aligned16(a.w_scale) && aligned16(a.zero);
  if (!fast) return launch_scalar<XT>(a, st);
  // whether a plan exists, and its items, do not depend on how many clusters the device holds
  const W4Plan p = w4_plan(a.m, a.n, a.k, a.group, a.zero != nullptr, ctx->sm_count, -1);
  if (p.cluster == 0) return launch_scalar<XT>(a, st);
  if (a.group == 32) return launch_zero<1>(a, p.item_k, x_dtype, ctx, st);
  if (a.group == 64) return launch_zero<2>(a, p.item_k, x_dtype, ctx, st);
  return launch_zero<4>(a, p.item_k, x_dtype, ctx, st);
}

}  // namespace

// Named for groups of 128 without zero points.
void gemv_w4_variant_name(int64_t m, int64_t n, int64_t k, const DeviceCtx* ctx, int device, char* buf, int len) {
  const W4Plan p = w4_plan(m, n, k, 128, false, ctx->sm_count, device);
  if (k % kStep != 0 || p.cluster == 0) snprintf(buf, len, "gemv_w4_scalar_warp_per_element");
  else snprintf(buf, len, "gemv_w4_mma_m%d_k%d_s%d_cluster%d", m <= 8 ? 8 : 16, p.item_k, p.sh.stages, p.cluster);
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
  if (x_dtype == DTAS_I8) return launch_x<int8_t>(a, x_dtype, ctx, st);
  if (x_dtype == DTAS_E4M3) return launch_x<__nv_fp8_e4m3>(a, x_dtype, ctx, st);
  return launch_x<__half>(a, x_dtype, ctx, st);
}

}  // namespace dtas
