// The product of cx_product.cuh on the fifth-generation tensor cores, for 16-bit operands.
//
// A persistent grid of CTAs, or of pairs of CTAs that share a tile, walks over the output's tiles.  One thread per CTA
// brings 64-deep slices of both operands into a ring of stages with tile copies, one thread per tile issues the matrix
// instructions, whose sums stay in tensor memory, and eight warps take finished sums from there: the tensor memory holds
// two tiles, so the matrix instructions of a tile run under the epilogue of the tile before.  Each layout of the operands
// is read as it lies: consecutive along k or along m and n is a bit of the instruction and another shape of the copy.
#include "cx_product.cuh"
#include "cx_tensor.cuh"

namespace {

constexpr int kDepth = 64;               // elements of k in a stage: one 128-byte line
constexpr int kThreads = 384;            // warp 0 copies, warp 1 multiplies, warp 2 has the tensor memory, 4 to 11 finish
constexpr int kJoinThreads = 256;
constexpr int kPitch = 36;               // floats of a row of the epilogue's scratch: 16-byte accesses without conflicts
constexpr int kFinish = 8;               // finishing warps: four have the left half of a tile's columns, four the right one
constexpr int kScratch = kFinish * 32 * kPitch * 4;
constexpr int kShared = 232448;          // of a CTA
constexpr int kGroup = 8;                // tiles along m that are walked together: their operands stay in L2

template <int CG, int BN>
struct Shape {
  static constexpr int kA = 128 * kDepth * 2, kB = BN / CG * kDepth * 2, kStage = kA + kB;
  static constexpr int kFit = (kShared - 1024 - 512 - kScratch) / kStage;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kBytes = 1024 + 512 + kScratch + kStages * kStage;
  static constexpr int kColumns = 2 * BN;
};

struct Plan {
  CxProduct p;
  int tiles_m, tiles_n, splits;
  int slices, slices_per;      // of kDepth along k: all, and per split
  float* partial;              // sums of the splits: [split][m][part_ld]
  int64_t part_ld;
  uint32_t* status;            // set when a wait has run out
  int wide_out, wide_add, wide_res, wide_bias;   // 16-byte accesses are aligned
};

struct Unit {
  int tm, tn, split, s0, s1;
};
__device__ __forceinline__ Unit unit_of(const Plan& t, int u) {
  Unit r;
  const int tiles = t.tiles_m * t.tiles_n;
  r.split = u / tiles;
  const int tile = u - r.split * tiles, per = kGroup * t.tiles_n, first = tile / per * kGroup;
  const int rows = min(kGroup, t.tiles_m - first), in = tile % per;
  r.tm = first + in % rows;
  r.tn = in / rows;
  r.s0 = r.split * t.slices_per;
  r.s1 = min(t.slices, r.s0 + t.slices_per);
  return r;
}

// What is done to sums (kOut, kSums) of R rows, `apart` rows apart, each 8 neighbouring columns.
template <typename T, int R>
__device__ __forceinline__ void finish(const Plan& t, int64_t row, int apart, int64_t col, float (&v)[8 * R]) {
  const CxProduct& p = t.p;
  const int left = (int)min((int64_t)8, p.n - col);
  if (left <= 0) return;
  float x[8];
  if (p.has_addend) {
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (row + j * apart < p.m) {
        cxprod::load8(p.addend + (row + j * apart) * p.n + col, left == 8 && t.wide_add, left, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * j + i] += x[i];
      }
  }
  if (p.mode == kSums) {
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (row + j * apart < p.m) {
        float* at = p.addend + (row + j * apart) * p.n + col;
        if (left == 8 && t.wide_add) {
          *reinterpret_cast<float4*>(at) = make_float4(v[8 * j], v[8 * j + 1], v[8 * j + 2], v[8 * j + 3]);
          *reinterpret_cast<float4*>(at + 4) = make_float4(v[8 * j + 4], v[8 * j + 5], v[8 * j + 6], v[8 * j + 7]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < left) at[i] = v[8 * j + i];
        }
      }
    return;
  }
  const bool wide = left == 8 && t.wide_out;
  if (p.scale) {
    const float f = *p.scale;
#pragma unroll
    for (int i = 0; i < 8 * R; ++i) v[i] *= f;
  }
  if (p.bias) {
    cxprod::load8(reinterpret_cast<const T*>(p.bias) + col, left == 8 && t.wide_bias, left, x);
#pragma unroll
    for (int i = 0; i < 8 * R; ++i) v[i] += x[i % 8];
  }
  if (p.pre) {
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (row + j * apart < p.m)
        cxprod::store8(reinterpret_cast<T*>(p.pre) + (row + j * apart) * p.ldo + col, wide, left, v + 8 * j);
  }
  cxprod::activate(v, p.act);
#pragma unroll
  for (int j = 0; j < R; ++j)
    if (row + j * apart < p.m) {
      if (p.residual) {
        cxprod::load8(reinterpret_cast<const T*>(p.residual) + (row + j * apart) * p.ldr + col, left == 8 && t.wide_res, left, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * j + i] += x[i];
      }
      cxprod::store8(reinterpret_cast<T*>(p.out) + (row + j * apart) * p.ldo + col, wide, left, v + 8 * j);
    }
}

// Rows of the warp's 32 x 32 sums, one per lane, through shared memory to four lanes per row: every access of the
// output is then 16 bytes, 64 neighbouring bytes a row.
template <typename T>
__device__ __forceinline__ void finish32(const Plan& t, int split, int64_t row0, int64_t col, float* scratch, const uint32_t (&r)[32]) {
  const int lane = threadIdx.x & 31, c = lane % 4 * 8;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint4*>(scratch + lane * kPitch + 4 * j) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
  __syncwarp();
  float v[32];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float* at = scratch + (8 * j + lane / 4) * kPitch + c;
    *reinterpret_cast<float4*>(v + 8 * j) = *reinterpret_cast<const float4*>(at);
    *reinterpret_cast<float4*>(v + 8 * j + 4) = *reinterpret_cast<const float4*>(at + 4);
  }
  __syncwarp();
  row0 += lane / 4;
  col += c;
  if (!t.partial) return finish<T, 4>(t, row0, 8, col, v);
  if (col >= t.p.n) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (row0 + 8 * j < t.p.m) {                              // part_ld is a multiple of 8
      float* at = t.partial + ((int64_t)split * t.p.m + row0 + 8 * j) * t.part_ld + col;
      *reinterpret_cast<float4*>(at) = make_float4(v[8 * j], v[8 * j + 1], v[8 * j + 2], v[8 * j + 3]);
      *reinterpret_cast<float4*>(at + 4) = make_float4(v[8 * j + 4], v[8 * j + 5], v[8 * j + 6], v[8 * j + 7]);
    }
}

// The same for values that only have to be rounded and stored: they go through shared memory in 16 bits.
template <typename T>
__device__ __forceinline__ void store32(const Plan& t, int64_t row0, int64_t col, float* scratch, const uint32_t (&r)[32]) {
  const int lane = threadIdx.x & 31, c = lane % 4 * 8;
  const CxProduct& p = t.p;
  uint4* mine = reinterpret_cast<uint4*>(scratch) + lane * 5;          // 64 bytes of a row, 16 of padding
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint2 lo, hi;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r[8 * j + i]);
    cxprod::pack4(x, &lo, T());
    cxprod::pack4(x + 4, &hi, T());
    mine[j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  __syncwarp();
  uint4 q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = reinterpret_cast<const uint4*>(scratch)[(8 * j + lane / 4) * 5 + lane % 4];
  __syncwarp();
  const int left = (int)min((int64_t)8, p.n - col - c);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t row = row0 + 8 * j + lane / 4;
    if (row >= p.m || left <= 0) continue;
    T* at = reinterpret_cast<T*>(p.out) + row * p.ldo + col + c;
    if (left == 8 && t.wide_out) {
      *reinterpret_cast<uint4*>(at) = q[j];
    } else {
      const T* e = reinterpret_cast<const T*>(&q[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) at[i] = e[i];
    }
  }
}

// A finishing warp's part of a tile: 32 rows, WIDTH columns from col0 on.
template <typename T, int WIDTH>
__device__ __forceinline__ void finish_part(const Plan& t, int split, int64_t part, int64_t row0, int64_t col0, uint32_t tmem, float* scratch) {
  const CxProduct& p = t.p;
  const int lane = threadIdx.x & 31;
  const int64_t row = row0 + lane;
  const bool in = row < p.m;
  uint32_t r[32];
  if (p.mode == kStats) {
    if (col0 >= p.n) return;
    const int64_t hot = (in ? p.targets[row] : -1) - p.col0 - col0;      // where the row's target is in this part
    float top = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int c = 0; c < WIDTH; c += 32) {
      if (col0 + c >= p.n) break;
      cxt::tmem_load32(tmem + c, r);
      cxt::tmem_load_wait();
      if (col0 + c + 32 > p.n) {
        const int left = (int)(p.n - col0 - c);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j >= left) r[j] = 0xFF800000u;
      }
      if (hot >= c && hot < c + 32) {
        float x = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (hot == c + j) x = __uint_as_float(r[j]);
        p.target_logit[row] = x;
      }
      float m[4] = {top, top, top, top}, add[4] = {};
#pragma unroll
      for (int j = 0; j < 32; ++j) m[j % 4] = fmaxf(m[j % 4], __uint_as_float(r[j]));
      m[0] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
      const float base = (m[0] == -INFINITY ? 0.f : m[0]) * cxprod::kLog2e;
#pragma unroll
      for (int j = 0; j < 32; ++j) add[j % 4] += cxprod::pow2(__fmaf_rn(__uint_as_float(r[j]), cxprod::kLog2e, -base));
      sum = sum * cxprod::pow2(__fmaf_rn(top, cxprod::kLog2e, -base)) + ((add[0] + add[1]) + (add[2] + add[3]));   // (top = -inf: 0)
      top = m[0];
    }
    if (in) p.part[part * p.m + row] = make_float2(top, sum);
    return;
  }
  if (p.mode == kProb) {
    const float lse = in ? p.lse[row] : 0.f, factor = in ? p.row_factor[row] : 0.f;
    const int64_t hot = in ? p.targets[row] - p.col0 - col0 : -1;
#pragma unroll 1
    for (int c = 0; c < WIDTH; c += 32) {
      if (col0 + c >= p.n) break;
      cxt::tmem_load32(tmem + c, r);
      cxt::tmem_load_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(cxprod::pow2(__fmaf_rn(__uint_as_float(r[j]), cxprod::kLog2e, -lse)) * factor);
      if (hot >= c && hot < c + 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (hot == c + j) r[j] = __float_as_uint(__uint_as_float(r[j]) - factor);
      }
      if (factor == 0.f) {                 // a row that does not count, whatever its logits are
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = 0;
      }
      store32<T>(t, row0, col0 + c, scratch, r);
    }
    return;
  }
  const bool plain = p.mode == kOut && !t.partial && !p.has_addend && !p.bias && !p.pre && !p.residual && p.act == CX_ACT_NONE;
  const float scale = plain && p.scale ? *p.scale : 1.f;
#pragma unroll 1
  for (int c = 0; c < WIDTH; c += 32) {
    if (col0 + c >= p.n) break;
    cxt::tmem_load32(tmem + c, r);
    cxt::tmem_load_wait();
    if (plain) {
#pragma unroll
      for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * scale);
      store32<T>(t, row0, col0 + c, scratch, r);
    } else {
      finish32<T>(t, split, row0, col0 + c, scratch, r);
    }
  }
}

template <int CG, int BN, int LAYOUT>
__global__ void __launch_bounds__(kThreads, 1)
tensor_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ Plan t) {
  using S = Shape<CG, BN>;
  extern __shared__ char shared_raw[];
  char* shared = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~(uintptr_t)1023);
  char* stages = shared;
  float* scratch = reinterpret_cast<float*>(shared + S::kStages * S::kStage);
  uint64_t* bars = reinterpret_cast<uint64_t*>(shared + S::kStages * S::kStage + kScratch);
  const uint32_t bar_full = cx::smem_u32(bars), bar_empty = bar_full + 8 * S::kStages, bar_sums = bar_empty + 8 * S::kStages,
                 bar_taken = bar_sums + 16, tmem_cell = bar_taken + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cxt::cluster_rank() : 0;
  const int units = t.tiles_m * t.tiles_n * t.splits, first = blockIdx.x / CG, step = gridDim.x / CG;
  cx::pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      cx::mbar_init(bars + i, 1);
      cx::mbar_init(bars + S::kStages + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      cx::mbar_init(bars + 2 * S::kStages + i, 1);
      cx::mbar_init(bars + 2 * S::kStages + 2 + i, kFinish * CG);
    }
    cxt::fence_barrier_init();
    cxt::prefetch_map(&map_a);
    cxt::prefetch_map(&map_b);
  }
  if (warp == 2) cxt::tmem_alloc<CG>(tmem_cell, S::kColumns);
  cxt::fence_before_sync();
  if (CG == 2) cxt::cluster_sync();
  else __syncthreads();
  cxt::fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(bars + 2 * S::kStages + 4);
  cx::pdl_wait();                        // everything above needs nothing from the kernel in front
  bool gave_up = false;

  if (warp == 0 && lane == 0) {
    int stage = 0;
    uint32_t phase = 0, filled = 0;
    for (int u = first; u < units && !gave_up; u += step) {
      const Unit w = unit_of(t, u);
      const int m0 = (w.tm * CG + (int)rank) * 128, n0 = w.tn * BN + (int)rank * (BN / CG);
      for (int s = w.s0; s < w.s1; ++s) {
        if (!cxt::wait(bar_empty + 8 * stage, phase ^ 1u)) {
          gave_up = true;
          break;
        }
        const uint32_t full = CG == 2 ? cxt::in_cta(bar_full + 8 * stage, 0) : bar_full + 8 * stage;
        if (rank == 0) cxt::expect_bytes(bar_full + 8 * stage, CG * S::kStage);
        const uint32_t a = cx::smem_u32(stages + stage * S::kStage), b = a + S::kA;
        if (LAYOUT == kTN) {
#pragma unroll
          for (int i = 0; i < 2; ++i) cxt::load_tile<CG>(a + i * 8192, &map_a, m0 + 64 * i, s * kDepth, full);
        } else {
          cxt::load_tile<CG>(a, &map_a, s * kDepth, m0, full);
        }
        if (LAYOUT == kNT) {
          cxt::load_tile<CG>(b, &map_b, s * kDepth, n0, full);
        } else {
#pragma unroll
          for (int i = 0; i < BN / CG / 64; ++i) cxt::load_tile<CG>(b + i * 8192, &map_b, n0 + 64 * i, s * kDepth, full);
        }
        ++filled;
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // until the stages are free again: no copy is in flight, and no arrival of the pair's on its way, when the CTA ends
    for (int i = 0; i < S::kStages && i < (int)filled; ++i) {
      if (--stage < 0) {
        stage = S::kStages - 1;
        phase ^= 1u;
      }
      if (!cxt::wait(bar_empty + 8 * stage, phase)) {
        gave_up = true;
        break;
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    const uint32_t instr = cxt::instruction(t.p.dtype == CX_BF16, LAYOUT == kTN, LAYOUT != kNT, 128 * CG, BN);
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    for (int u = first; u < units && !gave_up; u += step, ++turn) {
      const Unit w = unit_of(t, u);
      if (!cxt::wait(bar_taken + 8 * (turn & 1), ((turn >> 1) & 1) ^ 1u)) {
        gave_up = true;
        break;
      }
      cxt::fence_after_sync();
      const uint32_t sums = tmem + (turn & 1) * BN;
      for (int s = w.s0; s < w.s1; ++s) {
        if (!cxt::wait(bar_full + 8 * stage, phase)) {
          gave_up = true;
          break;
        }
        cxt::fence_after_sync();
        const uint32_t a = cx::smem_u32(stages + stage * S::kStage), b = a + S::kA;
#pragma unroll
        for (int k = 0; k < kDepth / 16; ++k)         // 16 of k: 32 bytes along a line, or 16 lines
          cxt::mma<CG>(sums, cxt::smem_operand(a + k * (LAYOUT == kTN ? 2048 : 32), LAYOUT == kTN ? 8192 : 16),
                       cxt::smem_operand(b + k * (LAYOUT != kNT ? 2048 : 32), LAYOUT != kNT ? 8192 : 16), instr, s > w.s0 || k > 0);
        cxt::commit<CG>(bar_empty + 8 * stage);
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      cxt::commit<CG>(bar_sums + 8 * (turn & 1));
    }
  } else if (warp >= 4) {
    const uint32_t taken = CG == 2 ? cxt::in_cta(bar_taken, 0) : bar_taken;
    float* mine = scratch + (warp - 4) * 32 * kPitch;
    int turn = 0;
    for (int u = first; u < units; u += step, ++turn) {
      const Unit w = unit_of(t, u);
      if (!cxt::wait(bar_sums + 8 * (turn & 1), (turn >> 1) & 1)) {
        gave_up = true;
        break;
      }
      cxt::fence_after_sync();
      const int quarter = warp % 4, half = (warp - 4) / 4;
      const int64_t row0 = (int64_t)(w.tm * CG + (int)rank) * 128 + quarter * 32, col0 = (int64_t)w.tn * BN + half * (BN / 2);
      const uint32_t at = tmem + (turn & 1) * BN + half * (BN / 2) + ((uint32_t)quarter * 32u << 16);
      if (t.p.dtype == CX_BF16) finish_part<__nv_bfloat16, BN / 2>(t, w.split, 2 * w.tn + half, row0, col0, at, mine);
      else finish_part<__half, BN / 2>(t, w.split, 2 * w.tn + half, row0, col0, at, mine);
      cxt::fence_before_sync();
      __syncwarp();
      if (lane == 0) cxt::arrive_cluster(taken + 8 * (turn & 1));
    }
  }
  if (gave_up) *reinterpret_cast<volatile uint32_t*>(t.status) = CX_ST_TIMEOUT;
  __syncwarp();
  cxt::fence_before_sync();
  if (CG == 2) cxt::cluster_sync();
  else __syncthreads();
  cxt::fence_after_sync();
  if (warp == 2) cxt::tmem_free<CG>(tmem, S::kColumns);
}

// the splits' sums, added in their order, and the rest of the epilogue
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_splits_kernel(const __grid_constant__ Plan t) {
  cx::pdl_trigger();
  cx::pdl_wait();
  const int64_t per = t.part_ld / 8, i = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x;
  if (i >= t.p.m * per) return;
  const int64_t row = i / per, col = i % per * 8;
  float v[8] = {};
  for (int s = 0; s < t.splits; ++s) {
    const float* at = t.partial + ((int64_t)s * t.p.m + row) * t.part_ld + col;
    const float4 lo = *reinterpret_cast<const float4*>(at), hi = *reinterpret_cast<const float4*>(at + 4);
    v[0] += lo.x; v[1] += lo.y; v[2] += lo.z; v[3] += lo.w;
    v[4] += hi.x; v[5] += hi.y; v[6] += hi.z; v[7] += hi.w;
  }
  finish<T, 1>(t, row, 1, col, v);
}

// ---- host ----------------------------------------------------------------------------------------------------------

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      p = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// a matrix of `rows` rows of `cols` elements, `ld` apart, copied in boxes of `box_rows` rows of 64 elements
int make_map(CUtensorMap* map, const void* base, int dtype, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {kDepth, (cuuint32_t)box_rows}, step[2] = {1, 1};
  EncodeTiled encode = encode_tiled();
  if (!encode) return cx_set_error("cx_product: this driver has no tile copies", 0);
  if (encode(map, dtype == CX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims,
             strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cx_set_error("cx_product: an operand cannot be described to the tile copies", 0);
  return 0;
}

// a word that kernels set and the host reads
uint32_t* status_word(bool host) {
  static uint32_t* word = [] {
    void* p = nullptr;
    if (cudaHostAlloc(&p, 64, cudaHostAllocMapped | cudaHostAllocPortable) != cudaSuccess) return static_cast<uint32_t*>(nullptr);
    *static_cast<uint32_t*>(p) = 0;
    return static_cast<uint32_t*>(p);
  }();
  if (host || !word) return word;
  void* d = nullptr;
  return cudaHostGetDevicePointer(&d, word, 0) == cudaSuccess ? static_cast<uint32_t*>(d) : nullptr;
}

struct Choice {
  int cg, bn, splits;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

Choice choose(const CxProduct& p) {
  const int64_t slices = ceil_div(p.k, kDepth);
  Choice best = {1, 128, 1};
  if (p.mode == kStats || p.mode == kProb) {
    if (ceil_div(p.m, 256) * ceil_div(p.n, 256) >= 74) best = {2, 256, 1};
    return best;
  }
  if (ceil_div(p.m, 256) * ceil_div(p.n, 256) >= 60) return {2, 256, 1};
  const int64_t tiles = ceil_div(p.m, 128) * ceil_div(p.n, 128);
  if (tiles < 74) best.bn = 64;
  const int64_t now = ceil_div(p.m, 128) * ceil_div(p.n, best.bn);
  int64_t splits = 148 / now;
  if (splits > slices / 8) splits = slices / 8;
  best.splits = (int)(splits < 1 ? 1 : splits);
  return best;
}

template <int CG, int BN, int LAYOUT>
int launch(Plan& t, cudaStream_t s) {
  using S = Shape<CG, BN>;
  CUtensorMap a, b;
  const CxProduct& p = t.p;
  int rc = LAYOUT == kTN ? make_map(&a, p.a, p.dtype, p.k, p.m, p.lda, kDepth) : make_map(&a, p.a, p.dtype, p.m, p.k, p.lda, 128);
  if (rc) return rc;
  rc = LAYOUT == kNT ? make_map(&b, p.b, p.dtype, p.n, p.k, p.ldb, BN / CG) : make_map(&b, p.b, p.dtype, p.k, p.n, p.ldb, kDepth);
  if (rc) return rc;
  static const int ready = (int)cudaFuncSetAttribute(tensor_product_kernel<CG, BN, LAYOUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
  if (ready) return cx_set_error("cx_product", ready);
  const int64_t units = (int64_t)t.tiles_m * t.tiles_n * t.splits, most = cx_sm_count() / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CG * (units < most ? units : most)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cx_pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, tensor_product_kernel<CG, BN, LAYOUT>, a, b, t);
  cx_note_launch();
  return e == cudaSuccess ? 0 : cx_set_error("cx_product", (int)e);
}

template <int CG, int BN>
int launch_layout(Plan& t, cudaStream_t s) {
  switch (t.p.layout) {
    case kNT: return launch<CG, BN, kNT>(t, s);
    case kNN: return launch<CG, BN, kNN>(t, s);
    default: return launch<CG, BN, kTN>(t, s);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

bool cx_tensor_product_takes(const CxProduct& p) {
  return p.dtype != CX_F32 && aligned16(p.a) && aligned16(p.b) && p.lda % 8 == 0 && p.ldb % 8 == 0;
}
int cx_tensor_product_stat_columns(const CxProduct& p) { return choose(p).bn / 2; }
int64_t cx_tensor_product_workspace_bytes(const CxProduct& p) {
  const Choice c = choose(p);
  return c.splits > 1 ? c.splits * p.m * ((p.n + 7) / 8 * 8) * 4 : 0;
}

int cx_tensor_product(const CxProduct& p, cudaStream_t s) {
  const Choice c = choose(p);
  uint32_t* said = status_word(true);
  if (!said) return cx_set_error("cx_product: no pinned memory for the status word", 0);
  if (*reinterpret_cast<volatile uint32_t*>(said)) {
    *reinterpret_cast<volatile uint32_t*>(said) = 0;
    return cx_set_error("cx_product: an earlier product gave up waiting, its results are not valid", 0);
  }
  if (ceil_div(p.m, 128 * c.cg) * ceil_div(p.n, c.bn) > 0x7FFFFFFF / (c.splits + 1))
    return cx_set_error("cx_product: too many tiles", 0);
  Plan t = {};
  t.p = p;
  t.tiles_m = (int)ceil_div(p.m, 128 * c.cg);
  t.tiles_n = (int)ceil_div(p.n, c.bn);
  t.slices = (int)ceil_div(p.k, kDepth);
  t.slices_per = (int)ceil_div(t.slices, c.splits);
  t.splits = (int)ceil_div(t.slices, t.slices_per);
  t.status = status_word(false);
  t.wide_out = aligned16(p.out) && aligned16(p.pre) && p.ldo % 8 == 0;
  t.wide_add = aligned16(p.addend) && p.n % 4 == 0;
  t.wide_res = aligned16(p.residual) && p.ldr % 8 == 0;
  t.wide_bias = aligned16(p.bias);
  if (t.splits > 1) {
    if (p.ws_bytes < cx_tensor_product_workspace_bytes(p)) return cx_set_error("cx_product: workspace too small", 0);
    t.partial = reinterpret_cast<float*>(p.workspace);
    t.part_ld = (p.n + 7) / 8 * 8;
  }
  int rc = c.cg == 2 ? launch_layout<2, 256>(t, s) : c.bn == 128 ? launch_layout<1, 128>(t, s) : launch_layout<1, 64>(t, s);
  if (rc || t.splits == 1) return rc;
  const int grid = (int)ceil_div(p.m * (t.part_ld / 8), kJoinThreads);
  if (p.dtype == CX_BF16) cx_launch_pdl2(join_splits_kernel<__nv_bfloat16>, dim3(grid), kJoinThreads, s, t);
  else cx_launch_pdl2(join_splits_kernel<__half>, dim3(grid), kJoinThreads, s, t);
  cx_note_launch();
  return cx_check_launch("cx_product");
}
