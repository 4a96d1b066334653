// The product of cx_product.cuh on the fifth-generation tensor cores, for 16-bit operands.
//
// A persistent grid of CTAs, or of pairs of CTAs that share a tile, walks over the output's tiles.  Two warps per
// CTA bring 64-deep slices of the operands into a ring of stages with tile copies, one per tile issues the matrix
// instructions, whose sums stay in tensor memory, and eight warps take finished sums from there: the tensor memory holds
// two tiles, so the matrix instructions of a tile run under the epilogue of the tile before.  Each layout of the operands
// is read as it lies: consecutive along k or along m and n is a bit of the instruction and another shape of the copy.
// Every wait is bounded: where one runs out, the tiles that did not come are filled with NaN and a word is set for the host.
//
// What bounds it: a pair's slice of 256 x 256 x 64 is 512 cycles of matrix instructions and 64 KB from L2, at 2.3 PFLOP/s
// while the clock is 1.9 GHz and 1.3 to 1.4 when the power limit is reached; a slice of smaller tiles about 340 cycles of
// waits and issues; a launch 4 to 6 us from its start to its first results (tensor memory 0.35, the first copies 0.5, the
// epilogue 0.7, the end 1).  8192 x 4096 x 1024 50 us, x 4096 177 us (1.55 PFLOP/s), 8192 x 1024 x 4096 50 us
// (operands from memory, after a pause).
#include <atomic>
#include <mutex>

#include "cx_product.cuh"
#include "cx_tensor.cuh"

namespace {

constexpr int kDepth = 64;               // elements of k in a stage: one 128-byte line
constexpr int kThreads = 384;            // warps 0 and 3 copy, 1 multiplies, 2 has the tensor memory, 4 to 11 finish
constexpr int kFinish = 8;               // finishing warps: four have the left half of a tile's columns, four the right one
constexpr int kJoinThreads = 256;
constexpr int kShared = 232448;          // of a CTA

template <int CG, int BN>
struct Shape {
  static constexpr int kA = 128 * kDepth * 2, kB = BN / CG * kDepth * 2, kStage = kA + kB;
  static constexpr int kBias = kFinish * BN / 2 * 4;
  static constexpr int kFit = (kShared - 1024 - 512 - kBias) / kStage;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kBytes = 1024 + 512 + kBias + kStages * kStage;
  static constexpr int kColumns = 2 * BN;
};

// Division of numbers below 2^31 by a number that is known at launch: n / d = n m >> (31 + l), l = ceil(log2 d), m =
// ceil(2^(31 + l) / d).
struct Divisor {
  uint32_t d, m, shift;
  void set(uint32_t by) {
    d = by;
    shift = 0;
    while ((1ull << shift) < by) ++shift;
    m = (uint32_t)(((1ull << (31 + shift)) + by - 1) / by);
    shift += 31;
  }
  __device__ __forceinline__ int of(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> shift); }
};

struct Job {
  CxProduct p;
  int tiles_m, tiles_n, units;
  Divisor tiles, per, group, last;   // tiles; tiles of a group: `group` rows of tiles (the last one: `last`) are walked
                                     // together, column after column
  int slices, slices_per;      // of kDepth along k: all, and per split
  float* partial;              // sums of the splits: [split][m][part_ld]
  int64_t part_ld;
  int splits;
  int wide_out, wide_pre, wide_res, wide_bias;   // alignment of their rows: 2 for 32 bytes, 1 for 16, 0 for less
  int plain;                   // kOut with nothing to it but a factor
};

// The units of the first job go round the workers, those of the second one fill up: `extra` workers have one more of the
// first and take `few` of the second, the others `many`.
struct Plan {
  Job job[2];
  int extra, few, many;
  uint32_t* status;            // set when a wait has run out
};

struct Walk {
  const Plan& t;
  int worker, workers, job, u, end;
  __device__ __forceinline__ Walk(const Plan& plan, int w, int n) : t(plan), worker(w), workers(n), job(0), u(w), end(plan.job[0].units) {
    if (u >= end) second();
  }
  __device__ __forceinline__ void second() {
    job = 1;
    u = worker < t.extra ? worker * t.few : t.extra * t.few + (worker - t.extra) * t.many;
    end = min(u + (worker < t.extra ? t.few : t.many), t.job[1].units);
  }
  __device__ __forceinline__ bool more() const { return u < end; }
  __device__ __forceinline__ void next() {
    u += job ? 1 : workers;
    if (!job && u >= end) second();
  }
};

struct Unit {
  int tm, tn, split, s0, s1;
};
__device__ __forceinline__ Unit unit_of(const Job& t, int u) {
  Unit r;
  r.split = t.tiles.of(u);
  const int tile = u - r.split * (int)t.tiles.d, g = t.per.of(tile), in = tile - g * (int)t.per.d, first = g * (int)t.group.d;
  const Divisor& rows = first + (int)t.group.d <= t.tiles_m ? t.group : t.last;
  r.tn = rows.of(in);
  r.tm = first + in - r.tn * (int)rows.d;
  r.s0 = r.split * t.slices_per;
  r.s1 = min(t.slices, r.s0 + t.slices_per);
  return r;
}

// ---- neighbouring columns of one row: a lane has a row, so it moves whole 32-byte sectors ---------------------------
__device__ __forceinline__ void load_words8(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
}
__device__ __forceinline__ void store_words8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, int W>
__device__ __forceinline__ void store_row(T* at, int wide, int left, const float (&v)[W]) {
  if (left >= W && wide) {
    uint32_t w[W / 2];
#pragma unroll
    for (int i = 0; i < W / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    if (W >= 16 && wide == 2) {
#pragma unroll
      for (int i = 0; i < W / 16; ++i) store_words8(at + 16 * i, w + 8 * i);
    } else {
#pragma unroll
      for (int i = 0; i < W / 8; ++i) reinterpret_cast<uint4*>(at)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < left) at[i] = cx::Elem<T>::from_f(v[i]);
  }
}
template <typename T, int W>
__device__ __forceinline__ void add_row(const T* at, int wide, int left, float (&v)[W]) {
  if (left >= W && wide) {
    uint32_t w[W / 2];
    if (W >= 16 && wide == 2) {
#pragma unroll
      for (int i = 0; i < W / 16; ++i) load_words8(at + 16 * i, reinterpret_cast<uint32_t(&)[8]>(w[8 * i]));
    } else {
#pragma unroll
      for (int i = 0; i < W / 8; ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(at)[i];
        w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
      }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += cx::Elem<T>::to_f(reinterpret_cast<const T*>(w)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < left) v[i] += cx::Elem<T>::to_f(at[i]);
  }
}
// 32-bit sums in aligned rows, whole groups of 8
template <int W>
__device__ __forceinline__ void store_sums(float* at, int left, const float (&v)[W]) {
#pragma unroll
  for (int i = 0; i < W / 8; ++i)
    if (8 * i < left) store_words8(at + 8 * i, reinterpret_cast<const uint32_t*>(v) + 8 * i);
}
template <int W>
__device__ __forceinline__ void add_sums(const float* at, int left, float (&v)[W]) {
#pragma unroll
  for (int i = 0; i < W / 8; ++i)
    if (8 * i < left) {
      uint32_t w[8];
      load_words8(at + 8 * i, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[8 * i + k] += __uint_as_float(w[k]);
    }
}

// What the descriptor says of a row's results from column `col` on, in registers: read from the descriptor for each few
// columns it took 880 cycles for 16 of them.
template <typename T>
struct Row {
  T *out, *pre;
  const T *residual, *bias;
  float* addend;
  float scale;
  int left, act, wide_out, wide_pre, wide_res, wide_bias;
  __device__ __forceinline__ Row(const Job& t, int64_t row, int64_t col) {
    const CxProduct& p = t.p;
    out = reinterpret_cast<T*>(p.out) + row * p.ldo + col;
    pre = p.pre ? reinterpret_cast<T*>(p.pre) + row * p.ldpre + col : nullptr;
    residual = p.residual ? reinterpret_cast<const T*>(p.residual) + row * p.ldr + col : nullptr;
    bias = p.bias ? reinterpret_cast<const T*>(p.bias) + col : nullptr;
    addend = p.addend + row * p.ldadd + col;
    scale = p.scale ? *p.scale : 1.f;
    left = (int)min((int64_t)0x40000000, p.n - col);
    act = p.act;
    wide_out = t.wide_out;
    wide_pre = t.wide_pre;
    wide_res = t.wide_res;
    wide_bias = t.wide_bias;
  }
};

// A finishing warp's part of a tile, 32 rows, one per lane, 32 columns at a time.  The loop is not unrolled: fetching
// instructions that a tile needs once costs more than they do.
template <int WIDTH, typename F>
__device__ __forceinline__ void each32(uint32_t tmem, int left, const F& work) {
#pragma unroll 1
  for (int c = 0; c < WIDTH && c < left; c += 32) {
    uint32_t r[32];
    cxt::tmem_load32(tmem + c, r);
    cxt::tmem_load_wait(r);
    work(c, reinterpret_cast<float(&)[32]>(r));
  }
}

template <typename T, int WIDTH>
__device__ __forceinline__ void finish_stats(const Job& t, const Unit& u, int half, int64_t row, int64_t col0, uint32_t tmem) {
  const CxProduct& p = t.p;
  const bool in = row < p.m;
  const int left = (int)min((int64_t)WIDTH, p.n - col0);
  const int64_t hot = (in ? p.targets[row] : -1) - p.col0 - col0;      // where the row's target is in this part
  float top = -INFINITY, sum = 0.f;
  each32<WIDTH>(tmem, left, [&](int c, float(&v)[32]) {
    if (c + 32 > left) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j >= left) v[j] = -INFINITY;
    }
    if (hot >= c && hot < c + 32) {
      float x = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (hot == c + j) x = v[j];
      p.target_logit[row] = x;
    }
    float m[4] = {top, top, top, top}, add[4] = {};
#pragma unroll
    for (int j = 0; j < 32; ++j) m[j % 4] = fmaxf(m[j % 4], v[j]);
    m[0] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    const float base = (m[0] == -INFINITY ? 0.f : m[0]) * cxprod::kLog2e;
#pragma unroll
    for (int j = 0; j < 32; ++j) add[j % 4] += cxprod::pow2(__fmaf_rn(v[j], cxprod::kLog2e, -base));
    sum = sum * cxprod::pow2(__fmaf_rn(top, cxprod::kLog2e, -base)) + ((add[0] + add[1]) + (add[2] + add[3]));   // (top = -inf: 0)
    top = m[0];
  });
  if (in) p.part[(2ll * u.tn + half) * p.m + row] = make_float2(top, sum);
}

template <typename T, int WIDTH>
__device__ __forceinline__ void finish_prob(const Job& t, int64_t row, int64_t col0, uint32_t tmem) {
  const CxProduct& p = t.p;
  const bool in = row < p.m;
  const int left = (int)min((int64_t)WIDTH, p.n - col0), wide = t.wide_out;
  const float lse = in ? p.lse[row] : 0.f, factor = in ? p.row_factor[row] : 0.f;
  const int64_t hot = in ? p.targets[row] - p.col0 - col0 : -1;
  T* out = reinterpret_cast<T*>(p.out) + row * p.ldo + col0;
  each32<WIDTH>(tmem, left, [&](int c, float(&v)[32]) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = cxprod::pow2(__fmaf_rn(v[j], cxprod::kLog2e, -lse)) * factor;
    if (hot >= c && hot < c + 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (hot == c + j) v[j] -= factor;
    }
    if (factor == 0.f) {                 // a row that does not count, whatever its logits are
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = 0.f;
    }
    if (in) store_row(out + c, wide, left - c, v);
  });
}

// kOut without anything to it but a factor
template <typename T, int WIDTH>
__device__ __forceinline__ void finish_plain(const Job& t, int64_t row, int64_t col0, uint32_t tmem) {
  const CxProduct& p = t.p;
  const bool in = row < p.m;
  const int left = (int)min((int64_t)WIDTH, p.n - col0), wide = t.wide_out;
  const float scale = p.scale ? *p.scale : 1.f;
  T* out = reinterpret_cast<T*>(p.out) + row * p.ldo + col0;
  each32<WIDTH>(tmem, left, [&](int c, float(&v)[32]) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= scale;
    if (in) store_row(out + c, wide, left - c, v);
  });
}

// 32-bit sums: of a split, or those that a later product goes on with
template <int WIDTH>
__device__ __forceinline__ void finish_sums(float* at, bool add, bool in, int left, uint32_t tmem) {
  each32<WIDTH>(tmem, left, [&](int c, float(&v)[32]) {
    if (!in) return;
    if (add) add_sums(at + c, left - c, v);
    store_sums(at + c, left - c, v);
  });
}

// kOut with all that can be in it.  The residual's next 32 columns are on their way while these are worked on.
template <typename T, int WIDTH>
__device__ __forceinline__ void finish_linear(const Job& t, int64_t row, int64_t col0, uint32_t tmem, const float* bias) {
  const Row<T> to(t, row, col0);
  const bool in = row < t.p.m, add = t.p.has_addend, ahead = to.residual && to.wide_res == 2 && in && to.left >= WIDTH;
  uint32_t next[16];
  if (ahead) {
    load_words8(to.residual, reinterpret_cast<uint32_t(&)[8]>(next[0]));
    load_words8(to.residual + 16, reinterpret_cast<uint32_t(&)[8]>(next[8]));
  }
  each32<WIDTH>(tmem, min(to.left, WIDTH), [&](int c, float(&v)[32]) {
    const int have = to.left - c;
    if (add && in) add_sums(to.addend + c, have, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 b = reinterpret_cast<const float4*>(bias + c)[i];      // zeros where there is none
      v[4 * i] = __fmaf_rn(v[4 * i], to.scale, b.x);
      v[4 * i + 1] = __fmaf_rn(v[4 * i + 1], to.scale, b.y);
      v[4 * i + 2] = __fmaf_rn(v[4 * i + 2], to.scale, b.z);
      v[4 * i + 3] = __fmaf_rn(v[4 * i + 3], to.scale, b.w);
    }
    if (to.pre && in) store_row(to.pre + c, to.wide_pre, have, v);
    cxprod::activate<T>(v, to.act);
    if (ahead) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += cx::Elem<T>::to_f(reinterpret_cast<const T*>(next)[i]);
      if (c + 32 < WIDTH) {
        load_words8(to.residual + c + 32, reinterpret_cast<uint32_t(&)[8]>(next[0]));
        load_words8(to.residual + c + 48, reinterpret_cast<uint32_t(&)[8]>(next[8]));
      }
    } else if (to.residual && in) {
      add_row(to.residual + c, to.wide_res, have, v);
    }
    if (in) store_row(to.out + c, to.wide_out, have, v);
  });
}

// A finishing warp's part of a tile: rows row0 to row0 + 31, WIDTH columns from col0 on.
template <typename T, int WIDTH>
__device__ __forceinline__ void finish_part(const Job& t, const Unit& u, int half, int64_t row0, int64_t col0, uint32_t tmem, const float* bias) {
  const CxProduct& p = t.p;
  const int64_t row = row0 + (threadIdx.x & 31);
  if (col0 >= p.n) return;
  const int left = (int)min((int64_t)WIDTH, p.n - col0);
  if (p.mode == kStats) return finish_stats<T, WIDTH>(t, u, half, row, col0, tmem);
  if (p.mode == kProb) return finish_prob<T, WIDTH>(t, row, col0, tmem);
  if (t.partial) return finish_sums<WIDTH>(t.partial + ((int64_t)u.split * p.m + row) * t.part_ld + col0, false, row < p.m, left, tmem);
  if (p.mode == kSums) return finish_sums<WIDTH>(p.addend + row * p.ldadd + col0, p.has_addend, row < p.m, left, tmem);
  if (t.plain) return finish_plain<T, WIDTH>(t, row, col0, tmem);
  finish_linear<T, WIDTH>(t, row, col0, tmem, bias);
}

// What a finishing warp leaves of its part of a tile when the sums never came: no numbers, so that nothing that follows can take
// the call for a valid one.  (The host learns of it at the device's next product.)
template <int WIDTH>
__device__ __noinline__ void spoil_part(const Job& t, const Unit& u, int half, int64_t row, int64_t col0) {
  const CxProduct& p = t.p;
  if (row >= p.m || col0 >= p.n) return;
  const int left = (int)min((int64_t)WIDTH, p.n - col0);
  if (p.mode == kStats) {
    p.part[(2ll * u.tn + half) * p.m + row] = make_float2(-INFINITY, NAN);
    return;
  }
  float* sums = t.partial ? t.partial + ((int64_t)u.split * p.m + row) * t.part_ld + col0 : p.mode == kSums ? p.addend + row * p.ldadd + col0 : nullptr;
  uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + row * p.ldo + col0;
  uint16_t* pre = p.mode == kOut && p.pre ? reinterpret_cast<uint16_t*>(p.pre) + row * p.ldpre + col0 : nullptr;
  for (int i = 0; i < left; ++i) {
    if (sums) {
      sums[i] = NAN;
    } else {
      out[i] = 0x7FFF;                 // no number in bf16 and in fp16
      if (pre) pre[i] = 0x7FFF;
    }
  }
}

template <int CG, int BN>
__global__ void __launch_bounds__(kThreads, 1)
tensor_product_kernel(const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_b0,
                      const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_b1, const __grid_constant__ Plan t) {
  using S = Shape<CG, BN>;
  extern __shared__ char shared_raw[];
  char* shared = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~(uintptr_t)1023);
  char* stages = shared;
  uint64_t* bars = reinterpret_cast<uint64_t*>(shared + S::kStages * S::kStage + S::kBias);
  const uint32_t bar_full = cx::smem_u32(bars), bar_empty = bar_full + 8 * S::kStages, bar_sums = bar_empty + 8 * S::kStages,
                 bar_taken = bar_sums + 16, tmem_cell = bar_taken + 16;
  const int warp = __shfl_sync(0xFFFFFFFFu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cxt::cluster_rank() : 0;
  Walk w(t, blockIdx.x / CG, gridDim.x / CG);
  Unit u = unit_of(t.job[w.job], w.u);       // (under the allocation below)
  cx::pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      cx::mbar_init(bars + i, 2);
      cx::mbar_init(bars + S::kStages + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      cx::mbar_init(bars + 2 * S::kStages + i, 1);
      cx::mbar_init(bars + 2 * S::kStages + 2 + i, kFinish * CG);
    }
    cxt::fence_barrier_init();
    cxt::prefetch_map(&map_a0);
    cxt::prefetch_map(&map_b0);
  }
  if (warp == 2) cxt::tmem_alloc<CG>(tmem_cell, S::kColumns);
  cxt::fence_before_sync();
  if (CG == 2) cxt::cluster_sync();
  else __syncthreads();
  cxt::fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(bars + 2 * S::kStages + 4);
  cx::pdl_wait();                        // everything above needs nothing from the kernel in front
  bool gave_up = false;

  if (warp == 0 || warp == 3) {
    // Each has an operand: a turn of such a loop takes 200 cycles whatever it copies, a slice's matrix instructions 128
    // to 512 (one warp for both operands: 360 a slice).
    const bool is_b = warp == 3;
    const uint32_t lead_full = CG == 2 ? cxt::in_cta(bar_full, 0) : bar_full;      // the pair's matrix instructions wait there
    const uint32_t base = cx::smem_u32(stages) + (is_b ? S::kA : 0), bytes = CG * (is_b ? S::kB : S::kA);
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool ready = true;
    for (; w.more(); w.next()) {
      const Job& job = t.job[w.job];
      if (filled) u = unit_of(job, w.u);
      const CUtensorMap* map = is_b ? (w.job ? &map_b1 : &map_b0) : (w.job ? &map_a1 : &map_a0);
      const bool across = is_b ? job.p.layout != kNT : job.p.layout == kTN;          // consecutive along m or n, not along k
      const int first = is_b ? u.tn * BN + (int)rank * (BN / CG) : (u.tm * CG + (int)rank) * 128;
      const int boxes = !across ? 1 : is_b ? BN / CG / 64 : 2;
      for (int s = u.s0; s < u.s1; ++s) {
        // a lane whose wait has run out copies nothing more and waits no more; the warp stays together
        if (!ready && !gave_up) gave_up = !cxt::wait(bar_empty + 8 * stage, phase ^ 1u);
        const uint32_t full = lead_full + 8 * stage, at = base + stage * S::kStage, own = bar_full + 8 * stage;
        if (filled < S::kStages) ++filled;
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
        ready = filled < S::kStages || cxt::look(bar_empty + 8 * stage, phase ^ 1u);
        if (cxt::elect_one() && !gave_up) {
          if (rank == 0) cxt::expect_bytes(own, bytes);
          if (!across) {
            cxt::load_tile<CG>(at, map, s * kDepth, first, full);
          } else {
#pragma unroll 1
            for (int i = 0; i < boxes; ++i) cxt::load_tile<CG>(at + i * 8192, map, first + 64 * i, s * kDepth, full);
          }
        }
        __syncwarp();
      }
    }
    // until the stages are free again: no copy is in flight, and no arrival of the pair's on its way, when the CTA ends
    for (int i = 0; i < filled; ++i) {
      if (--stage < 0) {
        stage = S::kStages - 1;
        phase ^= 1u;
      }
      if (!gave_up) gave_up = !cxt::wait(bar_empty + 8 * stage, phase);
    }
  } else if (warp == 1 && rank == 0) {
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    bool ready = false;
    for (; w.more(); w.next(), ++turn) {
      const Job& job = t.job[w.job];
      if (turn) u = unit_of(job, w.u);
      const bool along_m = job.p.layout == kTN, along_n = job.p.layout != kNT;
      const uint32_t instr = cxt::instruction(job.p.dtype == CX_BF16, along_m, along_n, 128 * CG, BN);
      // 16 of k: 32 bytes along a line, or 16 lines
      const uint32_t step_a = along_m ? 128 : 2, step_b = along_n ? 128 : 2;
      const uint32_t first_a = cxt::operand_at(cx::smem_u32(stages), along_m ? 8192 : 16);
      const uint32_t first_b = cxt::operand_at(cx::smem_u32(stages) + S::kA, along_n ? 8192 : 16);
      if (!gave_up) gave_up = !cxt::wait(bar_taken + 8 * (turn & 1), ((turn >> 1) & 1) ^ 1u);
      cxt::fence_after_sync();
      const uint32_t sums = tmem + (turn & 1) * BN;
      for (int s = u.s0; s < u.s1; ++s) {
        if (!ready && !gave_up) gave_up = !cxt::wait(bar_full + 8 * stage, phase);
        cxt::fence_after_sync();
        const uint32_t a = first_a + stage * (S::kStage >> 4), b = first_b + stage * (S::kStage >> 4), free = bar_empty + 8 * stage;
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
        ready = cxt::look(bar_full + 8 * stage, phase);
        if (cxt::elect_one() && !gave_up) {
#pragma unroll
          for (int k = 0; k < kDepth / 16; ++k) cxt::mma<CG>(sums, a + k * step_a, b + k * step_b, instr, s > u.s0 || k > 0);
          cxt::commit<CG>(free);
        }
        __syncwarp();
      }
      if (cxt::elect_one() && !gave_up) cxt::commit<CG>(bar_sums + 8 * (turn & 1));
      __syncwarp();
    }
  } else if (warp >= 4) {
    const uint32_t taken = CG == 2 ? cxt::in_cta(bar_taken, 0) : bar_taken;
    const int quarter = warp % 4, half = (warp - 4) / 4;
    float* bias = reinterpret_cast<float*>(shared + S::kStages * S::kStage) + (warp - 4) * (BN / 2);
    int turn = 0;
    for (; w.more(); w.next(), ++turn) {
      const Job& job = t.job[w.job];
      if (turn) u = unit_of(job, w.u);
      const int64_t row0 = (int64_t)(u.tm * CG + (int)rank) * 128 + quarter * 32, col0 = (int64_t)u.tn * BN + half * (BN / 2);
      if (!job.plain && job.p.mode == kOut && !job.partial) {      // before the sums are there: nothing waits for it
        for (int i = lane; i < BN / 2; i += 32) {
          const bool have = job.p.bias && col0 + i < job.p.n;
          bias[i] = !have ? 0.f : job.p.dtype == CX_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(job.p.bias)[col0 + i])
                                                         : __half2float(reinterpret_cast<const __half*>(job.p.bias)[col0 + i]);
        }
        __syncwarp();
      }
      if (!cxt::wait_together(bar_sums + 8 * (turn & 1), (turn >> 1) & 1)) {
        gave_up = true;
        break;
      }
      __syncwarp();
      cxt::fence_after_sync();
      const uint32_t at = tmem + (turn & 1) * BN + half * (BN / 2) + ((uint32_t)quarter * 32u << 16);
      if (job.p.dtype == CX_BF16) finish_part<__nv_bfloat16, BN / 2>(job, u, half, row0, col0, at, bias);
      else finish_part<__half, BN / 2>(job, u, half, row0, col0, at, bias);
      cxt::fence_before_sync();
      __syncwarp();
      if (lane == 0) cxt::arrive_cluster(taken + 8 * (turn & 1));
    }
    if (gave_up) {                       // this unit's sums, and those of all that would have followed
      for (; w.more(); w.next()) {
        const Unit left = unit_of(t.job[w.job], w.u);
        spoil_part<BN / 2>(t.job[w.job], left, half, (int64_t)(left.tm * CG + (int)rank) * 128 + quarter * 32 + lane, (int64_t)left.tn * BN + half * (BN / 2));
      }
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

// the splits' sums, added in their order, and the rest of the epilogue; a block has a part of one of the jobs
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_splits_kernel(const __grid_constant__ Plan t) {
  cx::pdl_trigger();
  cx::pdl_wait();
  const Job& job = t.job[blockIdx.y];
  if (!job.partial) return;
  const int64_t per = job.part_ld / 8, i = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x;
  if (i >= job.p.m * per) return;
  const int64_t row = i / per, col = i % per * 8;
  float v[8] = {};
  for (int s = 0; s < job.splits; ++s) add_sums(job.partial + ((int64_t)s * job.p.m + row) * job.part_ld + col, 8, v);
  const Row<T> to(job, row, col);
  if (job.p.has_addend) add_sums(to.addend, to.left, v);
  if (job.p.mode == kSums) return store_sums(to.addend, to.left, v);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] *= to.scale;
  if (to.bias) add_row(to.bias, to.wide_bias, to.left, v);
  if (to.pre) store_row(to.pre, to.wide_pre, to.left, v);
  cxprod::activate<T>(v, to.act);
  if (to.residual) add_row(to.residual, to.wide_res, to.left, v);
  store_row(to.out, to.wide_out, to.left, v);
}

// Rows of the jobs' results from aligned rows in the workspace to where they belong, neighbouring elements by neighbouring
// threads: what a result whose rows are not 16-byte aligned goes through.  (A lane per row, element by element, the
// 8192 x 50257 logits took 4.1 ms.)
struct Spread {
  const uint16_t* from[2];
  uint16_t* to[2];
  int64_t rows[2], cols[2], from_ld[2], to_ld[2];
};
__global__ void __launch_bounds__(kJoinThreads) spread_kernel(const __grid_constant__ Spread d) {
  cx::pdl_trigger();
  cx::pdl_wait();
  const int j = blockIdx.y;
  for (int64_t row = blockIdx.x; row < d.rows[j]; row += gridDim.x) {
    const uint16_t* from = d.from[j] + row * d.from_ld[j];
    uint16_t* to = d.to[j] + row * d.to_ld[j];
    // single elements up to a 4-byte boundary, then pairs
    const int64_t odd = reinterpret_cast<uintptr_t>(to) & 2 ? 1 : 0;
    if (odd && threadIdx.x == 0) to[0] = from[0];
    const int64_t pairs = (d.cols[j] - odd) / 2;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < pairs; i += kJoinThreads) {
      const uint32_t lo = from[odd + 2 * i], hi = from[odd + 2 * i + 1];
      reinterpret_cast<uint32_t*>(to + odd)[i] = lo | hi << 16;
    }
    if (threadIdx.x == 0 && odd + 2 * pairs < d.cols[j]) to[odd + 2 * pairs] = from[odd + 2 * pairs];
  }
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

// A word of the current device that its kernels set and the host reads: `host`, and where they find it.  Made at the device's
// first product, which may be under a stream's capture: allocating is not part of what is captured.
struct Word {
  uint32_t* host;
  uint32_t* device;
};
Word status_word() {
  constexpr int kDevices = 64;
  static std::atomic<uint32_t*> words[kDevices];
  static std::mutex making;
  int dev = 0;
  Word w = {nullptr, nullptr};
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return w;
  uint32_t* at = words[dev].load(std::memory_order_acquire);
  if (!at) {
    const std::lock_guard<std::mutex> lock(making);
    at = words[dev].load(std::memory_order_acquire);
    if (!at) {
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
      if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return w;
      void* p = nullptr;
      const cudaError_t e = cudaHostAlloc(&p, 64, cudaHostAllocMapped | cudaHostAllocPortable);
      cudaThreadExchangeStreamCaptureMode(&mode);
      if (e != cudaSuccess) return w;
      at = static_cast<uint32_t*>(p);
      *at = 0;
      words[dev].store(at, std::memory_order_release);
    }
  }
  void* d = nullptr;
  if (cudaHostGetDevicePointer(&d, at, 0) != cudaSuccess) return w;
  w.host = at;
  w.device = static_cast<uint32_t*>(d);
  return w;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Choice {
  int cg, bn, splits[2];
  double time;
};

// Who takes what: a unit lasts as long as its slices.  The first job's `a` units go round the workers, the second one's
// are given out so that the last worker is done as early as can be; returns that time.
int64_t share_out(int64_t a, int64_t la, int64_t b, int64_t lb, int64_t workers, int* extra, int* few, int* many) {
  const int64_t rounds = a / workers, more = a % workers, base = b * lb / workers / (lb ? lb : 1);
  int64_t f = 0, m = 0;
  // with one first unit more a worker takes la / lb fewer of the others: start below that and add the cheapest one
  if (base > 4) {
    const int64_t gap = lb ? la / lb + 2 : 0;
    m = base - 4;
    f = m > gap ? m - gap : 0;
    while (m > 0 && more * f + (workers - more) * m > b) --m;
  }
  while (more * f + (workers - more) * m < b) {
    const int64_t end_few = (rounds + 1) * la + (f + 1) * lb, end_many = rounds * la + (m + 1) * lb;
    if (!more || end_many <= end_few) ++m;
    else ++f;
  }
  *extra = (int)more;
  *few = (int)f;
  *many = (int)m;
  const int64_t t_few = more ? (rounds + 1) * la + f * lb : 0, t_many = rounds * la + m * lb;
  return t_few > t_many ? t_few : t_many;
}

// What a launch takes, in us: `fixed`, and for the last worker `slice` for each of its slices of k and `tile` for each of
// its units.  Measured alone on the GPU at 1.9 GHz: 128 x 64 tiles 5.4 / 6.5 / 13.5 us for one unit of 8 / 16 / 64 slices and
// 47 for 14 units of 16, 128 x 128 tiles 6.1 / 7.4 / 14.7 and 35 for 7 of 16, pairs' 256 x 256 tiles 7.9 / 11.6 / 24 and 29.5
// for 4 of 16; joining the splits of 1 M results 3.1 us for two, 3.9 for four.
struct Cost {
  int cg, bn;
  double fixed, slice, tile;
};
constexpr Cost kCosts[3] = {{2, 256, 5.7, 0.27, 1.3}, {1, 128, 4.2, 0.17, 1.0}, {1, 64, 3.7, 0.146, 0.65}};
constexpr double kJoin = 2.2, kJoinBytes = 6e6;      // us, and bytes of partial sums a us

// The tile and the splits along k that are done first.  A product is split where its own units are longer than an even
// share of all there is: few rows (or few results of a long sum) fill the GPU so, others are not worth the joining.
Choice search(const CxProduct* p, int count, bool sums) {
  Choice best = {};
  for (const Cost& c : kCosts) {
    const int64_t most = cx_sm_count() / c.cg;
    int64_t tiles[2] = {}, slices[2] = {}, total = 0;
    for (int i = 0; i < count; ++i) {
      tiles[i] = ceil_div(p[i].m, 128 * c.cg) * ceil_div(p[i].n, c.bn);
      slices[i] = ceil_div(p[i].k, kDepth);
      total += tiles[i] * slices[i];
    }
    int64_t limit[2] = {1, 1};
    for (int i = 0; i < count; ++i)
      if (sums && slices[i] * most > total + total / 4) limit[i] = slices[i] / 4 < 16 ? slices[i] / 4 : 16;
    for (int64_t s0 = 1; s0 == 1 || s0 <= limit[0]; s0 += s0 < 4 ? 1 : s0 / 2)
      for (int64_t s1 = 1; s1 == 1 || s1 <= limit[1]; s1 += s1 < 4 ? 1 : s1 / 2) {
        const int64_t split[2] = {s0, s1};
        int64_t units[2] = {}, len[2] = {}, all = 0;
        double join = 0;
        for (int i = 0; i < count; ++i) {
          len[i] = ceil_div(slices[i], split[i]);
          units[i] = tiles[i] * ceil_div(slices[i], len[i]);
          all += units[i];
          if (split[i] > 1) join += (double)split[i] * p[i].m * p[i].n * 4 / kJoinBytes;
        }
        int extra, few, many;
        const int64_t workers = all < most ? all : most;
        const bool swap = len[0] < len[1];
        const int64_t last = share_out(units[swap], len[swap], units[!swap], len[!swap], workers, &extra, &few, &many);
        const double time = c.fixed + c.slice * last + c.tile * ceil_div(all, workers) + (join > 0 ? join + kJoin : 0);
        if (!best.cg || time < best.time) best = {c.cg, c.bn, {(int)s0, (int)s1}, time};
      }
  }
  return best;
}

// The search takes 5 to 20 us of the host, a call asks two to four times: the answers for the sizes seen last are kept.
Choice choose(const CxProduct* p, int count) {
  struct Seen {
    int64_t key[7];
    Choice choice;
  };
  static thread_local Seen seen[64];
  const bool sums = p[0].mode == kOut || p[0].mode == kSums;
  const int64_t key[7] = {count * 2 + sums, p[0].m, p[0].n, p[0].k, count > 1 ? p[1].m : 0, count > 1 ? p[1].n : 0, count > 1 ? p[1].k : 0};
  uint64_t h = 0;
  for (int64_t v : key) h = (h ^ (uint64_t)v) * 0x9E3779B97F4A7C15ull;
  Seen& at = seen[h >> 58];
  if (memcmp(at.key, key, sizeof(key)) != 0) {
    at.choice = search(p, count, sums);
    memcpy(at.key, key, sizeof(key));
  }
  return at.choice;
}

int align_of(const void* p, int64_t ld) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * 2);
  return a % 32 == 0 ? 2 : a % 16 == 0 ? 1 : 0;
}

template <int CG, int BN>
int launch(const Plan& t, int count, cudaStream_t s) {
  using S = Shape<CG, BN>;
  CUtensorMap map[4] = {};
  int rc = 0;
  for (int i = 0; i < count && !rc; ++i) {
    const CxProduct& p = t.job[i].p;
    rc = p.layout == kTN ? make_map(&map[2 * i], p.a, p.dtype, p.k, p.m, p.lda, kDepth) : make_map(&map[2 * i], p.a, p.dtype, p.m, p.k, p.lda, 128);
    if (!rc)
      rc = p.layout == kNT ? make_map(&map[2 * i + 1], p.b, p.dtype, p.n, p.k, p.ldb, BN / CG)
                           : make_map(&map[2 * i + 1], p.b, p.dtype, p.k, p.n, p.ldb, kDepth);
  }
  if (rc) return rc;
  static std::atomic<uint64_t> ready{0};           // devices that know of the kernel's shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 63;
  if (dev >= 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(tensor_product_kernel<CG, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
    if (e != cudaSuccess) return cx_set_error("cx_product", (int)e);
    if (dev < 63) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  Plan plan = t;
  const int64_t units = (int64_t)t.job[0].units + t.job[1].units, most = cx_sm_count() / CG, workers = units < most ? units : most;
  share_out(t.job[0].units, t.job[0].slices_per, t.job[1].units, t.job[1].slices_per, workers, &plan.extra, &plan.few, &plan.many);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CG * workers));
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, tensor_product_kernel<CG, BN>, map[0], map[1], map[2], map[3], plan);
  cx_note_launch();
  return e == cudaSuccess ? 0 : cx_set_error("cx_product", (int)e);
}

}  // namespace

double cx_tensor_product_time(const CxProduct* p, int count) { return choose(p, count).time; }
int cx_tensor_product_stat_columns(const CxProduct& p) { return choose(&p, 1).bn / 2; }

int cx_tensor_product(CxProduct* p, int count, cxprod::Arena& ws, cudaStream_t s) {
  const Choice c = choose(p, count);
  Plan t = {};
  Spread spread = {};
  int spreads = 0;
  int64_t most = 0, units = 0, spread_rows = 0;
  for (int i = 0; i < count; ++i) units += ceil_div(p[i].m, 128 * c.cg) * ceil_div(p[i].n, c.bn) * c.splits[i];       // (at least as many)
  if (units > 0x3FFFFFFF) return cx_set_error("cx_product: too many tiles", 0);
  // the longer units first
  const bool swap = count == 2 && ceil_div(ceil_div(p[0].k, kDepth), c.splits[0]) < ceil_div(ceil_div(p[1].k, kDepth), c.splits[1]);
  for (int i = 0; i < count; ++i) {
    const int from = swap ? 1 - i : i;
    Job& job = t.job[i];
    const CxProduct& q = job.p = p[from];
    const int64_t tm = ceil_div(q.m, 128 * c.cg), tn = ceil_div(q.n, c.bn);
    job.slices = (int)ceil_div(q.k, kDepth);
    job.slices_per = (int)ceil_div(job.slices, c.splits[from]);
    job.splits = (int)ceil_div(job.slices, job.slices_per);
    job.tiles_m = (int)tm;
    job.tiles_n = (int)tn;
    job.units = (int)(tm * tn * job.splits);
    // The rows of A that a group walks with stay in L2 while B goes by once: as many as take 32 MB, or where k is long
    // about as many rows as columns at a time.  (8192 x 50257 x 1024, 8 / 16 rows of tiles: 700 / 684 us; 8192^3,
    // 4 / 8 / 16: 877 / 855 / 881 us.)
    const int64_t fit = (32ll << 20) / (q.k * 2 * 128 * c.cg);
    const int64_t group = fit < 8 ? 8 : fit < tm ? fit : tm;
    job.tiles.set((uint32_t)(tm * tn));
    job.per.set((uint32_t)(group * tn));
    job.group.set((uint32_t)group);
    job.last.set((uint32_t)(tm % group ? tm % group : group));
    if ((q.mode == kOut || q.mode == kProb) && align_of(q.out, q.ldo) == 0 && job.splits == 1) {
      const int64_t ld = (q.n + 63) / 64 * 64;
      spread.from[spreads] = reinterpret_cast<const uint16_t*>(ws.take(q.m * ld * 2));
      spread.to[spreads] = reinterpret_cast<uint16_t*>(q.out);
      spread.rows[spreads] = q.m;
      spread.cols[spreads] = q.n;
      spread.from_ld[spreads] = ld;
      spread.to_ld[spreads] = q.ldo;
      job.p.out = const_cast<uint16_t*>(spread.from[spreads++]);
      job.p.ldo = ld;
      spread_rows = spread_rows > q.m ? spread_rows : q.m;
    }
    job.wide_out = align_of(q.out, q.ldo);
    job.wide_pre = align_of(q.pre, q.ldpre);
    job.wide_res = align_of(q.residual, q.ldr);
    job.wide_bias = align_of(q.bias, 0);
    job.plain = q.mode == kOut && !q.has_addend && !q.bias && !q.pre && !q.residual && q.act == CX_ACT_NONE;
    if (job.splits > 1) {
      job.part_ld = (q.n + 7) / 8 * 8;
      job.partial = reinterpret_cast<float*>(ws.take((int64_t)job.splits * q.m * job.part_ld * 4));
      const int64_t blocks = ceil_div(q.m * (job.part_ld / 8), kJoinThreads);
      if (blocks > most) most = blocks;
    }
  }
  if (!ws.base) return 0;
  if (!ws.ok()) return cx_set_error("cx_product: workspace too small", 0);
  const Word said = status_word();
  if (!said.host) return cx_set_error("cx_product: no pinned memory for the status word", 0);
  if (*reinterpret_cast<volatile uint32_t*>(said.host)) {
    *reinterpret_cast<volatile uint32_t*>(said.host) = 0;
    return cx_set_error("cx_product: an earlier product of this device gave up waiting, its results are not valid", 0);
  }
  t.status = said.device;
  const int rc = c.cg == 2 ? launch<2, 256>(t, count, s) : c.bn == 128 ? launch<1, 128>(t, count, s) : launch<1, 64>(t, count, s);
  if (rc) return rc;
  if (most) {
    const dim3 grid((unsigned)most, (unsigned)count);
    if (p[0].dtype == CX_BF16) cx_launch_pdl2(join_splits_kernel<__nv_bfloat16>, grid, kJoinThreads, s, t);
    else cx_launch_pdl2(join_splits_kernel<__half>, grid, kJoinThreads, s, t);
    cx_note_launch();
  }
  if (spreads) {
    const int64_t blocks = (int64_t)cx_sm_count() * 8;
    cx_launch_pdl2(spread_kernel, dim3((unsigned)(spread_rows < blocks ? spread_rows : blocks), (unsigned)spreads), kJoinThreads, s, spread);
    cx_note_launch();
  }
  return cx_check_launch("cx_product");
}
