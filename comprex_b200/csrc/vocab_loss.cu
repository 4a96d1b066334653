// Softmax cross entropy of s = h w^T over a vocabulary, and its gradients, without the logits in memory.
//
//   loss_r = log sum_v exp(s_rv) - s_r,t(r)      P_rv = (exp(s_rv - lse_r) - [v = t(r)]) g_r      dh = P w      dw = P^T h
//
// Forward: the product's epilogue leaves per row and tile of columns the largest logit and the sum of exponentials under
// it, and the target's logit; a second kernel joins a row's tiles and a third one sums the losses.  Backward goes over
// the vocabulary in pieces: the piece's logits are computed once more, P of the piece goes to a workspace in 16 bits,
// and two products, in one launch, take it from there.  dh grows over the pieces in 32 bits, in a fixed order.
//
// Bound by the tensor cores and, for long, by the power limit: 8 N V D operations where a call that kept the logits would
// do 6 N V D.  8192 rows, V = 50257, D = 1024 in bf16: forward 0.52 ms from a cold start (1.6 PFLOP/s) and 0.65 at the power
// limit, forward and backward 2.7 ms (1.23 PFLOP/s with the logits counted twice).
//
// P in 16 bits: a probability of a large vocabulary times the 1 / rows of a mean is below what fp16 can hold, so P is
// stored relative to the largest finite |g_r|, times 2^14, and both products take that out at the end, in 32 bits.  So a gradient that
// all rows share is not rounded: times a power of two alone, its own rounding was a common error of all probabilities (bf16, 255
// rows: 2^-8 of dh and dw).  One factor for all rows, since dw adds rows up.  What it costs in fp16 where rows are weighted far apart:
// dh of a row at 2^-16 / 2^-20 / 2^-24 / 2^-28 of the largest g is 2.1e-4 / 3.9e-4 / 3e-3 / 3e-2 of itself off (2.0e-4 at the largest: its own
// rounding; 50257 words).  Such rows count for less in dw than its rounding, and 2^-30 is the whole range of fp16.
#include "cx_product.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int64_t kPieceBytes = 208ll << 20;

struct Join {
  const float2* part;
  const float* target_logit;
  const int64_t* targets;
  int64_t rows, tiles, vocab, ignore;
  float* lse;
  float* row_loss;
};

// Joins the tiles of 32 rows: 8 threads of a row take every eighth tile, then join among themselves, in a fixed order.
// (One thread a row, tile after tile, took 42 us for 8192 rows of 197 tiles: each step waits for the one before.)
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ Join j) {
  __shared__ float2 part[8][32];
  cx::pdl_trigger();
  cx::pdl_wait();
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  const int64_t r = (int64_t)blockIdx.x * 32 + lane;
  // a tile without a finite logit has top -inf, and its sum is 0, or NaN where a logit was no number
  float top = -INFINITY, sum = 0.f;
  if (r < j.rows) {
    for (int64_t i0 = group; i0 < j.tiles; i0 += 32) {
      float2 s[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = i0 + 8 * k < j.tiles ? j.part[(i0 + 8 * k) * j.rows + r] : make_float2(-INFINITY, 0.f);
      const float m = fmaxf(fmaxf(top, fmaxf(s[0].x, s[1].x)), fmaxf(s[2].x, s[3].x)), base = m == -INFINITY ? 0.f : m;
      sum *= exp2f((top - base) * cxprod::kLog2e);
#pragma unroll
      for (int k = 0; k < 4; ++k) sum += s[k].y * exp2f((s[k].x - base) * cxprod::kLog2e);
      top = m;
    }
  }
  part[group][lane] = make_float2(top, sum);
  __syncthreads();
  if (group || r >= j.rows) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) top = fmaxf(top, part[k][lane].x);
  const float base = top == -INFINITY ? 0.f : top;
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += part[k][lane].y * exp2f((part[k][lane].x - base) * cxprod::kLog2e);
  const int64_t t = j.targets[r];
  const bool ignored = t == j.ignore, inside = t >= 0 && t < j.vocab;
  float lse = top + logf(sum);
  if (!ignored && !inside) lse = NAN;
  j.lse[r] = lse;
  j.row_loss[r] = ignored ? 0.f : inside ? lse - j.target_logit[r] : NAN;
}

struct Total {
  const float* row_loss;
  const int64_t* targets;
  int64_t rows, ignore;
  int reduction;
  float* loss;
  float* count;
};

// one block: the sum of the rows' losses and the number of rows that count, in a fixed order
__global__ void __launch_bounds__(1024) total_kernel(const __grid_constant__ Total d) {
  __shared__ float s_sum[32], s_cnt[32];
  cx::pdl_trigger();
  cx::pdl_wait();
  float sum = 0.f, cnt = 0.f;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < d.rows; r += 1024) {
    sum += d.row_loss[r];
    cnt += d.targets[r] == d.ignore ? 0.f : 1.f;
  }
  for (int k = 16; k; k >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, k);
    cnt += __shfl_xor_sync(0xFFFFFFFFu, cnt, k);
  }
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_cnt[threadIdx.x >> 5] = cnt;
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  sum = s_sum[threadIdx.x];
  cnt = s_cnt[threadIdx.x];
  for (int k = 16; k; k >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, k);
    cnt += __shfl_xor_sync(0xFFFFFFFFu, cnt, k);
  }
  if (threadIdx.x == 0) {
    *d.count = cnt;
    *d.loss = d.reduction == CX_REDUCE_MEAN ? sum / cnt : sum;
  }
}

struct Factors {
  const float* grad;
  const int64_t* targets;
  const float* lse;
  const float* count;
  int64_t rows, grad_stride, ignore;
  int reduction;
  float* lse2;          // [rows] lse in units of log 2
  float* factor;        // [rows] 2^14 g_r / base
  float* scale;         // base / 2^14
};

__device__ __forceinline__ float row_grad(const Factors& f, int64_t r) {
  if (f.targets[r] == f.ignore) return 0.f;
  return f.grad[f.reduction == CX_REDUCE_NONE ? r * f.grad_stride : 0];
}

// Every block looks at all rows for the largest |g_r| (at most 16 blocks) where each row has one of its own, and then
// makes the factors of its share.
__global__ void __launch_bounds__(1024) factor_kernel(const __grid_constant__ Factors f) {
  __shared__ uint32_t s_top;
  cx::pdl_trigger();
  cx::pdl_wait();
  const float per = f.reduction == CX_REDUCE_MEAN ? *f.count : 1.f;
  uint32_t top = 0;
  if (f.reduction == CX_REDUCE_NONE) {
    if (threadIdx.x == 0) s_top = 0;
    __syncthreads();
#pragma unroll 4
    for (int64_t r = threadIdx.x; r < f.rows; r += 1024) {
      const uint32_t bits = __float_as_uint(row_grad(f, r)) & 0x7FFFFFFFu;
      top = max(top, bits < 0x7F800000u ? bits : 0u);      // a gradient that is infinite or no number is its row's own matter
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((threadIdx.x & 31) == 0) atomicMax(&s_top, top);
    __syncthreads();
    top = s_top;
  } else {
    top = __float_as_uint(*f.grad / per) & 0x7FFFFFFFu;
  }
  // the largest itself, or a power of two where it is so far out that a quotient or product would leave the normal numbers
  const int e = (int)(top >> 23) - 127;
  const float base = e < -100 ? 0x1p-100f : e > 120 ? 0x1p120f : __uint_as_float(top);
  if (blockIdx.x == 0 && threadIdx.x == 0) *f.scale = base * 0x1p-14f;
  for (int64_t r = blockIdx.x * 1024ll + threadIdx.x; r < f.rows; r += gridDim.x * 1024ll) {
    const float g = row_grad(f, r);
    f.factor[r] = g == 0.f ? 0.f : g / per / base * 0x1p14f;
    f.lse2[r] = f.lse[r] * cxprod::kLog2e;
  }
}

// Both calls also run without a workspace: they launch nothing then and count the bytes that they need.
int forward(const CxVocabLoss& l, cxprod::Arena& ws, cudaStream_t s) {
  CxProduct p = {};
  p.m = l.rows; p.n = l.vocab; p.k = l.dim;
  p.a = l.h; p.lda = l.ldh; p.b = l.w; p.ldb = l.ldw;
  p.layout = kNT; p.mode = kStats; p.dtype = l.dtype; p.targets = l.targets;
  int rc = cx_product_operand(&p.a, &p.lda, l.dtype, l.rows, l.dim, ws, s);
  if (!rc) rc = cx_product_operand(&p.b, &p.ldb, l.dtype, l.vocab, l.dim, ws, s);
  if (rc) return rc;
  const int64_t bn = cx_product_stat_columns(p), tiles = (l.vocab + bn - 1) / bn;
  p.part = reinterpret_cast<float2*>(ws.take(tiles * l.rows * 8));
  p.target_logit = reinterpret_cast<float*>(ws.take(l.rows * 4));
  float* row_loss = l.reduction == CX_REDUCE_NONE ? l.loss : reinterpret_cast<float*>(ws.take(l.rows * 4));
  rc = cx_product(&p, 1, ws, s);
  if (rc || !ws.base) return rc;
  const Join j = {p.part, p.target_logit, l.targets, l.rows, tiles, l.vocab, l.ignore_index, l.lse, row_loss};
  cx_launch_pdl2(join_kernel, dim3((unsigned)((l.rows + 31) / 32)), kThreads, s, j);
  cx_note_launch();
  if (l.reduction != CX_REDUCE_NONE) {
    const Total d = {row_loss, l.targets, l.rows, l.ignore_index, l.reduction, l.loss, l.count};
    cx_launch_pdl2(total_kernel, dim3(1), 1024, s, d);
    cx_note_launch();
  }
  return cx_check_launch("cx_vocab_loss_forward");
}

// The products of a piece of the vocabulary, [v0, v0 + n): its probabilities, and what they give to the gradients.
struct Piece {
  CxProduct prob, both[2];
  int count;
  Piece(const CxVocabLoss& l, const void* h, int64_t ldh, const void* w, int64_t ldw, int64_t v0, int64_t n, void* p, int64_t ldp) : prob(), both(), count(0) {
    const int64_t size = l.dtype == CX_F32 ? 4 : 2;
    const void* at = reinterpret_cast<const char*>(w) + v0 * ldw * size;
    prob.m = l.rows; prob.n = n; prob.k = l.dim;
    prob.a = h; prob.lda = ldh; prob.b = at; prob.ldb = ldw;
    prob.layout = kNT; prob.mode = kProb; prob.dtype = l.dtype;
    prob.out = p; prob.ldo = ldp; prob.targets = l.targets; prob.col0 = v0;
    if (l.dh) {
      CxProduct& q = both[count++];
      q.m = l.rows; q.n = l.dim; q.k = n;
      q.a = p; q.lda = ldp; q.b = at; q.ldb = ldw;
      q.layout = kNN; q.dtype = l.dtype; q.has_addend = v0 > 0;
      q.mode = v0 + n < l.vocab ? kSums : kOut;
      q.out = l.dh; q.ldo = l.dim;
    }
    if (l.dw) {
      CxProduct& q = both[count++];
      q.m = n; q.n = l.dim; q.k = l.rows;
      q.a = p; q.lda = ldp; q.b = h; q.ldb = ldh;
      q.layout = kTN; q.dtype = l.dtype;
      q.out = reinterpret_cast<char*>(l.dw) + v0 * l.dim * size; q.ldo = l.dim;
    }
  }
};

// Columns of a piece.  One that stays in L2 between its making and its two readers saves power, which is what bounds these
// products for long; but its tiles must fill the GPU, and few of them leave a tenth of it idle.  So: of the sizes up to
// kPieceBytes the one that the model of the products says is fastest.  Backward call of 8192 rows, width 1024, vocabulary
// 50257 at the power limit, pieces of up to 72 / 144 / 208 / 288 / 424 MB and the whole: 2188 / 2160 / 2115 / 2200 / 2163 /
// 2255 us (at 1402 / 1250 / 1200 / 1085 / 1085 / 1060 MHz).
int64_t search_columns(const CxVocabLoss& l) {
  const int64_t size = l.dtype == CX_F32 ? 4 : 2, whole = (l.vocab + 7) / 8 * 8;
  int64_t most = kPieceBytes / (l.rows * size) / 256 * 256;
  if (most < 256) most = 256;
  if (whole <= most && l.rows * whole * size <= kPieceBytes / 4) return whole;
  if (l.dtype == CX_F32) return whole < most ? whole : most;
  int64_t best = whole < most ? whole : most;
  double least = 1e30;
  for (int64_t n = most; n >= 256 && n > most / 4; n -= 256) {
    const int64_t columns = n < whole ? n : whole, full = l.vocab / columns, rest = l.vocab % columns;
    const Piece a(l, nullptr, 8, nullptr, 8, 0, columns, nullptr, 8);
    double time = full * (cx_tensor_product_time(&a.prob, 1) + cx_tensor_product_time(a.both, a.count));
    if (rest) {
      const Piece b(l, nullptr, 8, nullptr, 8, 0, rest, nullptr, 8);
      time += cx_tensor_product_time(&b.prob, 1) + cx_tensor_product_time(b.both, b.count);
    }
    if (time < least) {
      least = time;
      best = columns;
    }
  }
  return best;
}
int64_t piece_columns(const CxVocabLoss& l) {
  static thread_local int64_t seen[6] = {};            // the sizes asked for last, and the answer
  const int64_t key[5] = {l.rows, l.vocab, l.dim, l.dtype, (l.dh ? 1 : 0) | (l.dw ? 2 : 0)};
  if (memcmp(seen, key, sizeof(key)) != 0) {
    seen[5] = search_columns(l);
    memcpy(seen, key, sizeof(key));
  }
  return seen[5];
}

int backward(const CxVocabLoss& l, cxprod::Arena& ws, cudaStream_t s) {
  const int64_t size = l.dtype == CX_F32 ? 4 : 2;
  const void *h = l.h, *w = l.w;
  int64_t ldh = l.ldh, ldw = l.ldw;
  int rc = cx_product_operand(&h, &ldh, l.dtype, l.rows, l.dim, ws, s);
  if (!rc) rc = cx_product_operand(&w, &ldw, l.dtype, l.vocab, l.dim, ws, s);
  if (rc) return rc;
  const int64_t piece = piece_columns(l);
  const int64_t ldp = (piece + 63) / 64 * 64;          // whole lines
  void* prob = ws.take(l.rows * ldp * size);
  const int64_t sums_ld = (l.dim + 7) / 8 * 8;
  float* sums = l.dh && piece < l.vocab ? reinterpret_cast<float*>(ws.take(l.rows * sums_ld * 4)) : nullptr;
  Factors f = {l.grad, l.targets, l.lse, l.count, l.rows, l.grad_stride, l.ignore_index, l.reduction, nullptr, nullptr, nullptr};
  f.lse2 = reinterpret_cast<float*>(ws.take(l.rows * 4));
  f.factor = reinterpret_cast<float*>(ws.take(l.rows * 4));
  f.scale = reinterpret_cast<float*>(ws.take(4));
  if (ws.base) {
    if (!ws.ok()) return cx_set_error("cx_vocab_loss_backward: workspace too small", 0);
    const int64_t blocks = (l.rows + 1023) / 1024;
    cx_launch_pdl2(factor_kernel, dim3((unsigned)(blocks < 16 ? blocks : 16)), 1024, s, f);
    cx_note_launch();
    rc = cx_check_launch("cx_vocab_loss_backward");
  }
  const int64_t begin = ws.used;               // what the products need is used again by the next piece
  int64_t most = begin;
  for (int64_t v0 = 0; v0 < l.vocab && !rc; v0 += piece) {
    ws.used = begin;
    Piece p(l, h, ldh, w, ldw, v0, piece < l.vocab - v0 ? piece : l.vocab - v0, prob, ldp);
    p.prob.lse = f.lse2;
    p.prob.row_factor = f.factor;
    for (int i = 0; i < p.count; ++i) {
      p.both[i].scale = f.scale;
      if (p.both[i].layout == kNN) {
        p.both[i].addend = sums;
        p.both[i].ldadd = sums_ld;
      }
    }
    rc = cx_product(&p.prob, 1, ws, s);
    if (!rc) rc = cx_product(p.both, p.count, ws, s);
    if (ws.used > most) most = ws.used;
  }
  ws.used = most;
  return rc;
}

}  // namespace

int64_t cx_vocab_loss_workspace_bytes_cuda(const CxVocabLoss* l, int back) {
  cxprod::Arena ws = {nullptr, 0, 0};
  (back ? backward : forward)(*l, ws, nullptr);
  return ws.used + 256;          // never none: without a base nothing runs
}
int cx_vocab_loss_forward_cuda(const CxVocabLoss* l, void* stream) {
  cxprod::Arena ws = {reinterpret_cast<char*>(l->workspace), 0, l->ws_bytes};
  return ws.base ? forward(*l, ws, static_cast<cudaStream_t>(stream)) : cx_set_error("cx_vocab_loss_forward: no workspace", 0);
}
int cx_vocab_loss_backward_cuda(const CxVocabLoss* l, void* stream) {
  cxprod::Arena ws = {reinterpret_cast<char*>(l->workspace), 0, l->ws_bytes};
  return ws.base ? backward(*l, ws, static_cast<cudaStream_t>(stream)) : cx_set_error("cx_vocab_loss_backward: no workspace", 0);
}
