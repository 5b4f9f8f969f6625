// Dense layer with its epilogue: y = act(x w^T + bias + residual), and its backward pass (1x1 convolutions and
// feed-forward layers of the cross-view attention block: det3d/models/necks/attention.py:36-41, :77-84, :127-146).
// The activation comes after the residual, as in the epilogue of the sparse convolutions.
//
// fp32 operands run as three exact bf16 planes (six of the nine products, fp32 accumulation), bf16 ones directly; both in the tiles of
// vx_tile.h. A reduction split over workgroups leaves fp32 slabs that one kernel adds in a fixed order: no atomics, bitwise
// reproducible.
#include <type_traits>

#include "vx_tile.h"

namespace {

constexpr int kActNone = VX_ACT_NONE, kActRelu = VX_ACT_RELU, kActGelu = VX_ACT_GELU, kActSilu = VX_ACT_SILU;

__device__ __forceinline__ float act_value(float a, int act) {
  if (act == kActRelu) return a < 0.0f ? 0.0f : a;      // NaN stays NaN
  if (act == kActGelu) return 0.5f * a * (1.0f + erff(a * 0.70710678118654752f));
  if (act == kActSilu) return a / (1.0f + expf(-a));
  return a;
}
// slope at the saved value: relu's output, the others' pre-activation
__device__ __forceinline__ float act_slope(float a, int act) {
  if (act == kActRelu) return a > 0.0f ? 1.0f : 0.0f;
  if (act == kActGelu)
    return 0.5f * (1.0f + erff(a * 0.70710678118654752f)) + a * 0.39894228040143268f * expf(-0.5f * a * a);
  if (act == kActSilu) {
    const float e = 1.0f / (1.0f + expf(-a));
    return e * (1.0f + a * (1.0f - e));
  }
  return 1.0f;
}

template <typename T>
struct FwdArgs {
  const T *x, *w, *bias, *res;
  T *y, *pre;
  long long ldx, ldw, ldr, m;
  int n, k, act, tiles_n;
};

// y[m][n .. n + 3] from the product v: `left` of the four exist
template <typename T>
__device__ __forceinline__ void linear_finish(const FwdArgs<T>& a, long long m, int n, int left, vx_f32x4 v) {
  if (a.bias) v += vx_load4(a.bias + n, left);
  if (a.res) v += vx_load4(a.res + m * a.ldr + n, left);
  const long long at = m * a.n + n;
  if (a.pre) vx_store4(a.pre + at, v, left);
  if (a.act != kActNone) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = act_value(v[i], a.act);
  }
  vx_store4(a.y + at, v, left);
}

// A workgroup owns TM x TN outputs. fp32 6400 x 384 -> 384 18 us (600 workgroups, 2.3 rounds on 256 CUs, 105 TFLOP/s; counters: matrix
// pipe and LDS 4.5 us each, vector pipe 6, the waves wait for loads and at the barriers of twelve steps), 204800 x 384 -> 512 495 us
// (163); bf16 141 us (571 TFLOP/s, 2.6 TB/s; matrix pipe, vector pipe and LDS 32 us each, one after the other in six steps of
// 64: staging through registers between the products).
template <typename T, int TM, int TN, bool FAST>
__global__ __launch_bounds__(kTileThreads, 2) void linear_fwd(const FwdArgs<T> a) {
  constexpr int BK = TM <= 64 ? 64 : VxType<T>::BK;        // 64 against 32 of fp32: 6400 x 384 -> 384 21 against 24 us
  // y of the small tiles goes past the caches: it would push out the rows of x that the next column tiles read. Measured with the layer
  // that reads y behind it (384 -> 512 -> 384, bf16; us of the pair, past / through): 64 x 64 tiles, 6400 rows 17.8 / 18.1, 16896 35.0 /
  // 38.1 (128 -> 512 of 60000 rows alone 24 / 35); 128 x 128 tiles, 60000 rows 93.8 / 85.4, 204800 305 / 308 (alone 121 / 142: what the layer gains the next one loses). fp32:
  // within 2 % either way, 6400 to 204800 rows
  constexpr bool ONCE = TM <= 64;
  __shared__ __attribute__((aligned(16))) char lds[vx_gemm_lds<T, TM, TN, BK>()];
  const unsigned t = vx_xcd_tile(blockIdx.x, gridDim.x);
  const long long m0 = (long long)(t / a.tiles_n) * TM;
  const int n0 = (int)(t % a.tiles_n) * TN;
  const int rows_m = (int)(a.m - m0 < TM ? a.m - m0 : TM), rows_n = a.n - n0 < TN ? a.n - n0 : TN;
  vx_f32x4 acc[TM / 32][TN / 32];
  vx_acc_zero(acc);
  vx_f32x4 bias[TN / 64][2];                   // of this lane's columns, there when the product is
  if (a.bias) {
    vx_acc_each<TM, TN>(acc, [&](int mi, int, int j, int n, const vx_f32x4&, const vx_f32x4&) {
      if (mi) return;
      bias[j][0] = vx_load4(a.bias + n0 + n, rows_n - n);
      bias[j][1] = vx_load4(a.bias + n0 + n + 4, rows_n - n - 4);
    });
  }
  const VxOperand<T> X{a.x + m0 * a.ldx, a.ldx, rows_m}, W{a.w + (long long)n0 * a.ldw, a.ldw, rows_n};
  vx_gemm_loop<T, KC, KC, TM, TN, FAST, BK>(X, W, 0, a.k, lds, acc);
  const long long at0 = m0 * a.n + n0;
  vx_acc_each<TM, TN>(acc, [&](int, int m, int j, int n, vx_f32x4 v, vx_f32x4 w) {
    const int left = rows_n - n;
    if (m >= rows_m || left <= 0) return;
    if (a.bias) {
      v += bias[j][0];
      w += bias[j][1];
    }
    if (a.res) {
      const T* r = a.res + (m0 + m) * a.ldr + n0 + n;
      v += vx_load4(r, left);
      w += vx_load4(r + 4, left - 4);
    }
    const long long at = at0 + (long long)m * a.n + n;
    if (a.pre) vx_store8<ONCE>(a.pre + at, v, w, left);
    if (a.act == kActRelu) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = act_value(v[i], kActRelu);
        w[i] = act_value(w[i], kActRelu);
      }
    } else if (a.act != kActNone) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = act_value(v[i], a.act);
        w[i] = act_value(w[i], a.act);
      }
    }
    vx_store8<ONCE>(a.y + at, v, w, left);
  });
}

// Few rows: what counts is latency. A workgroup owns 16 x 16 outputs, its four waves every fourth 32-k step each, with operands
// straight from memory in fragment order and four steps of loads in flight; the four partial sums meet in LDS, added in order.
// 7 x 384 -> 512 fp32: 4.1 us, of which the launch is most.
template <typename T, bool FAST>
__global__ __launch_bounds__(kTileThreads) void linear_few(const FwdArgs<T> a) {
  constexpr int NPL = VxType<T>::NPL, U = 4, E = sizeof(T);
  __shared__ vx_f32x4 sh[kTileThreads / 64][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const long long m0 = (long long)(blockIdx.x / a.tiles_n) * 16;
  const int n0 = (int)(blockIdx.x % a.tiles_n) * 16;
  const bool row_m = m0 + c < a.m, row_n = n0 + c < a.n;
  const T *px = a.x + m0 * a.ldx, *pw = a.w + (long long)n0 * a.ldw;
  vx_f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k0 = wave * 32; k0 < a.k; k0 += U * 128) {
    VxRow8<T> x[U], w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 128, left = a.k - k - g * 8;
      if constexpr (FAST) {
        x[u].load(vx_buffer(px + k), row_m && left > 0 ? (c * (int)a.ldx + g * 8) * E : kVxOut);
        w[u].load(vx_buffer(pw + k), row_n && left > 0 ? (c * (int)a.ldw + g * 8) * E : kVxOut);
      } else {
        x[u].load(px + c * a.ldx + k + g * 8, row_m ? left : 0);
        w[u].load(pw + c * a.ldw + k + g * 8, row_n ? left : 0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      VxFrag<NPL> fx, fw;
      x[u].planes(fx);
      w[u].planes(fw);
#pragma unroll
      for (int pr = 0; pr < VxProducts<NPL, NPL>::N; ++pr) acc = vx_mma(pr, fw, fx, acc);
    }
  }
  sh[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int i = 1; i < kTileThreads / 64; ++i) acc += sh[i][lane];
  const int n = n0 + g * 4;
  if (row_m && n < a.n) linear_finish(a, m0 + c, n, a.n - n, acc);
}

// ---- backward -------------------------------------------------------------------------------------------------------
// g = dy * act'(saved) (written where there is an activation) and the column sums of g per row chunk. wide: g unrounded for the two
// products, where its rounding to bf16 is one (gelu, silu: it would make the error of dx and dw 1.4 times that of their own rounding;
// relu's g is dy or 0). A lane owns 16 bytes of columns, `lanes` (a power of two, at most a wave) lanes a row, so that a wave reads whole rows; a workgroup owns `lanes` x 16 bytes
// of columns and a chunk of rows. Sums in fp32 per thread, then over the workgroup's rows in order. One pass: 102399 x 512 bf16, two
// reads and a write, 64 us (4.9 TB/s of the 5.1 that a copy reaches); gelu, with g in fp32 as well, 112 us (4.7).
template <typename T>
struct ActArgs {
  const T *dy, *saved;
  T* g;
  float *wide, *part;                          // wide: [m][n] or null
  long long ldy, m, chunk;
  int n, act, lanes, cols;                     // cols: workgroups along the columns
};
template <typename T>
__device__ __forceinline__ void act_rows(const ActArgs<T>& a, unsigned block, char* lds) {
  constexpr int V = 16 / sizeof(T), Q = V / 4, U = 2;              // columns and quads of a lane, rows in flight
  vx_f32x4(*sh)[Q] = reinterpret_cast<vx_f32x4(*)[Q]>(lds);
  const T *__restrict__ dy = a.dy, *__restrict__ saved = a.saved;
  T* __restrict__ g = a.g;
  float* __restrict__ part = a.part;
  const long long ldy = a.ldy, m = a.m, chunk = a.chunk;
  const int n = a.n, act = a.act, lanes = a.lanes;
  const unsigned bx = block % a.cols, by = block / a.cols;
  const int cl = threadIdx.x & (lanes - 1), rl = threadIdx.x / lanes, rows = 256 / lanes;
  const int c = (bx * lanes + cl) * V;
  const long long r0 = (long long)by * chunk, r1 = r0 + chunk < m ? r0 + chunk : m;
  vx_f32x4 sum[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) sum[q] = vx_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (c < n) {
    for (long long r = r0 + rl; r < r1; r += U * rows) {
      vx_f32x4 v[U][Q], s[U][Q];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long row = r + u * rows < r1 ? r + u * rows : r;
        vx_loadq(dy + row * ldy + c, n - c, v[u]);
        if (act != kActNone) vx_loadq(saved + row * n + c, n - c, s[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long row = r + u * rows;
        if (row >= r1) break;
        if (act != kActNone) {
#pragma unroll
          for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[u][q][i] = act == kActRelu ? (s[u][q][i] > 0.0f ? v[u][q][i] : 0.0f) : v[u][q][i] * act_slope(s[u][q][i], act);
          if constexpr (Q == 2)
            vx_store8(g + row * n + c, v[u][0], v[u][1], n - c);
          else
            vx_store4(g + row * n + c, v[u][0], n - c);
          if constexpr (Q == 2)
            if (a.wide) vx_store8(a.wide + row * n + c, v[u][0], v[u][1], n - c);
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) sum[q] += v[u][q];
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int q = 0; q < Q; ++q) sh[threadIdx.x][q] = sum[q];
  __syncthreads();
  if (rl == 0 && c < n) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      for (int i = 1; i < rows; ++i) sum[q] += sh[i * lanes + cl][q];
      vx_store4(part + (long long)by * n + c + q * 4, sum[q], n - c - q * 4);
    }
  }
}
template <typename T>
__global__ __launch_bounds__(256) void act_bwd(const ActArgs<T> a) {
  __shared__ __attribute__((aligned(16))) char lds[256 * 16 / sizeof(T) * 4];
  act_rows(a, blockIdx.x, lds);
}

template <typename T, typename G>
struct BwdArgs {
  const G* g;
  const T *x, *w;
  T *dx, *dw;
  float* slab;          // [splits][n][k] when splits > 1
  long long ldg, ldx, ldw, m, span;   // span: rows of one split
  int n, k, tiles_w, tiles_wk, tiles_xk;   // dw: tiles_w = all tiles of one split, tiles_wk along k; dx: tiles along k
  unsigned blocks_w, blocks_x;
};

// one launch for the gradients: workgroups [0, blocks_w) are tiles of dw = g^T x (reduction over the rows, split), the next blocks_x
// tiles of dx = g w (reduction over n), the others (no activation: g = dy) the column sums. 6400 x 512 -> 384 fp32 39 us (129 TFLOP/s),
// 102399 x 384 -> 512 bf16 129 us (624; LDS 44 us of it, a quarter of that bank conflicts, matrix pipe 32): dw's operands are transposed on
// their way to LDS.
// G: the type of g, fp32 beside bf16 operands where act_bwd wrote it so (two planes): 207 us
template <typename T, typename G, int TM, int TN, bool FAST>
__global__ __launch_bounds__(kTileThreads, 2) void linear_bwd(const BwdArgs<T, G> a, const ActArgs<T> sums) {
  constexpr int BK = VxType<T>::BK, PG = sizeof(G) == sizeof(T) ? VxType<T>::NPL : VxType<T>::NPL_F32;
  __shared__ __attribute__((aligned(16))) char lds[vx_gemm_lds<T, TM, TN, BK, PG>()];
  if (blockIdx.x >= a.blocks_w + a.blocks_x) {
    act_rows(sums, blockIdx.x - a.blocks_w - a.blocks_x, lds);
    return;
  }
  vx_f32x4 acc[TM / 32][TN / 32];
  vx_acc_zero(acc);
  if (blockIdx.x < a.blocks_w) {
    const unsigned t = vx_xcd_tile(blockIdx.x, a.blocks_w);
    const int split = (int)(t / a.tiles_w), tile = (int)(t % a.tiles_w);
    const int n0 = tile / a.tiles_wk * TM, k0 = tile % a.tiles_wk * TN;
    const long long r0 = split * a.span;
    const int rows = (int)(a.m - r0 < a.span ? a.m - r0 : a.span);
    const int rows_n = a.n - n0 < TM ? a.n - n0 : TM, rows_k = a.k - k0 < TN ? a.k - k0 : TN;
    const VxOperand<G> X{a.g + r0 * a.ldg + n0, a.ldg, rows_n};
    const VxOperand<T> W{a.x + r0 * a.ldx + k0, a.ldx, rows_k};
    vx_gemm_loop<T, KS, KS, TM, TN, FAST, BK, G, PG>(X, W, 0, rows, lds, acc);
    float* slab = a.slab ? a.slab + (long long)split * a.n * a.k : nullptr;
    vx_acc_each<TM, TN>(acc, [&](int, int m, int, int n, const vx_f32x4& v, const vx_f32x4& w) {
      const int left = rows_k - n;
      if (m >= rows_n || left <= 0) return;
      const long long at = (long long)(n0 + m) * a.k + k0 + n;
      if (slab) vx_store8(slab + at, v, w, left); else vx_store8(a.dw + at, v, w, left);
    });
  } else {
    const unsigned t = vx_xcd_tile(blockIdx.x - a.blocks_w, a.blocks_x);
    const long long m0 = (long long)(t / a.tiles_xk) * TM;
    const int k0 = (int)(t % a.tiles_xk) * TN;
    const int rows_m = (int)(a.m - m0 < TM ? a.m - m0 : TM), rows_k = a.k - k0 < TN ? a.k - k0 : TN;
    const VxOperand<G> X{a.g + m0 * a.ldg, a.ldg, rows_m};
    const VxOperand<T> W{a.w + k0, a.ldw, rows_k};
    vx_gemm_loop<T, KC, KS, TM, TN, FAST, BK, G, PG>(X, W, 0, a.n, lds, acc);
    const long long at0 = m0 * a.k + k0;
    vx_acc_each<TM, TN>(acc, [&](int, int m, int, int n, const vx_f32x4& v, const vx_f32x4& w) {
      if (m < rows_m && n < rows_k) vx_store8(a.dx + at0 + (long long)m * a.k + n, v, w, rows_k - n);
    });
  }
}

// out[i] = sum over the slabs of slab[s * len + i], in a fixed order. Two such sums in one launch: dw (few long slabs: a thread has
// four values, eight slabs in flight) and dbias (many short ones: lane group j of a workgroup, 16 of 16 lanes, adds the slabs
// j, j + 16, ..., then the 16 groups are added in order). 384 x 512 of 25 splits 5.8 us.
template <typename T>
__global__ __launch_bounds__(256) void slab_sum(const float* __restrict__ a, int count_a, long long len_a, T* __restrict__ out_a,
                                                const float* __restrict__ b, int count_b, long long len_b,
                                                T* __restrict__ out_b, unsigned blocks_a) {
  __shared__ vx_f32x4 sh[16][17];
  constexpr int U = 8;
  vx_f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  if (blockIdx.x < blocks_a) {
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= len_a) return;
    const int left = len_a - i < 4 ? (int)(len_a - i) : 4, last = count_a - 1;
    for (int c = 0; c < count_a; c += U) {
      vx_f32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = vx_load4(a + (c + u < last ? c + u : last) * len_a + i, left);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u > last) break;
        s += v[u];
      }
    }
    vx_store4(out_a + i, s, left);
    return;
  }
  const int cl = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const long long i = ((long long)(blockIdx.x - blocks_a) * 16 + cl) * 4;
  const int left = len_b - i < 4 ? (int)(len_b - i) : 4;
  if (left > 0) {
    for (int c = grp; c < count_b; c += 16 * U) {
      vx_f32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = vx_load4(b + (c + u * 16 < count_b ? c + u * 16 : c) * len_b + i, left);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u * 16 >= count_b) break;
        s += v[u];
      }
    }
  }
  sh[grp][cl] = s;
  __syncthreads();
  if (grp || left <= 0) return;
#pragma unroll
  for (int j = 1; j < 16; ++j) s += sh[j][cl];
  vx_store4(out_b + i, s, left);
}

struct BwdPlan {
  bool big;
  int64_t splits, span, chunks, chunk, lanes;      // lanes: of act_bwd, a row
};
BwdPlan bwd_plan(int64_t m, int64_t n, int64_t k, int32_t dtype) {
  BwdPlan p;
  const int64_t cus = vx_tile_cus(), bk = dtype == VX_F32 ? 32 : 64;
  // 128 x 128 tiles from here on; us of 64 / 128: fp32 6400 x 384 -> 384 (150 tiles of dx) 41 / 45, x 512 -> 384 (200) 50 / 47, 25600 x 384
  // -> 512 151 / 143; bf16 6400 x 512 -> 384 27 / 27, 12800 x 384 -> 512 39 / 37, 102400 192 / 147
  p.big = 4 * vx_cdiv(m, 128) * vx_cdiv(k, 128) >= 3 * cus;
  const int64_t t = p.big ? 128 : 64, tiles = vx_cdiv(n, t) * vx_cdiv(k, t);
  int64_t splits = vx_cdiv(2 * cus, tiles);
  const int64_t most = vx_cdiv(m, 8 * bk);
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  p.span = vx_cdiv(vx_cdiv(m, splits), bk) * bk;
  p.splits = vx_cdiv(m, p.span);
  const int64_t v = dtype == VX_F32 ? 4 : 8;
  p.lanes = 1;
  while (p.lanes < 64 && p.lanes * v < n) p.lanes *= 2;
  const int64_t rows = 256 / p.lanes;
  p.chunk = vx_cdiv(vx_cdiv(m, vx_cdiv(4 * cus, vx_cdiv(n, p.lanes * v))), rows) * rows;
  if (p.chunk < 8 * rows) p.chunk = 8 * rows;
  p.chunks = vx_cdiv(m, p.chunk);
  return p;
}

// linear_few instead of 64 x 64 tiles: time of a call in a graph, us, few / 64 x 64, 384 -> 512 and 640 -> 640: fp32 1 row 3.0 / 9.7,
// 4.1 / 14.9; 512 rows 8.2 / 10.6, 15.9 / 16.0 (1024, 1280 workgroups); 1024 rows 14.1 / 10.9. bf16 1 row 2.3 / 4.0; 256 rows
// 3.5 / 4.5, 5.8 / 5.9 (512, 640 workgroups); 512 rows 5.0 / 4.5.
bool few_rule(int64_t m, int64_t n, int64_t cus, bool f32) { return vx_cdiv(m, 16) * vx_cdiv(n, 16) <= (f32 ? 4 : 2) * cus; }

// 128 x 128 tiles instead of 64 x 64: half the reads per output, but fewer workgroups to hide a short sum's stores behind. us of 64 / 128:
// fp32 12800 x 512 -> 384 (300 tiles of 128) 38 / 45, 14400 x 384 -> 512 (452) 44 / 40, 60000 x 256 -> 512 (1876) 119 / 109, but 128 -> 512
// 66 / 74; bf16 of a long sum by tiles too, 16896 x 512 -> 384 (396) 16 / 16, 36000 (846) 37 / 31, of a shorter one from where the L2s
// (32 MiB in all) no longer keep x for its next column tile: 60000 x 256 -> 512 (29 MiB) 40 / 38, 100000 x 128 -> 512 (24) 40 / 45,
// 36000 x 384 -> 384 (26) 22 / 27, 52000 (38) 42 / 31
bool big_rule(int64_t m, int64_t n, int64_t k, int64_t cus, bool f32) {
  const int64_t tiles = vx_cdiv(m, 128) * vx_cdiv(n, 128);
  if (f32) return k >= 192 && 2 * tiles >= 3 * cus;
  return k >= 512 ? tiles >= 3 * cus : m * k * 2 >= 29 << 20;
}

template <typename T>
int32_t fwd_impl(const FwdArgs<T>& args, hipStream_t s) {
  FwdArgs<T> a = args;
  const int64_t cus = vx_tile_cus();
  const bool few = few_rule(a.m, a.n, cus, sizeof(T) == 4), use_big = big_rule(a.m, a.n, a.k, cus, sizeof(T) == 4);
  const int64_t t = few ? 16 : use_big ? 128 : 64;
  a.tiles_n = (int)vx_cdiv(a.n, t);
  const int64_t grid = vx_cdiv(a.m, t) * a.tiles_n;
  VX_REQUIRE(vx_launchable(grid, kTileThreads), "linear_fwd: too many rows");
  const bool fast = vx_fast(a.x, a.ldx, a.k, sizeof(T)) && vx_fast(a.w, a.ldw, a.k, sizeof(T));
  const auto kernel = few ? (fast ? linear_few<T, true> : linear_few<T, false>)
                          : use_big ? (fast ? linear_fwd<T, 128, 128, true> : linear_fwd<T, 128, 128, false>)
                                    : (fast ? linear_fwd<T, 64, 64, true> : linear_fwd<T, 64, 64, false>);
  kernel<<<(unsigned)grid, kTileThreads, 0, s>>>(a);
  VX_LAUNCH_CHECK();
  return VX_OK;
}

// bytes of the workspace: slabs of dw, column sums of row chunks, g unrounded
bool wide_g(int32_t act, int32_t dtype) { return dtype == VX_BF16 && (act == VX_ACT_GELU || act == VX_ACT_SILU); }
size_t slab_bytes(const BwdPlan& p, int64_t n, int64_t k) { return vx_align(p.splits > 1 ? (size_t)p.splits * n * k * 4 : 0); }
size_t part_bytes(const BwdPlan& p, int64_t n) { return vx_align((size_t)p.chunks * n * 4); }
size_t bwd_bytes(int64_t m, int64_t n, int64_t k, int32_t act, int32_t dtype) {
  const BwdPlan p = bwd_plan(m, n, k, dtype);
  return slab_bytes(p, n, k) + part_bytes(p, n) + (wide_g(act, dtype) ? vx_align((size_t)m * n * 4) : 0);
}

// dw, dx and, without an activation, the column sums
template <typename T, typename G>
int32_t launch_bwd(BwdArgs<T, G>& a, const BwdPlan& p, const ActArgs<T>& rows, int64_t sums, hipStream_t s) {
  const int64_t t = p.big ? 128 : 64;
  a.span = p.span;
  a.tiles_wk = (int)vx_cdiv(a.k, t);
  a.tiles_w = (int)(vx_cdiv(a.n, t) * a.tiles_wk);
  a.tiles_xk = a.tiles_wk;
  const int64_t bw = a.dw ? a.tiles_w * p.splits : 0, bx = a.dx ? vx_cdiv(a.m, t) * a.tiles_xk : 0;
  VX_REQUIRE(vx_launchable(bw + bx + sums, kTileThreads), "linear_bwd: too many rows");
  a.blocks_w = (unsigned)bw;
  a.blocks_x = (unsigned)bx;
  if (bw + bx + sums == 0) return VX_OK;
  const bool fast = vx_fast(a.g, a.ldg, a.n, sizeof(G)) && vx_fast(a.x, a.ldx, a.k, sizeof(T)) && vx_fast(a.w, a.ldw, a.k, sizeof(T));
  const auto kernel = p.big ? (fast ? linear_bwd<T, G, 128, 128, true> : linear_bwd<T, G, 128, 128, false>)
                            : (fast ? linear_bwd<T, G, 64, 64, true> : linear_bwd<T, G, 64, 64, false>);
  kernel<<<(unsigned)(bw + bx + sums), kTileThreads, 0, s>>>(a, rows);
  VX_LAUNCH_CHECK();
  return VX_OK;
}

template <typename T>
int32_t bwd_impl(const T* dy, int64_t lddy, const T* x, int64_t ldx, const T* w, int64_t ldw, const T* saved, int64_t m, int32_t n,
                 int32_t k, int32_t act, T* dpre, T* dx, T* dw, T* dbias, char* ws, int32_t dtype, hipStream_t s) {
  const BwdPlan p = bwd_plan(m, n, k, dtype);
  float *slab = (float*)ws, *part = (float*)(ws + slab_bytes(p, n, k));
  float* wide = wide_g(act, dtype) && (dx || dw) ? (float*)(ws + slab_bytes(p, n, k) + part_bytes(p, n)) : nullptr;
  const int64_t cols = vx_cdiv(n, p.lanes * (16 / (int64_t)sizeof(T)));
  const ActArgs<T> rows{dy, saved, dpre, wide, dbias ? part : nullptr, lddy, m, p.chunk, n, act, (int)p.lanes, (int)cols};
  VX_REQUIRE(vx_launchable(cols * p.chunks, 256), "linear_bwd: too many rows");
  if (act != VX_ACT_NONE) {
    act_bwd<T><<<(unsigned)(cols * p.chunks), 256, 0, s>>>(rows);
    VX_LAUNCH_CHECK();
  }
  const auto products = [&](const auto* g, int64_t ldg, int64_t sums) {
    using G = std::remove_const_t<std::remove_pointer_t<decltype(g)>>;
    BwdArgs<T, G> a{};
    a.g = g; a.x = x; a.w = w; a.dx = dx; a.dw = dw;
    a.slab = p.splits > 1 ? slab : nullptr;
    a.ldg = ldg; a.ldx = ldx; a.ldw = ldw; a.m = m; a.n = n; a.k = k;
    return launch_bwd(a, p, rows, sums, s);
  };
  int32_t rc;
  if (act == VX_ACT_NONE)
    rc = products(dy, lddy, dbias ? cols * p.chunks : 0);          // the column sums run beside the products
  else if (wide)
    rc = products((const float*)wide, n, 0);
  else
    rc = products((const T*)dpre, n, 0);
  if (rc) return rc;
  const int64_t len_w = dw && p.splits > 1 ? (int64_t)n * k : 0, len_b = dbias ? n : 0;
  const unsigned ga = (unsigned)vx_cdiv(len_w, 1024), gb = (unsigned)vx_cdiv(len_b, 64);
  if (ga + gb) {
    slab_sum<T><<<ga + gb, 256, 0, s>>>(slab, (int)p.splits, len_w, dw, part, (int)p.chunks, len_b, dbias, ga);
    VX_LAUNCH_CHECK();
  }
  return VX_OK;
}

}  // namespace

int vx_tile_cus() {
  static int cached[64];       // benign race: every writer stores the same value
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!cached[dev]) {
    int n = 0;
    cached[dev] = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0 ? n : 256;
  }
  return cached[dev];
}

static int32_t linear_check(const char* who, int64_t m, int32_t n, int32_t k, int32_t act, int32_t dtype) {
  VX_REQUIRE(dtype == VX_F32 || dtype == VX_BF16, "%s: dtype must be VX_F32 or VX_BF16", who);
  VX_REQUIRE(act >= VX_ACT_NONE && act <= VX_ACT_SILU, "%s: unknown activation %d", who, act);
  VX_REQUIRE(m >= 0 && m < (1LL << 31) && n >= 1 && k >= 1 && n <= (1 << 20) && k <= (1 << 20), "%s: bad sizes", who);
  return VX_OK;
}

extern "C" int32_t vx_linear_fwd(const void* d_x, int64_t ldx, const void* d_weight, int64_t ldw, const void* d_bias,
                                 const void* d_residual, int64_t ldr, int64_t m, int32_t n, int32_t k, int32_t act, void* d_y,
                                 void* d_pre, int32_t dtype, void* stream) {
  if (int32_t rc = linear_check("linear_fwd", m, n, k, act, dtype)) return rc;
  if (m == 0) return VX_OK;
  VX_REQUIRE(d_x && d_weight && d_y, "linear_fwd: null pointer");
  VX_REQUIRE(ldx >= 0 && ldw >= 0 && ldr >= 0, "linear_fwd: negative row stride");
  if (dtype == VX_F32)
    return fwd_impl<float>({(const float*)d_x, (const float*)d_weight, (const float*)d_bias, (const float*)d_residual, (float*)d_y,
                            (float*)d_pre, ldx, ldw, ldr, m, n, k, act, 0}, (hipStream_t)stream);
  return fwd_impl<__bf16>({(const __bf16*)d_x, (const __bf16*)d_weight, (const __bf16*)d_bias, (const __bf16*)d_residual,
                           (__bf16*)d_y, (__bf16*)d_pre, ldx, ldw, ldr, m, n, k, act, 0}, (hipStream_t)stream);
}

extern "C" size_t vx_linear_bwd_act_workspace_bytes(int64_t m, int32_t n, int32_t k, int32_t act, int32_t dtype) {
  return m <= 0 || n <= 0 || k <= 0 ? 0 : bwd_bytes(m, n, k, act, dtype);
}

extern "C" size_t vx_linear_bwd_workspace_bytes(int64_t m, int32_t n, int32_t k, int32_t dtype) {
  return vx_linear_bwd_act_workspace_bytes(m, n, k, VX_ACT_GELU, dtype);
}

extern "C" int32_t vx_linear_bwd(const void* d_dy, int64_t lddy, const void* d_x, int64_t ldx, const void* d_weight, int64_t ldw,
                                 const void* d_saved, int64_t m, int32_t n, int32_t k, int32_t act, void* d_dpre, void* d_dx,
                                 void* d_dw, void* d_dbias, int32_t dtype, void* d_workspace, size_t workspace_bytes,
                                 void* stream) {
  if (int32_t rc = linear_check("linear_bwd", m, n, k, act, dtype)) return rc;
  const hipStream_t s = (hipStream_t)stream;
  if (m == 0) {       // sums over no rows
    const int64_t nk = d_dw ? (int64_t)n * k : 0, nb = d_dbias ? n : 0;
    const size_t e = dtype == VX_F32 ? 4 : 2;
    if (nk)
      if (int32_t rc = vx_fill_async(d_dw, 0, nk * e, s)) return rc;
    if (nb)
      if (int32_t rc = vx_fill_async(d_dbias, 0, nb * e, s)) return rc;
    return VX_OK;
  }
  VX_REQUIRE(d_dy && d_x && d_weight, "linear_bwd: null pointer");
  VX_REQUIRE(lddy >= 0 && ldx >= 0 && ldw >= 0, "linear_bwd: negative row stride");
  VX_REQUIRE(act == VX_ACT_NONE || (d_saved && d_dpre), "linear_bwd: an activation needs d_saved and d_dpre");
  if (workspace_bytes < bwd_bytes(m, n, k, act, dtype) || !d_workspace) {
    vx_set_error("linear_bwd: workspace too small");
    return VX_ERR_WORKSPACE;
  }
  if (dtype == VX_F32)
    return bwd_impl<float>((const float*)d_dy, lddy, (const float*)d_x, ldx, (const float*)d_weight, ldw, (const float*)d_saved, m, n,
                           k, act, (float*)d_dpre, (float*)d_dx, (float*)d_dw, (float*)d_dbias, (char*)d_workspace, dtype, s);
  return bwd_impl<__bf16>((const __bf16*)d_dy, lddy, (const __bf16*)d_x, ldx, (const __bf16*)d_weight, ldw, (const __bf16*)d_saved, m,
                          n, k, act, (__bf16*)d_dpre, (__bf16*)d_dx, (__bf16*)d_dw, (__bf16*)d_dbias, (char*)d_workspace, dtype, s);
}
