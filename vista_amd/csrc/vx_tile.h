// Matrix-tile toolkit of the dense kernels (vx_linear.hip, vx_attn.hip): operand staging into LDS in the order in which
// v_mfma_f32_16x16x32_bf16 reads its fragments, for fp32 (exact three-plane bf16 split, six products) and bf16.
//
// A product is C[m][n] = sum_k X[m][k] * W[n][k]. The matrix instruction takes W as its row operand and X as its column
// operand, so that lane (c = lane & 15, g = lane >> 4) holds C[m0 + c][n0 + 4 g + 0..3]: four neighbours of one output row,
// one 16- or 8-byte store.
//
// LDS image of an operand tile: fragments of 16 rows x 32 k, 1 KB each and one per plane, in lane order -- lane (c, g) of a
// fragment read takes the 16 bytes {k = 8 g .. 8 g + 7} of row c with one ds_read_b128, 64 lanes over 1 KB: no bank
// conflicts. The 16-byte pieces of a fragment are XOR-ed by its row block (& 7), which also spreads the writes of a
// k-strided operand, whose lanes each own a few rows (16 lanes over 16 different pieces of the 256-byte bank row).
#pragma once
#include "vx_common.h"
#include "vx_split.h"

typedef float vx_f32x4u __attribute__((ext_vector_type(4), aligned(4)));      // vector accesses at element alignment
typedef float vx_f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef unsigned vx_u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned vx_u32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned vx_u32x1u __attribute__((aligned(2)));
typedef unsigned vx_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileThreads = 256;
constexpr int kFragBytes = 1024;

// consecutive tiles on one XCD (workgroups are dealt to the 8 XCDs round robin): they share operand rows in its L2
__device__ __forceinline__ unsigned vx_xcd_tile(unsigned b, unsigned n) {
  const unsigned q = n >> 3, r = n & 7, x = b & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (b >> 3);
}

template <typename T>
struct VxType;
template <>
struct VxType<float> {
  static constexpr int NPL = 3;   // bf16 planes per value
  static constexpr int BK = 32;   // reduction values per staged step of a GEMM
};
template <>
struct VxType<__bf16> {
  static constexpr int NPL = 1;
  static constexpr int BK = 64;
};

template <int NPL>
struct VxFrag {
  bf16x8 p[NPL];
};

// c += w * x; fp32: the six plane products down to 2^-24 of the largest, smallest first
__device__ __forceinline__ vx_f32x4 vx_mma(const VxFrag<1>& w, const VxFrag<1>& x, vx_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[0], x.p[0], c, 0, 0, 0);
}
__device__ __forceinline__ vx_f32x4 vx_mma(const VxFrag<3>& w, const VxFrag<3>& x, vx_f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[2], x.p[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[0], x.p[2], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[1], x.p[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[1], x.p[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[0], x.p[1], c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[0], x.p[0], c, 0, 0, 0);
}

// eight fp32 values -> operand planes (bf16: rounded to nearest even)
__device__ __forceinline__ void vx_planes(const float (&v)[8], VxFrag<3>& f) {
  const Planes p = split8s(v);
  f.p[0] = p.h;
  f.p[1] = p.m;
  f.p[2] = p.l;
}
__device__ __forceinline__ void vx_planes(const float (&v)[8], VxFrag<1>& f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f.p[0][i] = (__bf16)v[i];
}

// ---- eight k-consecutive values of one row ---------------------------------------------------------------------
template <typename T>
struct VxRow8;
template <>
struct VxRow8<float> {
  float v[8];
  // n: how many of the eight exist (<= 0: none); the others are 0
  __device__ __forceinline__ void load(const float* p, int n) {
    if (n >= 8) {
      const vx_f32x4u a = *reinterpret_cast<const vx_f32x4u*>(p), b = *reinterpret_cast<const vx_f32x4u*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
  }
  __device__ __forceinline__ void planes(VxFrag<3>& f) const { vx_planes(v, f); }
};
template <>
struct VxRow8<__bf16> {
  vx_u32x4 v;
  __device__ __forceinline__ void load(const __bf16* p, int n) {
    if (n >= 8) {
      v = *reinterpret_cast<const vx_u32x4u*>(p);
    } else {
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned lo = 2 * i < n ? q[2 * i] : 0u, hi = 2 * i + 1 < n ? q[2 * i + 1] : 0u;
        v[i] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ void planes(VxFrag<1>& f) const { f.p[0] = __builtin_bit_cast(bf16x8, v); }
};

// ---- W rows x eight k's of a k-strided operand (element (row, k) at p[k * ld + row]) ----------------------------
template <typename T, int W>
struct VxCol8;
template <int W>
struct VxCol8<float, W> {
  float v[8][W];
  // row k of the eight: W values from p, n of them exist (<= 0: none)
  __device__ __forceinline__ void load(int k, const float* p, int n) {
    if (n >= W) {
      if constexpr (W == 4) {
        const vx_f32x4u a = *reinterpret_cast<const vx_f32x4u*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][j] = a[j];
      } else if constexpr (W == 2) {
        const vx_f32x2u a = *reinterpret_cast<const vx_f32x2u*>(p);
        v[k][0] = a[0];
        v[k][1] = a[1];
      } else {
        v[k][0] = p[0];
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) v[k][j] = j < n ? p[j] : 0.0f;
    }
  }
  __device__ __forceinline__ void planes(int j, VxFrag<3>& f) const {
    const float x[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
    vx_planes(x, f);
  }
};
template <int W>
struct VxCol8<__bf16, W> {
  static_assert(W == 2 || W == 4, "pairs of 16-bit rows");
  unsigned v[8][W / 2];
  __device__ __forceinline__ void load(int k, const __bf16* p, int n) {
    if (n >= W) {
      if constexpr (W == 4) {
        const vx_u32x2u a = *reinterpret_cast<const vx_u32x2u*>(p);
        v[k][0] = a[0];
        v[k][1] = a[1];
      } else {
        v[k][0] = *reinterpret_cast<const vx_u32x1u*>(p);
      }
    } else {
      const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int j = 0; j < W / 2; ++j) {
        const unsigned lo = 2 * j < n ? q[2 * j] : 0u, hi = 2 * j + 1 < n ? q[2 * j + 1] : 0u;
        v[k][j] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ void planes(int j, VxFrag<1>& f) const {
    vx_u32x4 o;
    const unsigned sel = j & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_amdgcn_perm(v[2 * i + 1][j >> 1], v[2 * i][j >> 1], sel);
    f.p[0] = __builtin_bit_cast(bf16x8, o);
  }
};

// ---- LDS image --------------------------------------------------------------------------------------------------
// fragment (row block rb, k step ks) of an image with NK k steps per row block; planes are `plane` bytes apart
template <int NPL>
__device__ __forceinline__ void vx_frag_store(char* img, int plane, int frag, int key, int slot, const VxFrag<NPL>& f) {
  char* p = img + frag * kFragBytes + ((slot ^ (key & 7)) << 4);
#pragma unroll
  for (int i = 0; i < NPL; ++i) *reinterpret_cast<bf16x8*>(p + i * plane) = f.p[i];
}
template <int NPL>
__device__ __forceinline__ void vx_frag_load(const char* img, int plane, int frag, int key, int lane, VxFrag<NPL>& f) {
  const char* p = img + frag * kFragBytes + ((lane ^ (key & 7)) << 4);
#pragma unroll
  for (int i = 0; i < NPL; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(p + i * plane);
}

// ---- GEMM ---------------------------------------------------------------------------------------------------------
// operand tile: p points at (first row of the tile, k = 0)
//   KC (k contiguous): element (r, k) at p[r * ld + k];  KS (k strided): element (r, k) at p[k * ld + r]
// rows: rows that exist from the tile's first on; kmask (KS only): k's whose byte is 0 read as 0, whatever they hold
constexpr int KC = 0, KS = 1;
template <typename T>
struct VxOperand {
  const T* p;
  long long ld;
  int rows;
  const uint8_t* kmask;
};

// stages R rows x BK k's with 256 threads: registers first (load), then the LDS image (store)
template <typename T, int MODE, int R>
struct VxStage {
  static constexpr int BK = VxType<T>::BK, NPL = VxType<T>::NPL, NK = BK / 32;
  static constexpr int PLANE = (R / 16) * NK * kFragBytes;
  static constexpr int BYTES = PLANE * NPL;
  static constexpr int NI = R * BK / 8 / kTileThreads;            // 8-value items per thread (KC)
  static constexpr int W = R * BK / 8 / kTileThreads;             // rows per thread (KS)
  static_assert(R * BK / 8 % kTileThreads == 0, "every thread stages the same amount");
  struct Empty {};
  VxRow8<T> a[MODE == KC ? NI : 1];
  VxCol8<T, MODE == KS ? W : 2> b;

  __device__ __forceinline__ void load(const VxOperand<T>& o, int k0, int kend, int tid) {
    if constexpr (MODE == KC) {
      const int wave = tid >> 6, lane = tid & 63;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int frag = i * (kTileThreads / 64) + wave, r = frag / NK * 16 + (lane & 15);
        const int k = k0 + frag % NK * 32 + (lane >> 4) * 8;
        a[i].load(o.p + r * o.ld + k, r < o.rows ? kend - k : 0);
      }
    } else {
      const int r = tid % (R / W) * W, k = k0 + tid / (R / W) * 8;
      const T* p = o.p + k * o.ld + r;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool live = k + i < kend && (o.kmask == nullptr || o.kmask[k + i]);
        b.load(i, p + i * o.ld, live ? o.rows - r : 0);
      }
    }
  }
  __device__ __forceinline__ void store(char* img, int tid) const {
    VxFrag<NPL> f;
    if constexpr (MODE == KC) {
      const int wave = tid >> 6, lane = tid & 63;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int frag = i * (kTileThreads / 64) + wave;
        a[i].planes(f);
        vx_frag_store(img, PLANE, frag, frag / NK, lane, f);
      }
    } else {
      const int r = tid % (R / W) * W, kg = tid / (R / W);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        b.planes(j, f);
        const int rr = r + j, rb = rr >> 4;
        vx_frag_store(img, PLANE, rb * NK + (kg >> 2), rb, (rr & 15) + 16 * (kg & 3), f);
      }
    }
  }
};

// LDS bytes of vx_gemm_loop
template <typename T, int TM, int TN>
constexpr int vx_gemm_lds() {
  return (TM + TN) * VxType<T>::BK * 2 * VxType<T>::NPL;
}

// acc[mi][ni] += the TM x TN tile's product over k in [k0, kend); wave (wm, wn) of 2 x 2 owns TM/2 x TN/2. One LDS image,
// two barriers per step: the next step's operands travel to registers while this one's are multiplied, and the two or
// three workgroups of a CU cover each other's barriers. Ends with a barrier: the caller may reuse the LDS.
template <typename T, int XM, int WM, int TM, int TN>
__device__ __forceinline__ void vx_gemm_loop(const VxOperand<T>& X, const VxOperand<T>& W, int k0, int kend, char* lds,
                                             vx_f32x4 (&acc)[TM / 32][TN / 32]) {
  constexpr int BK = VxType<T>::BK, NPL = VxType<T>::NPL, NK = BK / 32;
  using SX = VxStage<T, XM, TM>;
  using SW = VxStage<T, WM, TN>;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  char *ix = lds, *iw = lds + SX::BYTES;
  SX sx;
  SW sw;
  if (k0 < kend) {
    sx.load(X, k0, kend, tid);
    sw.load(W, k0, kend, tid);
  }
  for (int k = k0; k < kend; k += BK) {
    sx.store(ix, tid);
    sw.store(iw, tid);
    __syncthreads();
    if (k + BK < kend) {
      sx.load(X, k + BK, kend, tid);
      sw.load(W, k + BK, kend, tid);
    }
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) {
      VxFrag<NPL> fx[TM / 32];
#pragma unroll
      for (int mi = 0; mi < TM / 32; ++mi) {
        const int rb = wm * (TM / 32) + mi;
        vx_frag_load(ix, SX::PLANE, rb * NK + ks, rb, lane, fx[mi]);
      }
#pragma unroll
      for (int ni = 0; ni < TN / 32; ++ni) {
        const int rb = wn * (TN / 32) + ni;
        VxFrag<NPL> fw;
        vx_frag_load(iw, SW::PLANE, rb * NK + ks, rb, lane, fw);
#pragma unroll
        for (int mi = 0; mi < TM / 32; ++mi) acc[mi][ni] = vx_mma(fw, fx[mi], acc[mi][ni]);
      }
    }
    __syncthreads();
  }
}

template <int A, int B>
__device__ __forceinline__ void vx_acc_zero(vx_f32x4 (&acc)[A][B]) {
#pragma unroll
  for (int i = 0; i < A; ++i)
#pragma unroll
    for (int j = 0; j < B; ++j) acc[i][j] = vx_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// f(m, n, value4) for every accumulator of this lane: m, n relative to the tile, n a multiple of 4
template <int TM, int TN, typename F>
__device__ __forceinline__ void vx_acc_each(const vx_f32x4 (&acc)[TM / 32][TN / 32], F&& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
#pragma unroll
  for (int mi = 0; mi < TM / 32; ++mi)
#pragma unroll
    for (int ni = 0; ni < TN / 32; ++ni)
      f(wm * (TM / 2) + mi * 16 + (lane & 15), wn * (TN / 2) + ni * 16 + (lane >> 4) * 4, acc[mi][ni]);
}

// ---- up to four neighbours of a row -------------------------------------------------------------------------------
__device__ __forceinline__ vx_f32x4 vx_load4(const float* p, int n) {
  if (n >= 4) return *reinterpret_cast<const vx_f32x4u*>(p);
  vx_f32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.0f;
  return v;
}
__device__ __forceinline__ vx_f32x4 vx_load4(const __bf16* p, int n) {
  vx_f32x4 v;
  if (n >= 4) {
    const vx_u32x2u a = *reinterpret_cast<const vx_u32x2u*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(i & 1 ? a[i >> 1] & 0xffff0000u : a[i >> 1] << 16);
    return v;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
  return v;
}
__device__ __forceinline__ void vx_store4(float* p, const vx_f32x4& v, int n) {
  if (n >= 4) {
    *reinterpret_cast<vx_f32x4u*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) p[i] = v[i];
}
__device__ __forceinline__ void vx_store4(__bf16* p, const vx_f32x4& v, int n) {
  if (n >= 4) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    bf16x4 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = (__bf16)v[i];
    *reinterpret_cast<vx_u32x2u*>(p) = __builtin_bit_cast(vx_u32x2u, h);
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) p[i] = (__bf16)v[i];
}

// compute units of the current device (cached per device; 256 if it cannot be asked)
int vx_tile_cus();
