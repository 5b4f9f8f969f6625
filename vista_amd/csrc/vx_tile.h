// Matrix-tile toolkit of the dense kernels (vx_linear.hip, vx_attn.hip): operand staging into LDS in the order in which
// v_mfma_f32_16x16x32_bf16 reads its fragments, for fp32 (exact three-plane bf16 split, six products) and bf16.
//
// A product is C[m][n] = sum_k X[m][k] * W[n][k]. The matrix instruction takes W as its row operand and X as its column
// operand, so that lane (c = lane & 15, g = lane >> 4) holds four neighbours of row m0 + c. The GEMMs deal the rows of W to
// the blocks of a 32-row group four at a time (vx_row_w), so that a lane's two accumulators of a group are eight neighbours
// C[m0 + c][n0 + 8 g + 0..7], and the four lanes of a row store 64 (bf16) or 128 (fp32) bytes in one piece.
//
// LDS image of an operand tile: fragments of 16 rows x 32 k, 1 KB each and one per plane, in lane order -- lane (c, g) of a
// fragment read takes the 16 bytes {k = 8 g .. 8 g + 7} of row c with one ds_read_b128, 64 lanes over 1 KB: no bank
// conflicts. Two more rules keep the writes free of them: the 16-byte pieces of a fragment are XOR-ed by their k group
// (a wave that writes whole 128-byte rows spreads a row's eight pieces over eight bank groups), and every block of 16 rows
// starts 16 bytes later (a k-strided operand's lanes each own a few rows: 16 lanes over 16 different pieces).
#pragma once
#include "vx_common.h"
#include "vx_split.h"

typedef float vx_f32x4u __attribute__((ext_vector_type(4), aligned(4)));      // vector accesses at element alignment
typedef float vx_f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef unsigned vx_u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned vx_u32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned vx_u32x1u __attribute__((aligned(2)));
typedef unsigned vx_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned vx_u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned vx_u32x3 __attribute__((ext_vector_type(3)));

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
  static constexpr int NPL_F32 = 3;   // ... of an fp32 intermediate that meets such values in a product
  static constexpr int BK = 32;   // reduction values per staged step of a GEMM (64: small tiles of k-contiguous operands)
};
template <>
struct VxType<__bf16> {
  static constexpr int NPL = 1;
  static constexpr int NPL_F32 = 2;
  static constexpr int BK = 64;
};

template <int NPL>
struct VxFrag {
  bf16x8 p[NPL];
};

// the plane products of c += w * x, in order: three planes each (fp32): six, down to 2^-21 of |w x|, smallest first
// (the next two would take the error of 18 calls down by 0 to 15 % and their time up by 10 to 18 %: it comes from the additions); one and two
// (bf16 and an fp32 intermediate rounded to 16 bits): both. Callers loop over independent accumulators inside a product, so that
// no matrix instruction waits for the one before it.
template <int PW, int PX>
struct VxProducts;
template <>
struct VxProducts<1, 1> {
  static constexpr int N = 1, W[1] = {0}, X[1] = {0};
};
template <>
struct VxProducts<1, 2> {
  static constexpr int N = 2, W[2] = {0, 0}, X[2] = {1, 0};
};
template <>
struct VxProducts<3, 3> {
  static constexpr int N = 6, W[6] = {2, 0, 1, 1, 0, 0}, X[6] = {0, 2, 1, 0, 1, 0};
};
template <int PW, int PX>
__device__ __forceinline__ vx_f32x4 vx_mma(int product, const VxFrag<PW>& w, const VxFrag<PX>& x, vx_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.p[VxProducts<PW, PX>::W[product]], x.p[VxProducts<PW, PX>::X[product]], c, 0, 0, 0);
}

// eight fp32 values -> operand planes (three: exact; one and two: rounded to nearest even, to 8 and 16 bits)
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
__device__ __forceinline__ void vx_planes(const float (&v)[8], VxFrag<2>& f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f.p[0][i] = (__bf16)v[i];
    f.p[1][i] = (__bf16)(v[i] - (float)f.p[0][i]);
  }
}

// ---- buffer loads -------------------------------------------------------------------------------------------------
// 32-bit offsets from a wave-uniform base, with a range check that returns 0: masked lanes and tails need no branch (a branch
// around a load whose other side writes zeros makes the load wait). kVxOut is past every range.
constexpr unsigned kVxRange = 0x80000000u;
constexpr int kVxOut = (int)0x80000000u;
typedef __amdgpu_buffer_rsrc_t vx_rsrc;
__device__ __forceinline__ vx_rsrc vx_buffer(const void* base, unsigned range = kVxRange) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)range, 0x00020000);   // raw, 32-bit data format
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
  __device__ __forceinline__ void load(vx_rsrc b, int at) {
    const vx_u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0), y = __builtin_amdgcn_raw_buffer_load_b128(b, at, 16, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __uint_as_float(x[i]);
      v[4 + i] = __uint_as_float(y[i]);
    }
  }
  template <int PL>
  __device__ __forceinline__ void planes(VxFrag<PL>& f) const { vx_planes(v, f); }
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
  __device__ __forceinline__ void load(vx_rsrc b, int at) { v = __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0); }
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
#pragma unroll
        for (int j = 0; j < W; ++j) v[k][j] = p[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) v[k][j] = j < n ? p[j] : 0.0f;
    }
  }
  __device__ __forceinline__ void load(int k, vx_rsrc b, int at) {
    if constexpr (W == 4) {
      const vx_u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k][j] = __uint_as_float(a[j]);
    } else if constexpr (W == 3) {
      const vx_u32x3 a = __builtin_amdgcn_raw_buffer_load_b96(b, at, 0, 0);
#pragma unroll
      for (int j = 0; j < 3; ++j) v[k][j] = __uint_as_float(a[j]);
    } else if constexpr (W == 2) {
      const vx_u32x2 a = __builtin_amdgcn_raw_buffer_load_b64(b, at, 0, 0);
      v[k][0] = __uint_as_float(a[0]);
      v[k][1] = __uint_as_float(a[1]);
    } else {
      v[k][0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, at, 0, 0));
    }
  }
  template <int PL>
  __device__ __forceinline__ void planes(int j, VxFrag<PL>& f) const {
    const float x[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
    vx_planes(x, f);
  }
};
template <int W>
struct VxCol8<__bf16, W> {
  static_assert(W == 2 || W == 4 || W == 6, "pairs of 16-bit rows");
  unsigned v[8][W / 2];
  __device__ __forceinline__ void load(int k, const __bf16* p, int n) {
    if (n >= W) {
      if constexpr (W == 4) {
        const vx_u32x2u a = *reinterpret_cast<const vx_u32x2u*>(p);
        v[k][0] = a[0];
        v[k][1] = a[1];
      } else {
#pragma unroll
        for (int j = 0; j < W / 2; ++j) v[k][j] = reinterpret_cast<const vx_u32x1u*>(p)[j];
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
  __device__ __forceinline__ void load(int k, vx_rsrc b, int at) {
    if constexpr (W == 4) {
      const vx_u32x2 a = __builtin_amdgcn_raw_buffer_load_b64(b, at, 0, 0);
      v[k][0] = a[0];
      v[k][1] = a[1];
    } else if constexpr (W == 6) {
      const vx_u32x3 a = __builtin_amdgcn_raw_buffer_load_b96(b, at, 0, 0);
#pragma unroll
      for (int j = 0; j < 3; ++j) v[k][j] = a[j];
    } else {
      v[k][0] = __builtin_amdgcn_raw_buffer_load_b32(b, at, 0, 0);
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

// ---- copies from memory to LDS ----------------------------------------------------------------------------------
// one fragment (1 KB, in lane order in memory too) straight to LDS, without registers; vx_arrived() waits for all of a wave's
__device__ __forceinline__ void vx_copy_frag(const void* from, char* to, int lane) {
  __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(const_cast<char*>((const char*)from) + lane * 16),
                                   (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
__device__ __forceinline__ void vx_arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- LDS image --------------------------------------------------------------------------------------------------
// byte of (row block rb, k step ks, slot) of an image with NK k steps; slot = row & 15 + 16 * k group
template <int NK>
constexpr int vx_image_block() { return NK * kFragBytes + 16; }
template <int NK>
__device__ __forceinline__ int vx_image_at(int rb, int ks, int slot) {
  return rb * vx_image_block<NK>() + ks * kFragBytes + ((slot ^ (slot >> 4 & 3) ^ (ks & 1) << 2) << 4);
}
template <int NPL>
__device__ __forceinline__ void vx_frag_store(char* p, int plane, const VxFrag<NPL>& f) {
#pragma unroll
  for (int i = 0; i < NPL; ++i) *reinterpret_cast<bf16x8*>(p + i * plane) = f.p[i];
}
template <int NPL>
__device__ __forceinline__ void vx_frag_load(const char* p, int plane, VxFrag<NPL>& f) {
#pragma unroll
  for (int i = 0; i < NPL; ++i) f.p[i] = *reinterpret_cast<const bf16x8*>(p + i * plane);
}

// ---- GEMM ---------------------------------------------------------------------------------------------------------
// operand tile: p points at (first row of the tile, k = 0)
//   KC (k contiguous): element (r, k) at p[r * ld + k];  KS (k strided): element (r, k) at p[k * ld + r]
// rows: rows that exist from the tile's first on.
// FAST operands are read by buffer loads: 16-byte aligned base and row stride, and (vx_fast) rows (KS) or the reduction (KC) in
// multiples of 8, ld no smaller than a row, the offsets of a tile in 31 bits; KS tiles of 192 rows want multiples of 24. The
// others are read element by element at their edges, and every load waits for its own branch.
constexpr int KC = 0, KS = 1;
template <typename T>
struct VxOperand {
  const T* p;
  long long ld;
  int rows;
};
static inline bool vx_fast(const void* p, int64_t ld, int64_t width, int64_t esize) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * esize % 16 == 0 && width % 8 == 0 && ld >= width && ld < (1 << 21);
}

// row n of a W tile -> its row in the image (block * 16 + row of the block), and back
__device__ __forceinline__ int vx_row_w(int n) { return (n & ~31) + (n & 4) * 4 + (n >> 1 & 12) + (n & 3); }
__device__ __forceinline__ int vx_row_n(int r) { return (r & ~31) + (r & 12) * 2 + (r >> 2 & 4) + (r & 3); }
// stages R rows x BK k's with 256 threads: registers first (load), then the LDS image (store)
template <typename T, int NPL, int MODE, int R, int BK, bool FAST, bool IS_W>
struct VxStage {
  static constexpr int NK = BK / 32, E = sizeof(T);
  static constexpr int PLANE = (R / 16) * vx_image_block<NK>();
  static constexpr int BYTES = PLANE * NPL;
  static constexpr int NI = R * BK / 8 / kTileThreads;            // KC: 8-value items per thread; KS: rows per thread
  static constexpr int W = NI;
  static_assert(R * BK / 8 % kTileThreads == 0, "every thread stages the same amount");
  VxRow8<T> a[MODE == KC ? NI : 1];
  VxCol8<T, MODE == KS ? W : 2> b;

  // KC item i of a thread: row (of the image) and k group. bf16: eight lanes read a row's 128 bytes; fp32: a lane's eight
  // values are two loads, four lanes a row
  static __device__ __forceinline__ void item(int i, int tid, int& row, int& kc) {
    const int wave = tid >> 6, l = tid & 63, blk = i * (kTileThreads / 64) + wave;
    if constexpr (NK == 2) {
      row = (blk >> 1) * 16 + (l >> 3 & 1) * 8 + (blk & 1) * 4 + (l >> 4);
      kc = l & 7;
    } else {
      row = blk * 16 + (l & 15);
      kc = l >> 4;
    }
  }
  // KS: k group of a thread. Where a wave's halves have a group each, the two are two apart: LDS serves lanes of both halves
  // together, and the XOR then keeps their pieces apart
  static __device__ __forceinline__ int group(int tid) {
    const int i = tid / (R / W);
    return R / W == 32 ? (i & 1) * 2 + (i >> 1 & 1) + (i & 4) : i;
  }
  __device__ __forceinline__ void load(const VxOperand<T>& o, int k0, int kend, int tid) {
    if constexpr (MODE == KC) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        int row, kc;
        item(i, tid, row, kc);
        if constexpr (IS_W) row = vx_row_n(row);
        if constexpr (FAST)
          a[i].load(vx_buffer(o.p + k0), row < o.rows && kc * 8 < kend - k0 ? row * (int)o.ld * E + kc * 8 * E : kVxOut);
        else
          a[i].load(o.p + row * o.ld + k0 + kc * 8, row < o.rows ? kend - k0 - kc * 8 : 0);
      }
    } else {
      const int r = tid % (R / W) * W, kg = group(tid) * 8;
      if constexpr (FAST) {
        // the range ends with the reduction: k's past it read as 0 (the whole offset is the lane's: the check sees all of it)
        const long long left = (long long)(kend - k0) * o.ld * E;
        const vx_rsrc buf = vx_buffer(o.p + (long long)k0 * o.ld, left < (long long)kVxRange ? (unsigned)left : kVxRange);
        const int at = r < o.rows ? kg * (int)o.ld * E + r * E : kVxOut;
#pragma unroll
        for (int i = 0; i < 8; ++i) b.load(i, buf, at + i * (int)o.ld * E);
      } else {
        const T* p = o.p + (long long)(k0 + kg) * o.ld + r;
#pragma unroll
        for (int i = 0; i < 8; ++i) b.load(i, p + i * o.ld, k0 + kg + i < kend ? o.rows - r : 0);
      }
    }
  }
  __device__ __forceinline__ void store(char* img, int tid) const {
    VxFrag<NPL> f;
    if constexpr (MODE == KC) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        int row, kc;
        item(i, tid, row, kc);
        a[i].planes(f);
        vx_frag_store(img + vx_image_at<NK>(row >> 4, kc >> 2, (row & 15) + 16 * (kc & 3)), PLANE, f);
      }
    } else {
      const int r = tid % (R / W) * W, kg = group(tid);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        b.planes(j, f);
        const int row = IS_W ? vx_row_w(r + j) : r + j;
        vx_frag_store(img + vx_image_at<NK>(row >> 4, kg >> 2, (row & 15) + 16 * (kg & 3)), PLANE, f);
      }
    }
  }
};

// LDS bytes of vx_gemm_loop
template <typename T, int TM, int TN, int BK = VxType<T>::BK, int PX = VxType<T>::NPL>
constexpr int vx_gemm_lds() {
  return (TM * PX + TN * VxType<T>::NPL) / 16 * vx_image_block<BK / 32>();
}

// acc[mi][ni] += the TM x TN tile's product over k in [k0, kend); wave (wm, wn) of 2 x 2 owns TM/2 x TN/2. One LDS image,
// two barriers per step: the next step's operands travel to registers while this one's are multiplied, and the two or
// three workgroups of a CU cover each other's barriers and splitting. Measured against it: two images with one barrier a step and
// the split of the next step among this one's products 4096^3 fp32 694 -> 869 us, 204800 x 384 -> 512 bf16 134 -> 170 us (one
// workgroup less a CU); two and three steps in flight: no difference. Ends with a barrier: the caller may reuse the LDS.
// TX, PX: the type and planes of X where they are not those of W
template <typename T, int XM, int WM, int TM, int TN, bool FAST, int BK = VxType<T>::BK, typename TX = T, int PX = VxType<T>::NPL>
__device__ __forceinline__ void vx_gemm_loop(const VxOperand<TX>& X, const VxOperand<T>& W, int k0, int kend, char* lds,
                                             vx_f32x4 (&acc)[TM / 32][TN / 32]) {
  constexpr int NPL = VxType<T>::NPL, NK = BK / 32;
  using SX = VxStage<TX, PX, XM, TM, BK, FAST, false>;
  using SW = VxStage<T, NPL, WM, TN, BK, FAST, true>;
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
      const char* px = ix + vx_image_at<NK>(wm * (TM / 32), ks, lane);
      const char* pw = iw + vx_image_at<NK>(wn * (TN / 32), ks, lane);
      VxFrag<PX> fx[TM / 32];
#pragma unroll
      for (int mi = 0; mi < TM / 32; ++mi) vx_frag_load(px + mi * vx_image_block<NK>(), SX::PLANE, fx[mi]);
      constexpr int G = TM / 32 >= 4 ? 1 : 2;     // W blocks at a time: four independent accumulators
#pragma unroll
      for (int ni = 0; ni < TN / 32; ni += G) {
        VxFrag<NPL> fw[G];
#pragma unroll
        for (int u = 0; u < G; ++u) vx_frag_load(pw + (ni + u) * vx_image_block<NK>(), SW::PLANE, fw[u]);
#pragma unroll
        for (int pr = 0; pr < VxProducts<NPL, PX>::N; ++pr)
#pragma unroll
          for (int u = 0; u < G; ++u)
#pragma unroll
            for (int mi = 0; mi < TM / 32; ++mi) acc[mi][ni + u] = vx_mma(pr, fw[u], fx[mi], acc[mi][ni + u]);
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

// f(mi, m, j, n, first, second) for every pair of accumulators of this lane: the values n .. n + 7 of row m, relative to the tile;
// mi and j are their compile-time numbers
template <int TM, int TN, typename F>
__device__ __forceinline__ void vx_acc_each(const vx_f32x4 (&acc)[TM / 32][TN / 32], F&& f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
#pragma unroll
  for (int mi = 0; mi < TM / 32; ++mi)
#pragma unroll
    for (int j = 0; j < TN / 64; ++j)
      f(mi, wm * (TM / 2) + mi * 16 + (lane & 15), j, wn * (TN / 2) + j * 32 + (lane >> 4) * 8, acc[mi][2 * j], acc[mi][2 * j + 1]);
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
// 16 bytes of a row as quads
__device__ __forceinline__ void vx_loadq(const float* p, int n, vx_f32x4 (&v)[1]) { v[0] = vx_load4(p, n); }
__device__ __forceinline__ void vx_loadq(const __bf16* p, int n, vx_f32x4 (&v)[2]) {
  if (n >= 8) {
    const vx_u32x4 a = *reinterpret_cast<const vx_u32x4u*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = __uint_as_float(i & 1 ? a[i >> 1] & 0xffff0000u : a[i >> 1] << 16);
    return;
  }
  v[0] = vx_load4(p, n);
  v[1] = vx_load4(p + 4, n - 4);
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

// eight neighbours, `n` of which exist; ONCE: past the caches, for what this launch does not read again
// (one function a type: a template's parameter would take the vector without its element alignment)
template <bool ONCE>
__device__ __forceinline__ void vx_put(const vx_f32x4u& v, vx_f32x4u* p) {
  if constexpr (ONCE)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}
template <bool ONCE>
__device__ __forceinline__ void vx_put(const vx_u32x4u& v, vx_u32x4u* p) {
  if constexpr (ONCE)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}
template <bool ONCE = false>
__device__ __forceinline__ void vx_store8(float* p, const vx_f32x4& a, const vx_f32x4& b, int n) {
  if (n >= 8) {
    vx_put<ONCE>(static_cast<vx_f32x4u>(a), reinterpret_cast<vx_f32x4u*>(p));
    vx_put<ONCE>(static_cast<vx_f32x4u>(b), reinterpret_cast<vx_f32x4u*>(p + 4));
    return;
  }
  vx_store4(p, a, n);
  vx_store4(p + 4, b, n - 4);
}
template <bool ONCE = false>
__device__ __forceinline__ void vx_store8(__bf16* p, const vx_f32x4& a, const vx_f32x4& b, int n) {
  if (n >= 8) {
    bf16x8 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = (__bf16)a[i];
      h[4 + i] = (__bf16)b[i];
    }
    vx_put<ONCE>(__builtin_bit_cast(vx_u32x4u, h), reinterpret_cast<vx_u32x4u*>(p));
    return;
  }
  vx_store4(p, a, n);
  vx_store4(p + 4, b, n - 4);
}

// whether a launch of `blocks` workgroups of `threads` has fewer than the 2^32 work items that one may have
static inline bool vx_launchable(int64_t blocks, int threads) { return blocks < (1LL << 32) / threads; }

// compute units of the current device (cached per device; 256 if it cannot be asked)
int vx_tile_cus();
