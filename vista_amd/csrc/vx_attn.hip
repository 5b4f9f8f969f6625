// Attention softmax(scale q k^T) v with a key mask, and its backward pass (cross-view attention:
// det3d/models/necks/attention.py:55-124, two read-outs -- query / key heads -- over one value map).
//
// Forward: one pass over the keys with a running maximum and sum per query; probabilities never leave the registers.
// Backward: probabilities recomputed from the saved (maximum, 1 / sum); see attn_pds below.
// fp32 operands run as three exact bf16 planes (six products, fp32 accumulation), bf16 ones directly (vx_tile.h). Softmax
// statistics, probabilities and sums over queries are fp32; for bf16 tensors the probabilities are rounded to 16 bits (two planes) where
// they become operands: to 8 bits, their errors would be about as large as the output's own rounding (2-norm 0.0024 of the output
// instead of 0.0017). The backward pass keeps P and dS in fp32; as operands beside bf16 ones they are two planes as well.
// A masked key has no part in anything, whatever its rows hold; a query without keys gives zeros, one whose scores all leave fp32's range
// NaN. No atomics: bitwise
// reproducible.
#include <float.h>

#include "vx_tile.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
struct AttnArgs {
  const T *q, *k, *v;
  const uint8_t* mask;                       // [batch][mask_b] bytes, or null
  long long q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h, mask_b;
  int sq, sk, h, gk, gv, d, dv;              // gk, gv: query heads per key / value head
  const int *index, *place, *count;          // attn_live's lists of the keys that take part, or null (no mask, or few queries)
  float scale2, sign;                        // scale * log2(e) as scale2 > 0 (1 for scale 0) and a sign of 1, -1 or 0, so that the
                                             // maximum of the scores is that of the scaled ones and masked ones stay -inf
};

template <typename T>
struct FwdArgs : AttnArgs<T> {
  const char *k_img, *v_img;                 // attn_pack's images, tile after tile of each key / value head
  T *out, *rest;                             // [b][sq][h][dv]; rest: what the rounding of out to bf16 left behind, or null
  float2* stats;                             // [b*h][sq] {max of scale2 * score, 1 / sum} or null
  float* part;                               // [splits][b*h][sq][dv] when the keys are split
  float2* part_ml;                           // [splits][b*h][sq]
  int tiles_q, splits, span;                 // span: key tiles of one split
};

// values n .. n + 3 of an output row, `left` of which exist
template <typename T>
__device__ __forceinline__ void attn_put(const FwdArgs<T>& a, long long at, vx_f32x4 v, int left) {
  vx_store4(a.out + at, v, left);
  if constexpr (sizeof(T) == 2) {
    if (!a.rest) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] -= (float)(T)v[i];
    vx_store4(a.rest + at, v, left);
  }
}

template <typename T>
struct AttnTile {
  static constexpr int KT = VxType<T>::BK;   // keys per staged tile
};

// bits: which keys of tile t take part (lane l < KT speaks for key t * KT + l)
template <typename T>
__device__ __forceinline__ bool attn_key_live(int keys, const uint8_t* mask, int t, int lane) {
  const int key = t * AttnTile<T>::KT + lane;
  return lane < AttnTile<T>::KT && key < keys && (mask == nullptr || mask[key] != 0);
}

// A workgroup owns 16 * RT * QG queries of one head: QG groups of 16 * RT, each with CS waves. Everything is kept transposed --
// S^T = K Q^T, O^T = V^T P^T -- so that a lane holds ONE query per block (c = lane & 15) and the softmax statistics, the
// rescaling and the operand form of P are lane-local. A lane's S values are keys {16 t + 4 g + i}; as an operand they are the
// eight k's of its group g in the order (t, i), and the V^T image is staged in that order of keys.
// CS = 2 (wide heads): the two waves of a group hold one half of the output columns each, compute the scores of one half of a
// tile's keys each, and swap them through LDS as they are (a lane reads what the same lane of the other wave wrote).
// A tile: V(t) travels under S(t), K(t + 1) under O += P V(t); each LDS image is rewritten only after the barrier behind its last
// reader. IMG: both come as finished images (attn_pack) and go straight to LDS; else (few queries) through registers, where
// they are split and V is transposed.
// Two heads of 192 / 384, 65 % of the keys live: 4 x 1600 x 480 fp32 46 us (200 workgroups on 256 CUs; 100 TFLOP/s of the live keys; without
// a mask 63 us, 113), 25600 x 1920 bf16 182 us (405; 143 us with P in one plane), fp32 467 us (158); 8 heads of 48, 2 x 2037 x 2037
// bf16 47 us. No pipe is full: counters say matrix pipe, vector pipe and LDS busy 11, 8 and 6 of 48 us, 50, 52 and 23 of 182, 180, 74
// and 92 of 491, 10, 21 and 8 of 48; waves wait 33 to 48 % of their cycles, at the two barriers a tile and for what the next one loads.
template <typename T, int DP, int DVP, int RT, int QG, int CS, bool IMG, bool FAST>
__global__ __launch_bounds__(64 * QG * CS, QG * CS == 8 ? 2 : DVP > 192 || (DVP > 64 && VxType<T>::NPL == 3) ? 1 : 2)
void attn_fwd(const FwdArgs<T> a) {
  constexpr int NPL = VxType<T>::NPL, PP = VxType<T>::NPL_F32, KT = AttnTile<T>::KT, NS = KT / 32;     // NS: 32-key steps of a tile
  constexpr int KD = DP / 32, NV = DVP / 16 / CS, NK = KT / 16, OWN = NK / CS, E = sizeof(T), NW = QG * CS;
  constexpr int K_FRAGS = NK * KD;
  constexpr int K_BLOCK = IMG ? KD * kFragBytes : vx_image_block<KD>(), V_BLOCK = IMG ? NS * kFragBytes : vx_image_block<NS>();
  constexpr int K_PLANE = NK * K_BLOCK, V_PLANE = DVP / 16 * V_BLOCK;
  constexpr int KI = (K_FRAGS + NW - 1) / NW;                                  // K fragments staged per wave
  constexpr int CB = DVP % 128 == 0 ? 128 : 64, VW = E == 2 ? CB / 32 : CB / 64;   // columns of a staged block and of a lane
  constexpr int LR = CB / VW, LG = 64 / LR;                                    // lanes of a row, key groups of a wave
  constexpr int V_UNITS = DVP / CB * (KT / 8) / LG, VI = (V_UNITS + NW - 1) / NW;
  constexpr int SWAP = CS == 2 ? NW * OWN * RT * kFragBytes : 0;
  __shared__ __attribute__((aligned(16))) char lds[(K_PLANE + V_PLANE) * NPL + SWAP];
  char *ik = lds, *iv = lds + K_PLANE * NPL, *swap = iv + V_PLANE * NPL;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int half = wave % CS;
  unsigned w = vx_xcd_tile(blockIdx.x, gridDim.x);
  const int tile_q = (int)(w % a.tiles_q);
  w /= a.tiles_q;
  const int split = (int)(w % a.splits);
  const int bh = (int)(w / a.splits), b = bh / a.h, h = bh % a.h;
  const int tiles_k = (a.sk + KT - 1) / KT;                                    // of the images
  const int keys = IMG && a.count ? a.count[b] : a.sk, tiles = (keys + KT - 1) / KT;
  const int t0 = split * a.span, t1 = t0 + a.span < tiles ? t0 + a.span : tiles;
  const T* kp = a.k + b * a.k_b + (h / a.gk) * a.k_h;
  const T* vp = a.v + b * a.v_b + (h / a.gv) * a.v_h;
  const uint8_t* mask = !IMG && a.mask ? a.mask + b * a.mask_b : nullptr;
  const int q0 = (tile_q * QG + wave / CS) * (16 * RT);

  VxFrag<NPL> qf[RT][KD];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = q0 + rt * 16 + c;
    const T* qp = a.q + b * a.q_b + q0 * a.q_s + h * a.q_h;
#pragma unroll
    for (int kd = 0; kd < KD; ++kd) {
      VxRow8<T> x;
      const int d = kd * 32 + g * 8;
      if constexpr (FAST)
        x.load(vx_buffer(qp), row < a.sq && d < a.d ? (rt * 16 + c) * (int)a.q_s * E + d * E : kVxOut);
      else
        x.load(qp + (rt * 16 + c) * a.q_s + d, row < a.sq ? a.d - d : 0);
      x.planes(qf[rt][kd]);
      if (a.sign != 1.0f) {                    // exact: -1 and 0 times the planes
#pragma unroll
        for (int i = 0; i < NPL; ++i) qf[rt][kd].p[i] = a.sign == 0.0f ? bf16x8{} : -qf[rt][kd].p[i];
      }
    }
  }
  float m[RT], l[RT];                          // reference of the exponents (log2), sum of this lane's keys
  vx_f32x4 o[RT][NV];
  vx_acc_zero(o);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.0f;
  }

  // fragment (key block, k step) i of a wave: lane offsets are loop constants, the rest of an address is wave-uniform
  const int k_lane = c * (int)a.k_s * E + g * 8 * E;
  auto load_k = [&](VxRow8<T> (&ks)[KI], int t) {
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int frag = i * NW + wave, kt = frag / KD, kd = frag % KD;
      const bool here = frag < K_FRAGS && t * KT + kt * 16 + c < a.sk && kd * 32 + g * 8 < a.d;
      const T* base = kp + (t * KT + kt * 16) * a.k_s + kd * 32;
      if constexpr (FAST)
        ks[i].load(vx_buffer(base), here ? k_lane : kVxOut);
      else
        ks[i].load(base + c * a.k_s + g * 8, here ? a.d - kd * 32 - g * 8 : 0);
    }
  };
  auto store_k = [&](const VxRow8<T> (&ks)[KI]) {
    VxFrag<NPL> f;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int frag = i * NW + wave;
      if (K_FRAGS % NW == 0 || frag < K_FRAGS) {
        ks[i].planes(f);
        vx_frag_store(ik + vx_image_at<KD>(frag / KD, frag % KD, lane), K_PLANE, f);
      }
    }
  };
  // V unit i of a wave: a block of CB columns and LG key groups of eight (operand order of the keys, see above)
  const int vl = lane % LR * VW, vg = lane / LR;
  const int v_lane = vg * 4 * (int)a.v_s * E + vl * E;
  auto load_v = [&](VxCol8<T, VW> (&vs)[VI], int t, unsigned long long live) {
    const unsigned long long bits = live >> (vg * 4);
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int u = i * NW + wave, nb = u % (DVP / CB) * CB, kg = u / (DVP / CB) * LG;
      const int at = u < V_UNITS && nb + vl < a.dv ? v_lane : kVxOut;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int kk = kg / 4 * 32 + (j >> 2) * 16 + kg % 4 * 4 + (j & 3);
        const bool here = bits >> kk & 1;
        const T* base = vp + (t * KT + kk) * a.v_s + nb;
        if constexpr (FAST)
          vs[i].load(j, vx_buffer(base), here ? at : kVxOut);
        else
          vs[i].load(j, base + vg * 4 * a.v_s + vl, here && u < V_UNITS ? a.dv - nb - vl : 0);
      }
    }
  };
  auto store_v = [&](const VxCol8<T, VW> (&vs)[VI]) {
    VxFrag<NPL> f;
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int u = i * NW + wave, nb = u % (DVP / CB) * CB, kg = u / (DVP / CB) * LG;
      if (V_UNITS % NW != 0 && u >= V_UNITS) continue;
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        vs[i].planes(j, f);
        vx_frag_store(iv + nb / 16 * vx_image_block<NS>() + vx_image_at<NS>((vl + j) >> 4, kg / 4, ((vl + j) & 15) + 16 * (kg % 4 + vg)),
                      V_PLANE, f);
      }
    }
  };
  // IMG: whole fragments, in the order of the images
  auto copy = [&](const char* from, char* to, int frags) {
#pragma unroll
    for (int i = wave; i < frags; i += NW) vx_copy_frag(from + i * kFragBytes, to + i * kFragBytes, lane);
  };
  const long long k_head = IMG ? ((long long)b * (a.h / a.gk) + h / a.gk) * tiles_k : 0;
  const long long v_head = IMG ? ((long long)b * (a.h / a.gv) + h / a.gv) * tiles_k : 0;
  const char *k_img = a.k_img + k_head * (K_PLANE * NPL), *v_img = a.v_img + v_head * (V_PLANE * NPL);
  auto frag_at = [&](int block, int rb, int ks) {
    return rb * block + ks * kFragBytes + (IMG ? lane : lane ^ (lane >> 4) ^ (ks & 1) << 2) * 16;
  };
  // the first tile from t on that has a key that takes part, and which of its keys do
  auto find = [&](int t, unsigned long long& live) {
    for (live = 0; t < t1; ++t) {
      live = __ballot(attn_key_live<T>(keys, mask, t, lane));
      if (live) break;
    }
    return t;
  };

  unsigned long long cur, nxt = 0;
  int t = find(t0, cur), tn = t1;
  const bool any = cur != 0;                   // this workgroup has keys
  if (cur) {
    tn = find(t + 1, nxt);
    if constexpr (IMG) {
      copy(k_img + (long long)t * (K_PLANE * NPL), ik, K_PLANE * NPL / kFragBytes);
      vx_arrived();
    } else {
      VxRow8<T> ks[KI];
      load_k(ks, t);
      store_k(ks);
    }
  }
  __syncthreads();
  while (cur) {
    const bool ahead = tn + 1 < t1 && attn_key_live<T>(keys, mask, tn + 1, lane);
    vx_f32x4 s[RT][NK];
    {
      VxCol8<T, VW> vs[VI];
      if constexpr (IMG)
        copy(v_img + (long long)t * (V_PLANE * NPL), iv, V_PLANE * NPL / kFragBytes);
      else
        load_v(vs, t, cur);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int k = 0; k < OWN; ++k) s[rt][k] = vx_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) {
        VxFrag<NPL> kf[OWN];
#pragma unroll
        for (int k = 0; k < OWN; ++k) vx_frag_load(ik + frag_at(K_BLOCK, half * OWN + k, kd), K_PLANE, kf[k]);
#pragma unroll
        for (int pr = 0; pr < VxProducts<NPL, NPL>::N; ++pr)
#pragma unroll
          for (int k = 0; k < OWN; ++k)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][k] = vx_mma(pr, kf[k], qf[rt][kd], s[rt][k]);
        if constexpr (DVP > 128) __builtin_amdgcn_sched_barrier(0);   // keeps later fragment reads out of the registers
      }
      if constexpr (CS == 2) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int k = 0; k < OWN; ++k)
            *reinterpret_cast<vx_f32x4*>(swap + (wave * OWN * RT + rt * OWN + k) * kFragBytes + lane * 16) = s[rt][k];
      }
      if constexpr (IMG) vx_arrived(); else store_v(vs);
    }
    __syncthreads();
    VxRow8<T> ks[KI];
    if (nxt) {
      if constexpr (IMG)
        copy(k_img + (long long)tn * (K_PLANE * NPL), ik, K_PLANE * NPL / kFragBytes);
      else
        load_k(ks, tn);
    }
    if constexpr (CS == 2) {                   // both halves, in the order of the keys
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int k = 0; k < NK; ++k)
          s[rt][k] = *reinterpret_cast<const vx_f32x4*>(swap + (((wave & ~1) + k / OWN) * OWN * RT + rt * OWN + k % OWN) * kFragBytes +
                                                        lane * 16);
    }
    VxFrag<PP> pf[RT][NS];
    if (cur != ~0ull >> (64 - KT)) {           // some keys take no part
      const unsigned long long bits = cur >> (g * 4);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[rt][k][i] = bits >> (k * 16 + i) & 1 ? s[rt][k][i] : -INFINITY;
    }
    float alpha[RT];
    bool moved = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][k][i]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale2;   // the maximum of the scaled scores
      // the reference follows the maximum only when it is 2^8 behind: values stay below 2^8, far from any limit of fp32, and the
      // accumulators are hardly ever rescaled
      const bool far = mx > m[rt] + 8.0f;
      alpha[rt] = far ? __builtin_amdgcn_exp2f(m[rt] - mx) : 1.0f;
      m[rt] = far ? mx : m[rt];
      moved |= far;
      const float ref = m[rt] == -INFINITY ? 0.0f : m[rt];
      float sum = 0.0f;
#pragma unroll
      for (int ns = 0; ns < NS; ++ns) {
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][ns * 2 + (j >> 2)][j & 3], a.scale2, -ref));
          sum += p[j];
        }
        vx_planes(p, pf[rt][ns]);
      }
      l[rt] = l[rt] * alpha[rt] + sum;
    }
    if (__any(moved)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int nv = 0; nv < NV; ++nv) o[rt][nv] *= alpha[rt];
    }
    constexpr int G = 2;                       // column blocks at a time: independent accumulators
#pragma unroll
    for (int nv = 0; nv < NV; nv += G) {
#pragma unroll
      for (int ns = 0; ns < NS; ++ns) {
        VxFrag<NPL> vf[G];
#pragma unroll
        for (int u = 0; u < G; ++u) vx_frag_load(iv + frag_at(V_BLOCK, half * NV + nv + u, ns), V_PLANE, vf[u]);
#pragma unroll
        for (int pr = 0; pr < VxProducts<NPL, PP>::N; ++pr)
#pragma unroll
          for (int u = 0; u < G; ++u)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) o[rt][nv + u] = vx_mma(pr, vf[u], pf[rt][ns], o[rt][nv + u]);
      }
      if (nv % 4 == 2) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (IMG)
      vx_arrived();
    else if (nxt)
      store_k(ks);
    __syncthreads();
    t = tn;
    cur = nxt;
    tn = tn + 1;
    nxt = __ballot(ahead);
    if (cur && !nxt) tn = find(tn + 1, nxt);
  }

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float sum = l[rt];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    const int row = q0 + rt * 16 + c;
    if (row >= a.sq) continue;
    const int n0 = half * NV * 16 + g * 4;
    if (a.splits > 1) {
      const long long at = ((long long)split * gridDim.x / (a.tiles_q * a.splits) + bh) * a.sq + row;
      // keys whose scores are all -inf count as keys: attn_join tells them from none by the maximum
      if (g == 0 && half == 0) a.part_ml[at] = make_float2(any && m[rt] == -INFINITY ? -FLT_MAX : m[rt], sum);
#pragma unroll
      for (int nv = 0; nv < NV; ++nv) vx_store4(a.part + at * a.dv + n0 + nv * 16, o[rt][nv], a.dv - n0 - nv * 16);
    } else {
      const float inv = any ? 1.0f / sum : 0.0f;         // a sum of 0 over keys: every score left the range, 0 / 0 = NaN
      if (a.stats && g == 0 && half == 0) a.stats[(long long)bh * a.sq + row] = make_float2(m[rt], inv);
      const long long at = (((long long)b * a.sq + row) * a.h + h) * a.dv + n0;
#pragma unroll
      for (int nv = 0; nv < NV; ++nv) attn_put(a, at + nv * 16, o[rt][nv] * inv, a.dv - n0 - nv * 16);
    }
  }
}

// Which keys take part, once per call: index[b][j] = the j-th of them, place[b][key] = its j or -1, count[b]. Everything behind
// works on the keys that take part alone, in their order, so a masked key costs nothing. One workgroup per batch, four keys a
// thread and sweep.
struct LiveArgs {
  const uint8_t* mask;
  long long mask_b;
  int sk;
  int *index, *place, *count;
};
// the whole workgroup (256 threads); GLOBAL: writes the lists; local (if not null): the keys in their order; returns the count
template <bool GLOBAL>
__device__ __forceinline__ int live_keys(const LiveArgs& a, int b, int* local) {
  __shared__ int sums[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint8_t* mask = a.mask + b * a.mask_b;
  int base = 0;
  for (int k0 = 0; k0 < a.sk; k0 += 1024) {
    const int key = k0 + threadIdx.x * 4;
    int live = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) live |= key + i < a.sk && mask[key + i] != 0 ? 1 << i : 0;
    int upto = __popc(live);                   // inclusive sum over the wave's lanes
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(upto, d, 64);
      if (lane >= d) upto += v;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int j = base + upto - __popc(live), all = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < wave) j += sums[i];
      all += sums[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool on = live >> i & 1;
      if (local && on) local[j] = key + i;
      if constexpr (GLOBAL) {
        if (on) a.index[(long long)b * a.sk + j] = key + i;
        if (key + i < a.sk) a.place[(long long)b * a.sk + key + i] = on ? j : -1;
      }
      j += on;
    }
    base += all;
    __syncthreads();
  }
  return base;
}
__device__ __forceinline__ void live_lists(const LiveArgs& a, int b) {
  const int n = live_keys<true>(a, b, nullptr);
  if (threadIdx.x == 0) a.count[b] = n;
}
__global__ __launch_bounds__(256) void attn_live(const LiveArgs a) { live_lists(a, blockIdx.x); }

// K and V as operand images: per head and tile of KT keys, planes of 1 KB fragments -- K: key block, 32-d step; V^T: column block,
// 32-key step in the operand order of the keys. A thread makes one lane's 16 bytes of a fragment (all planes). Widths are padded
// with 0 to the tile's, keys behind the last are 0. It costs one pass over k and v; each tile of queries then saves the split
// and the transposition. 4 x 480 keys, (2 x 192 + 384) wide, fp32: 8.6 us, bound by V's column reads; 1920 keys bf16 8.7 us.
// OWN: with a mask of at most kOwnKeys keys every workgroup finds the keys by itself, which saves the launch of attn_live.
constexpr int kOwnKeys = 2048;
template <typename T, bool OWN>
__global__ __launch_bounds__(256) void attn_pack(const AttnArgs<T> a, const LiveArgs own, char* __restrict__ k_img, char* __restrict__ v_img,
                                                 int tiles, int kd, int nv, long long k_slots, long long slots, unsigned per) {
  constexpr int NPL = VxType<T>::NPL, KT = AttnTile<T>::KT, NS = KT / 32, NK = KT / 16;
  __shared__ int list[OWN ? kOwnKeys : 1];
  const int b = blockIdx.x / per;              // `per` workgroups a batch
  const unsigned block = blockIdx.x % per;
  int keys = a.sk;
  const int* index = nullptr;
  if constexpr (OWN) {
    keys = live_keys<false>(own, b, list);
    index = list;
    if (block == 0 && threadIdx.x == 0) own.count[b] = keys;
  } else if (a.count) {
    keys = a.count[b];
    index = a.index + (long long)b * a.sk;
  }
  long long i = (long long)block * 256 + threadIdx.x;
  if (i >= slots) return;
  const bool is_k = i < k_slots;
  if (!is_k) i -= k_slots;
  const int lane = (int)(i & 63), c = lane & 15, g = lane >> 4;
  const int frags = is_k ? NK * kd : nv * NS, heads = is_k ? a.h / a.gk : a.h / a.gv;
  const long long ft = i >> 6, ht = ft / frags;
  const int frag = (int)(ft % frags), t = (int)(ht % tiles), head = (int)(ht / tiles);
  const long long tile_id = (long long)b * heads * tiles + ht;
  if (t * KT >= keys) return;                  // no query reads this tile
  VxFrag<NPL> f;
  if (is_k) {
    const int key = t * KT + frag / kd * 16 + c, d = frag % kd * 32 + g * 8;
    const bool live = key < keys;
    const int row = index && live ? index[key] : key;
    VxRow8<T> x;
    x.load(a.k + b * a.k_b + head * a.k_h + row * a.k_s + d, live ? a.d - d : 0);
    x.planes(f);
  } else {
    const int n = frag / NS * 16 + c, k0 = t * KT + frag % NS * 32 + g * 4;
    const T* p = a.v + b * a.v_b + head * a.v_h + (n < a.dv ? n : 0);
    float x[8];
    int row[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = k0 + (j >> 2) * 16 + (j & 3), last = keys - 1;
      row[j] = key < last ? key : last;
      if (index) row[j] = index[row[j]];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = (float)p[row[j] * a.v_s];
      x[j] = k0 + (j >> 2) * 16 + (j & 3) < keys && n < a.dv ? y : 0.0f;
    }
    vx_planes(x, f);
  }
  char* to = (is_k ? k_img : v_img) + tile_id * frags * (NPL * kFragBytes) + frag * kFragBytes + lane * 16;
#pragma unroll
  for (int q = 0; q < NPL; ++q) *reinterpret_cast<bf16x8*>(to + (long long)q * frags * kFragBytes) = f.p[q];
}

// joins the splits of a row: weights 2^(m_s - m). A workgroup has 256 / J quads of output values, J lanes each: lane j adds the
// splits j, j + J, ..., four of them in flight (few rows: what counts is latency), then the J sums are added in order. 2 rows of 15
// splits of 384: 4.0 us, of which the launch is most.
template <typename T, int J>
__global__ __launch_bounds__(256) void attn_join(const FwdArgs<T> a, long long items, int quads) {
  constexpr int U = 4, Q = 256 / J;
  __shared__ vx_f32x4 sh_o[J][Q];
  __shared__ float sh_l[J][Q];
  const int lane = threadIdx.x % Q, j = threadIdx.x / Q;
  const long long it = (long long)blockIdx.x * Q + lane;
  const bool here = it < items;
  const long long rowid = here ? it / quads : 0, rows = items / quads;      // bh * sq + row
  const int n = here ? (int)(it % quads) * 4 : 0, last = a.splits - 1;
  float m = -INFINITY;
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = a.part_ml[(s0 + u < last ? s0 + u : last) * rows + rowid].x;
#pragma unroll
    for (int u = 0; u < 8; ++u) m = fmaxf(m, x[u]);
  }
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  vx_f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = j; s0 < a.splits; s0 += U * J) {
    float2 ml[U];
    vx_f32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long at = (s0 + u * J < last ? s0 + u * J : last) * rows + rowid;
      ml[u] = a.part_ml[at];
      v[u] = vx_load4(a.part + at * a.dv + n, a.dv - n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * J > last) break;
      const float wgt = __builtin_amdgcn_exp2f(ml[u].x - ref);
      l += wgt * ml[u].y;
      o += v[u] * wgt;
    }
  }
  if constexpr (J > 1) {
    sh_o[j][lane] = o;
    sh_l[j][lane] = l;
    __syncthreads();
    if (j) return;
#pragma unroll
    for (int i = 1; i < J; ++i) {
      l += sh_l[i][lane];
      o += sh_o[i][lane];
    }
  }
  if (!here) return;
  const float inv = m == -INFINITY ? 0.0f : 1.0f / l;    // no keys in any split
  const int bh = (int)(rowid / a.sq), row = (int)(rowid % a.sq), b = bh / a.h, h = bh % a.h;
  attn_put(a, (((long long)b * a.sq + row) * a.h + h) * a.dv + n, o * inv, a.dv - n);
  if (a.stats && n == 0) a.stats[rowid] = make_float2(m, inv);
}

// ---- backward -------------------------------------------------------------------------------------------------------
template <typename T>
struct BwdArgs : AttnArgs<T> {
  const T *out, *rest, *go;                  // out [b][sq][h][dv] and its rest or null; go by strides
  long long go_b, go_s, go_h;
  const float2* stats;
  float* delta;                              // [b*h][sq]
  float *p, *ds;                             // [b*h][rows][skp] of the present chunk of queries
  T *dq, *dk, *dvv;                          // [b][sq][h][d], [b][sk][h/gk][d], [b][sk][h/gv][dv]; null: not wanted
  float *slab_k, *slab_v;                    // [splits][b*h][sk][d], [splits][b*h][sk][dv]
  float scale;
  int q0, rows, skp;                         // present chunk: queries [q0, q0 + rows); skp: sk rounded up to 8
  long long kc_b, kc_h, vc_b, vc_h;          // gathered k, v: [b][head][sk][d], [b][head][sk][dv]
  T *kc, *vc;
  int bh, span;                              // queries of one split
  bool add;                                  // a later chunk: the slabs hold the sums of the earlier ones
  int tqp, tkp;                              // tiles of attn_pds: queries, keys
  int tq, tk, td, tdv;                       // tiles of attn_grads: queries, keys, columns of dK and dQ, columns of dV
  unsigned n_v, n_k, n_q;                    // workgroups per problem
};

// k and v of the keys that take part, in their order: piece i (16 bytes where the rows allow it) of batch b. Behind this the GEMMs read
// plain rows. A copy, bound by its launch at the usual sizes (480 keys, 4 x (2 x 192 + 384) fp32: 5 us); four pieces a thread are
// no faster
struct GatherArgs {
  int pieces_k, pieces_v;                      // of a row
  long long items_k, items;                    // of a batch: k, k and v
  unsigned per;                                // workgroups a batch
};
template <typename T>
__device__ __forceinline__ void gather_piece(const BwdArgs<T>& a, const GatherArgs& g, int b, long long i, int keys, const int* index) {
  constexpr int P = 16 / sizeof(T);
  if (i >= g.items) return;
  const bool is_k = i < g.items_k;
  if (!is_k) i -= g.items_k;
  const int pieces = is_k ? g.pieces_k : g.pieces_v, width = is_k ? a.d : a.dv;
  const int n = (int)(i % pieces) * P;
  i /= pieces;
  const int j = (int)(i % a.sk), head = (int)(i / a.sk);
  if (j >= keys) return;
  const int key = index[j];
  const T* from = (is_k ? a.k + b * a.k_b + key * a.k_s + head * a.k_h : a.v + b * a.v_b + key * a.v_s + head * a.v_h) + n;
  T* to = (is_k ? a.kc + b * a.kc_b + head * a.kc_h : a.vc + b * a.vc_b + head * a.vc_h) + (long long)j * width + n;
  if (width - n >= P) {
    vx_u32x4u v;
    __builtin_memcpy(&v, from, 16);
    __builtin_memcpy(to, &v, 16);
  } else {
    for (int e = 0; e < width - n; ++e) to[e] = from[e];
  }
}
template <typename T>
__global__ __launch_bounds__(256) void attn_gather(const BwdArgs<T> a, const GatherArgs g) {
  const int b = blockIdx.x / g.per;
  gather_piece(a, g, b, (long long)(blockIdx.x % g.per) * 256 + threadIdx.x, a.count[b], a.index + (long long)b * a.sk);
}

// delta = sum_n go * out per query, out with its rest: a row that one key dominates has dP of that key next to delta, and a bf16 out alone
// would leave 3 times the gradients' own rounding (scores of 200 to 1000 keys with standard deviation 8). One wave per row, more rows a
// wave past 2^22 of them. With a mask the first `head` workgroups make its lists; OWN (at most kOwnKeys keys):
// they gather the keys as well, each with a list of its own, which saves a launch (a step of 4 x 1600 x 480, 2 heads of 192 / 384, fp32:
// 187 -> 182 us). One read of go and out (and rest): 4 x 2 x 1600 x 384 fp32 39 MB 11 us with the gather, 2 x 25600 x 384 157 MB 29 us,
// bf16 118 MB 35 us
template <typename T, bool OWN>
__global__ __launch_bounds__(256) void attn_delta(const BwdArgs<T> a, long long rows, const LiveArgs live, const GatherArgs gather,
                                                  unsigned head) {
  __shared__ int list[OWN ? kOwnKeys : 1];
  if (blockIdx.x < head) {
    if constexpr (OWN) {
      const int b = blockIdx.x / gather.per;
      const unsigned block = blockIdx.x % gather.per;
      const int keys = block ? live_keys<false>(live, b, list) : live_keys<true>(live, b, list);
      if (block == 0 && threadIdx.x == 0) live.count[b] = keys;
      gather_piece(a, gather, b, (long long)block * 256 + threadIdx.x, keys, list);
    } else {
      live_lists(live, blockIdx.x);
    }
    return;
  }
  const int lane = threadIdx.x & 63;
  for (long long r = (long long)(blockIdx.x - head) * 4 + (threadIdx.x >> 6); r < rows; r += (long long)(gridDim.x - head) * 4) {
    const int bh = (int)(r / a.sq), row = (int)(r % a.sq), b = bh / a.h, h = bh % a.h;
    const T* go = a.go + b * a.go_b + row * a.go_s + h * a.go_h;
    const long long o = (((long long)b * a.sq + row) * a.h + h) * a.dv;
    float s = 0.0f;
    for (int n = lane * 4; n < a.dv; n += 256) {
      vx_f32x4 y = vx_load4(a.out + o + n, a.dv - n);
      if (sizeof(T) == 2 && a.rest) y += vx_load4(a.rest + o + n, a.dv - n);
      const vx_f32x4 x = vx_load4(go + n, a.dv - n) * y;
      s += (x[0] + x[1]) + (x[2] + x[3]);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d, 64);
    if (lane == 0) a.delta[r] = s;
  }
}

constexpr int kPdsN = 128;                   // keys of an attn_pds tile
// P and dS of a TM-query x TN-key tile: scores and dP = go v^T are two products with one epilogue,
// P = 2^(scale2 s - max) / sum, dS = scale P (dP - delta).
// Both go out in fp32: rounded to bf16 they would make the error of dq and dk 1.4 times that of their own rounding (3 x 777 x 301).
// ONE: all keys are in the tile. delta is then the tile's own sum of P dP: over few keys the rounding of a bf16 output inside delta would
// not average out (terms that nearly cancel): relative 2-norm of dq and dk over 16 keys 0.0020 so, 0.0017 their own rounding.
// 4 x 2 x 1600 x 480, 192 / 384, fp32 57 us, 25600 x 1920 487 us: matrix pipe 14 and 180 of it, vector pipe (split into planes) 13 and 162,
// LDS 7 and 90, one after the other behind two barriers a step. bf16 25600 x 1920 209 us, of which the writes of P and dS (0.5 GB) are
// half; 3 x 4 x 777 x 301, 96 / 192 12.0 us, where 468 workgroups of 64 x 128 are two rounds.
template <typename T, int TM, int TN, bool FAST, bool ONE>
__global__ __launch_bounds__(kTileThreads, 2) void attn_pds(const BwdArgs<T> a) {
  constexpr int BK = TM <= 64 ? 64 : VxType<T>::BK;
  __shared__ __attribute__((aligned(16))) char lds[vx_gemm_lds<T, TM, TN, BK>()];
  unsigned w = vx_xcd_tile(blockIdx.x, gridDim.x);
  const int n0 = (int)(w % a.tkp) * TN;
  w /= a.tkp;
  const int m0 = (int)(w % a.tqp) * TM;
  const int bh = (int)(w / a.tqp), b = bh / a.h, h = bh % a.h;
  const int keys = a.count ? a.count[b] : a.sk;
  if (n0 >= keys) return;
  const int rows_m = a.rows - m0 < TM ? a.rows - m0 : TM, rows_n = keys - n0 < TN ? keys - n0 : TN;
  const long long q = a.q0 + m0;
  vx_f32x4 s[TM / 32][TN / 32], dp[TM / 32][TN / 32];
  vx_acc_zero(s);
  vx_acc_zero(dp);
  vx_gemm_loop<T, KC, KC, TM, TN, FAST, BK>({a.q + b * a.q_b + q * a.q_s + h * a.q_h, a.q_s, rows_m},
                                  {a.k + b * a.k_b + (h / a.gk) * a.k_h + n0 * a.k_s, a.k_s, rows_n}, 0, a.d, lds, s);
  vx_gemm_loop<T, KC, KC, TM, TN, FAST, BK>({a.go + b * a.go_b + q * a.go_s + h * a.go_h, a.go_s, rows_m},
                                  {a.v + b * a.v_b + (h / a.gv) * a.v_h + n0 * a.v_s, a.v_s, rows_n}, 0, a.dv, lds, dp);
  unsigned live[TN / 64];                      // of this lane's eight keys
  vx_acc_each<TM, TN>(s, [&](int mi, int, int j, int n, const vx_f32x4&, const vx_f32x4&) {
    if (mi) return;
    live[j] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) live[j] |= n + i < rows_n ? 1u << i : 0u;
  });
  float2 st[TM / 32];
  float delta[TM / 32];
  vx_acc_each<TM, TN>(s, [&](int mi, int m, int j, int, const vx_f32x4&, const vx_f32x4&) {
    if (j) return;
    const long long r = (long long)bh * a.sq + a.q0 + m0 + (m < rows_m ? m : 0);
    st[mi] = a.stats[r];
    delta[mi] = ONE ? 0.0f : a.delta[r];
  });
  const long long at0 = ((long long)bh * a.rows + m0) * a.skp + n0;
#pragma unroll
  for (int mi = 0; mi < TM / 32; ++mi)
#pragma unroll
    for (int ni = 0; ni < TN / 32; ++ni)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool on = live[ni / 2] >> (ni % 2 * 4 + i) & 1;
        s[mi][ni][i] = on ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[mi][ni][i] * a.sign, a.scale2, -st[mi].x)) * st[mi].y : 0.0f;
        dp[mi][ni][i] = on ? dp[mi][ni][i] : 0.0f;
        if constexpr (ONE) delta[mi] = __builtin_fmaf(s[mi][ni][i], dp[mi][ni][i], delta[mi]);
      }
  if constexpr (ONE) {                         // over the lane groups, then over the two waves of a row
    float* sh = reinterpret_cast<float*>(lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int mi = 0; mi < TM / 32; ++mi) {
      delta[mi] += __shfl_xor(delta[mi], 16, 64);
      delta[mi] += __shfl_xor(delta[mi], 32, 64);
      if (lane < 16) sh[(wave * (TM / 32) + mi) * 16 + lane] = delta[mi];
    }
    __syncthreads();
#pragma unroll
    for (int mi = 0; mi < TM / 32; ++mi)
      delta[mi] = sh[((wave & 2) * (TM / 32) + mi) * 16 + (lane & 15)] + sh[((wave | 1) * (TM / 32) + mi) * 16 + (lane & 15)];
  }
#pragma unroll
  for (int mi = 0; mi < TM / 32; ++mi)
#pragma unroll
    for (int ni = 0; ni < TN / 32; ++ni)
#pragma unroll
      for (int i = 0; i < 4; ++i) dp[mi][ni][i] = s[mi][ni][i] * (dp[mi][ni][i] - delta[mi]) * a.scale;
  vx_acc_each<TM, TN>(s, [&](int mi, int m, int j, int n, const vx_f32x4& v, const vx_f32x4& w) {
    if (m >= rows_m || n0 + n >= a.skp) return;
    const long long at = at0 + (long long)m * a.skp + n;
    vx_store8(a.p + at, v, w, 8);
    vx_store8(a.ds + at, dp[mi][2 * j], dp[mi][2 * j + 1], 8);
  });
}

// the three gradients of a chunk in one launch: dV slabs = P^T go, dK slabs = dS^T q (reduction over the queries of a split),
// dQ = dS k (reduction over the keys)
// P and dS are fp32; beside bf16 operands they are two planes
// 4 x 2 x 1600 x 480, 192 / 384 fp32 66 us, 25600 x 1920 567 us: as attn_pds (matrix pipe 15 and 240 of it, vector pipe 14 and 155, LDS 14
// and 150, a third of that bank conflicts); dV and dK read both operands along their rows, transposed on the way to LDS. bf16 25600 x
// 1920 265 us, 3 x 4 x 777 x 301, 96 / 192 15.6 us
template <typename T, int TM, int TN, bool FAST>
__global__ __launch_bounds__(kTileThreads, 2) void attn_grads(const BwdArgs<T> a) {
  constexpr int BK = VxType<T>::BK, PX = VxType<T>::NPL_F32;
  __shared__ __attribute__((aligned(16))) char lds[vx_gemm_lds<T, TM, TN, BK, PX>()];
  vx_f32x4 acc[TM / 32][TN / 32];
  vx_acc_zero(acc);
  if (blockIdx.x < a.n_v + a.n_k) {
    const bool is_v = blockIdx.x < a.n_v;
    const int tn = is_v ? a.tdv : a.td, width = is_v ? a.dv : a.d;
    unsigned w = is_v ? vx_xcd_tile(blockIdx.x, a.n_v) : vx_xcd_tile(blockIdx.x - a.n_v, a.n_k);
    const int n0 = (int)(w % tn) * TN;
    w /= tn;
    const int m0 = (int)(w % a.tk) * TM;
    w /= a.tk;
    const int bh = (int)(w % a.bh), sp = (int)(w / a.bh), b = bh / a.h, h = bh % a.h;
    const int keys = a.count ? a.count[b] : a.sk;
    if (m0 >= keys) return;
    const int r0 = sp * a.span, len = a.rows - r0 < a.span ? a.rows - r0 : a.span;
    const int rows_m = keys - m0 < TM ? keys - m0 : TM, rows_n = width - n0 < TN ? width - n0 : TN;
    const long long q = a.q0 + r0;
    const VxOperand<float> X{(is_v ? a.p : a.ds) + ((long long)bh * a.rows + r0) * a.skp + m0, a.skp, a.skp - m0};
    const VxOperand<T> W{is_v ? a.go + b * a.go_b + q * a.go_s + h * a.go_h + n0 : a.q + b * a.q_b + q * a.q_s + h * a.q_h + n0,
                         is_v ? a.go_s : a.q_s, rows_n};
    vx_gemm_loop<T, KS, KS, TM, TN, FAST, BK, float, PX>(X, W, 0, len, lds, acc);
    float* slab = (is_v ? a.slab_v : a.slab_k) + ((long long)sp * a.bh + bh) * a.sk * width;
    vx_acc_each<TM, TN>(acc, [&](int, int m, int, int n, vx_f32x4 v, vx_f32x4 w) {
      if (m >= rows_m || n >= rows_n) return;
      float* at = slab + (long long)(m0 + m) * width + n0 + n;
      if (a.add) {
        v += vx_load4(at, rows_n - n);
        w += vx_load4(at + 4, rows_n - n - 4);
      }
      vx_store8(at, v, w, rows_n - n);
    });
  } else {
    unsigned w = vx_xcd_tile(blockIdx.x - a.n_v - a.n_k, a.n_q);
    const int n0 = (int)(w % a.td) * TN;
    w /= a.td;
    const int m0 = (int)(w % a.tq) * TM;
    const int bh = (int)(w / a.tq), b = bh / a.h, h = bh % a.h;
    const int rows_m = a.rows - m0 < TM ? a.rows - m0 : TM, rows_n = a.d - n0 < TN ? a.d - n0 : TN;
    const VxOperand<float> X{a.ds + ((long long)bh * a.rows + m0) * a.skp, a.skp, rows_m};
    const VxOperand<T> W{a.k + b * a.k_b + (h / a.gk) * a.k_h + n0, a.k_s, rows_n};
    const int keys = a.count ? a.count[b] : a.sk;    // dS is 0 from there to its tile's end
    vx_gemm_loop<T, KC, KS, TM, TN, FAST, BK, float, PX>(X, W, 0, keys, lds, acc);
    vx_acc_each<TM, TN>(acc, [&](int, int m, int, int n, const vx_f32x4& v, const vx_f32x4& w) {
      if (m < rows_m && n < rows_n)
        vx_store8(a.dq + (((long long)b * a.sq + a.q0 + m0 + m) * a.h + h) * a.d + n0 + n, v, w, rows_n - n);
    });
  }
}

// dk, dv = sums of the slabs over a head's query heads and the splits, in that order; masked keys get zeros. One read of the slabs:
// 4 x 480 keys of 2 x 192 and 384, 6.5 us
template <typename T>
__global__ __launch_bounds__(256) void attn_slab_sum(const BwdArgs<T> a, int splits, unsigned blocks_v, long long items_v,
                                                     long long items_k) {
  const bool is_v = blockIdx.x < blocks_v;
  const int width = is_v ? a.dv : a.d, group = is_v ? a.gv : a.gk, quads = (width + 3) / 4;
  const long long it = (long long)(is_v ? blockIdx.x : blockIdx.x - blocks_v) * 256 + threadIdx.x;
  if (it >= (is_v ? items_v : items_k)) return;
  const int n = (int)(it % quads) * 4, left = width - n;
  long long r = it / quads;                        // (b * heads + head) * sk + key
  const int key = (int)(r % a.sk);
  r /= a.sk;
  const int heads = a.h / group, head = (int)(r % heads), b = (int)(r / heads);
  vx_f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  const int row = a.place ? a.place[(long long)b * a.sk + key] : key;
  if (row >= 0) {
    const float* slab = is_v ? a.slab_v : a.slab_k;
    constexpr int U = 8;                           // slabs in flight
    const int last = group * splits - 1;
    for (int i = 0; i <= last; i += U) {
      vx_f32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = i + u < last ? i + u : last, j = at / splits, sp = at % splits;
        v[u] = vx_load4(slab + (((long long)sp * a.bh + b * a.h + head * group + j) * a.sk + row) * width + n, left);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u > last) break;
        s += v[u];
      }
    }
  }
  vx_store4((is_v ? a.dvv : a.dk) + (((long long)b * a.sk + key) * heads + head) * width + n, s, left);
}

// ---- host -----------------------------------------------------------------------------------------------------------
struct Shape {
  int64_t b, sq, sk, h, hk, hv, d, dv;
};
Shape shape_of(const int64_t* s) { return {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]}; }

int32_t check(const char* who, const int64_t* shape, int32_t dtype) {
  VX_REQUIRE(shape, "%s: null shape", who);
  const Shape s = shape_of(shape);
  VX_REQUIRE(dtype == VX_F32 || dtype == VX_BF16, "%s: dtype must be VX_F32 or VX_BF16", who);
  VX_REQUIRE(s.b >= 0 && s.sq >= 0 && s.sk >= 0 && s.b < (1 << 24) && s.sq < (1LL << 30) && s.sk < (1LL << 30), "%s: bad lengths", who);
  VX_REQUIRE(s.h >= 1 && s.hk >= 1 && s.hv >= 1 && s.h % s.hk == 0 && s.h % s.hv == 0 && s.h < (1 << 16),
             "%s: key and value heads must divide the query heads", who);
  VX_REQUIRE(s.d >= 1 && s.d <= VX_ATTN_MAX_DIM && s.dv >= 1 && s.dv <= VX_ATTN_MAX_VDIM, "%s: dim must be in [1, %d], v_dim in [1, %d]",
             who, VX_ATTN_MAX_DIM, VX_ATTN_MAX_VDIM);
  VX_REQUIRE(s.b * s.h < (1LL << 24), "%s: too many heads", who);
  return VX_OK;
}

// strides: q, k, v (batch, position, head), mask (batch)
template <typename T>
void fill_args(AttnArgs<T>& a, const Shape& s, const int64_t* st, const void* q, const void* k, const void* v, const uint8_t* mask,
               float scale) {
  a.q = (const T*)q; a.k = (const T*)k; a.v = (const T*)v; a.mask = mask;
  a.q_b = st[0]; a.q_s = st[1]; a.q_h = st[2];
  a.k_b = st[3]; a.k_s = st[4]; a.k_h = st[5];
  a.v_b = st[6]; a.v_s = st[7]; a.v_h = st[8];
  a.mask_b = st[9];
  a.sq = (int)s.sq; a.sk = (int)s.sk; a.h = (int)s.h;
  a.gk = (int)(s.h / s.hk); a.gv = (int)(s.h / s.hv); a.d = (int)s.d; a.dv = (int)s.dv;
  a.scale2 = scale == 0.0f ? 1.0f : fabsf(scale) * kLog2e;
  a.sign = scale == 0.0f ? 0.0f : scale < 0.0f ? -1.0f : 1.0f;
}

// whether every row of a [batch, position, head, width] tensor can be read by buffer loads
bool heads_fast(const void* p, int64_t b, int64_t s, int64_t h, int64_t width, int64_t e) {
  return vx_fast(p, s, width, e) && b * e % 16 == 0 && h * e % 16 == 0;
}
template <typename T>
bool args_fast(const AttnArgs<T>& a) {
  return heads_fast(a.q, a.q_b, a.q_s, a.q_h, a.d, sizeof(T)) && heads_fast(a.k, a.k_b, a.k_s, a.k_h, a.d, sizeof(T)) &&
         heads_fast(a.v, a.v_b, a.v_s, a.v_h, a.dv, sizeof(T));
}

// the smallest tile that holds both widths
constexpr int kClasses = 6, kWideF32 = 3;
constexpr int kDims[kClasses][2] = {{32, 64}, {64, 64}, {64, 128}, {128, 128}, {96, 192}, {192, 384}};
int class_of(int64_t d, int64_t dv) {
  int i = 0;
  while (d > kDims[i][0] || dv > kDims[i][1]) ++i;
  return i;
}

// attn_live's lists
size_t live_bytes(const Shape& s) { return 2 * vx_align((size_t)s.b * s.sk * 4) + vx_align((size_t)s.b * 4); }
template <typename T>
LiveArgs live_args(AttnArgs<T>& a, const Shape& s, char* ws) {
  const size_t list = vx_align((size_t)s.b * s.sk * 4);
  const LiveArgs l{a.mask, a.mask_b, a.sk, (int*)ws, (int*)(ws + list), (int*)(ws + 2 * list)};
  a.index = l.index;
  a.place = l.place;
  a.count = l.count;
  return l;
}

struct FwdPlan {
  bool many, img;            // 128 queries per workgroup instead of 64; operand images
  int64_t tiles_q, splits, span, tiles_k;
  size_t k_img, v_img, live; // bytes
};
FwdPlan fwd_plan(const Shape& s, int32_t dtype) {
  FwdPlan p;
  const int64_t cus = vx_tile_cus(), bh = s.b * s.h, kt = dtype == VX_F32 ? 32 : 64, tiles_k = vx_cdiv(s.sk, kt);
  // 128 queries a workgroup share a staged tile, 64 fill the CUs sooner. us of 64 / 128 at 1024 keys, 8 heads, n 128-query tiles:
  // 192 / 384 wide, fp32: n = 128 125 / 180, 256 239 / 206, 2048 1887 / 1489; bf16: 63 / 75, 107 / 88, 699 / 556: a tile takes 1.45
  // times as long, so whole rounds over the CUs decide. 64 / 64, fp32: 256 70 / 76, 512 104 / 101, 2048 358 / 317; bf16: 29 / 33,
  // 43 / 41, 138 / 128: two workgroups of 64 fit a CU. 96 / 192 and 128 / 128, fp32: 128 loses everywhere (831 / 973, 746 / 845:
  // one wave a SIMD) and is not built.
  const int64_t n128 = vx_cdiv(s.sq, 128) * bh, n64 = vx_cdiv(s.sq, 64) * bh;
  const int c = class_of(s.d, s.dv);
  // images pay from about five tiles of 64 queries on; us with / without, 480 and 4096 keys, 4 x 2 heads of 192 / 384 fp32: 64 queries
  // 33 / 25, 60 / 42; 256 34 / 33, 98 / 92; 512 41 / 42, 152 / 165; 2 x 8 heads of 64 / 64 bf16: 64 14 / 11, 26 / 16; 512 18 / 15, 55 / 54
  p.img = vx_cdiv(s.sq, 64) > 4;
  if (!p.img)                // the form without images has 64 queries a workgroup, however many heads there are
    p.many = false;
  else if (c == kClasses - 1)
    p.many = 1.45 * vx_cdiv(n128, cus) < vx_cdiv(n64, cus);
  else
    p.many = n128 >= 2 * cus && !(dtype == VX_F32 && c >= kWideF32);
  p.tiles_q = vx_cdiv(s.sq, p.many ? 128 : 64);
  // few workgroups: split the keys so that every CU has one
  int64_t splits = p.tiles_q * bh > 0 ? cus / (p.tiles_q * bh) : 1;
  if (splits > tiles_k) splits = tiles_k;
  if (splits < 1) splits = 1;
  p.span = tiles_k ? vx_cdiv(tiles_k, splits) : 1;
  p.splits = tiles_k ? vx_cdiv(tiles_k, p.span) : 1;
  p.tiles_k = tiles_k;
  const size_t row = dtype == VX_F32 ? 6 : 2;      // bytes of a value's planes
  p.k_img = p.img ? (size_t)s.b * s.hk * tiles_k * kt * kDims[c][0] * row : 0;
  p.v_img = p.img ? (size_t)s.b * s.hv * tiles_k * kt * kDims[c][1] * row : 0;
  p.live = p.img ? live_bytes(s) : 0;
  return p;
}
size_t fwd_bytes(const Shape& s, int32_t dtype) {
  const FwdPlan p = fwd_plan(s, dtype);
  const size_t rows = p.splits > 1 ? (size_t)p.splits * s.b * s.h * s.sq : 0;
  return p.k_img + p.v_img + p.live + vx_align(rows * s.dv * 4) + vx_align(rows * 8);
}

// refuses a plan whose tiles are not those of the launched form: rows would stay unwritten
int32_t covers(int64_t tiles, int64_t rows, int64_t sq) {
  VX_REQUIRE(tiles * rows >= sq && (tiles - 1) * rows < sq, "attn_fwd: %lld tiles of %lld queries for %lld", (long long)tiles,
             (long long)rows, (long long)sq);
  return VX_OK;
}
template <typename T, int C>
int32_t launch_fwd(const FwdArgs<T>& a, const FwdPlan& p, unsigned grid, hipStream_t s) {
  constexpr int DP = kDims[C][0], DVP = kDims[C][1];
  constexpr bool WIDE = C == kClasses - 1, F32 = sizeof(T) == 4, MANY = WIDE || !F32 || C < kWideF32;
  constexpr int RT = 1, QG = 4, CS = WIDE ? 2 : 1;       // 64 queries; wide heads: two waves a query group
  // 128 queries: 32 a wave, but 16 and twice the waves for wide fp32 heads, whose registers hold no more
  constexpr int RT2 = WIDE && F32 ? 1 : 2, QG2 = WIDE && F32 ? 8 : 4, CS2 = WIDE && F32 ? 1 : CS;
  if (int32_t rc = covers(p.tiles_q, MANY && p.img && p.many ? 16 * RT2 * QG2 : 16 * RT * QG, a.sq)) return rc;
  if (MANY && p.img && p.many) {
    if constexpr (MANY) attn_fwd<T, DP, DVP, RT2, QG2, CS2, true, false><<<grid, 64 * QG2 * CS2, 0, s>>>(a);
  } else if (p.img) {
    attn_fwd<T, DP, DVP, RT, QG, CS, true, false><<<grid, 64 * QG * CS, 0, s>>>(a);
  } else {
    const auto kernel = args_fast(a) ? attn_fwd<T, DP, DVP, RT, QG, CS, false, true> : attn_fwd<T, DP, DVP, RT, QG, CS, false, false>;
    kernel<<<grid, 64 * CS * QG, 0, s>>>(a);
  }
  VX_LAUNCH_CHECK();
  return VX_OK;
}

template <typename T>
int32_t fwd_impl(FwdArgs<T>& a, const Shape& sh, int32_t dtype, char* ws, hipStream_t s) {
  const FwdPlan p = fwd_plan(sh, dtype);
  const int64_t bh = sh.b * sh.h, grid = p.tiles_q * p.splits * bh;
  VX_REQUIRE(vx_launchable(grid, 512), "attn_fwd: too many tiles");      // (the largest workgroup has 512)
  a.tiles_q = (int)p.tiles_q;
  a.splits = (int)p.splits;
  a.span = (int)p.span;
  const size_t rows = (size_t)p.splits * bh * sh.sq;
  a.k_img = ws;
  a.v_img = ws + p.k_img;
  char* lists = ws + p.k_img + p.v_img;
  a.part = (float*)(lists + p.live);
  a.part_ml = (float2*)(lists + p.live + vx_align(rows * sh.dv * 4));
  if (p.img && p.tiles_k) {
    const int c = class_of(sh.d, sh.dv), kd = kDims[c][0] / 32, nv = kDims[c][1] / 16, kt = AttnTile<T>::KT;
    const int64_t ks = sh.hk * p.tiles_k * (kt / 16) * kd * 64, all = ks + sh.hv * p.tiles_k * nv * (kt / 32) * 64;     // of a batch
    const int64_t per = vx_cdiv(all, 256);
    VX_REQUIRE(vx_launchable(per * sh.b, 256), "attn_fwd: too many keys");
    const bool own = a.mask && sh.sk <= kOwnKeys;
    LiveArgs live{};
    if (a.mask) {
      live = live_args(a, sh, lists);
      if (!own) {
        attn_live<<<(unsigned)sh.b, 256, 0, s>>>(live);
        VX_LAUNCH_CHECK();
      }
    }
    const auto pack = own ? attn_pack<T, true> : attn_pack<T, false>;
    pack<<<(unsigned)(per * sh.b), 256, 0, s>>>(a, live, ws, ws + p.k_img, (int)p.tiles_k, kd, nv, ks, all, (unsigned)per);
    VX_LAUNCH_CHECK();
  }
  int32_t rc;
  switch (class_of(sh.d, sh.dv)) {
    case 0: rc = launch_fwd<T, 0>(a, p, (unsigned)grid, s); break;
    case 1: rc = launch_fwd<T, 1>(a, p, (unsigned)grid, s); break;
    case 2: rc = launch_fwd<T, 2>(a, p, (unsigned)grid, s); break;
    case 3: rc = launch_fwd<T, 3>(a, p, (unsigned)grid, s); break;
    case 4: rc = launch_fwd<T, 4>(a, p, (unsigned)grid, s); break;
    default: rc = launch_fwd<T, 5>(a, p, (unsigned)grid, s); break;
  }
  if (rc) return rc;
  if (p.splits > 1) {
    const int quads = (a.dv + 3) / 4;
    const int64_t items = bh * sh.sq * quads;
    if (p.splits > 8)
      attn_join<T, 8><<<(unsigned)vx_cdiv(items, 32), 256, 0, s>>>(a, items, quads);
    else
      attn_join<T, 1><<<(unsigned)vx_cdiv(items, 256), 256, 0, s>>>(a, items, quads);
    VX_LAUNCH_CHECK();
  }
  return VX_OK;
}

struct BwdPlan {
  bool one;                                             // all keys fit one tile of attn_pds
  int64_t tp, tm, tn, skp, span, splits, chunk;         // queries per split, splits and queries per chunk
  size_t delta, pds, slab_k, slab_v, live, kc, vc;      // bytes
  size_t total() const { return delta + 2 * pds + slab_k + slab_v + live + kc + vc; }
};
// queries are cut into chunks, whose probabilities and score gradients are in memory at a time (at most kChunkBytes of both, but a
// tile of queries of every head at least), and a chunk into splits, one slab each; later chunks add to the slabs of the first
constexpr size_t kChunkBytes = (size_t)1 << 30;
BwdPlan bwd_plan(const Shape& s, int32_t dtype) {
  BwdPlan p;
  p.one = s.sk <= kPdsN;
  const int64_t cus = vx_tile_cus(), bh = s.b * s.h, e = dtype == VX_F32 ? 4 : 2, bk = dtype == VX_F32 ? 32 : 64;
  p.skp = vx_cdiv(s.sk, 8) * 8;
  // query rows of a tile; 4 x 2 heads, 1600 x 480, 192 / 384 wide, fp32 (416 tiles of 128): attn_pds 71 us with 64, 62 with 128,
  // attn_grads 82 and 84
  const int64_t t128 = vx_cdiv(s.sq, 128) * vx_cdiv(s.sk, 128) * bh;
  p.tp = !p.one && 2 * t128 >= 3 * cus ? 128 : 64;
  p.tm = !p.one && t128 >= 2 * cus ? 128 : 64;
  // wide heads: 192 and 384 columns without a ragged tile, and less staging per product (a lane stages 3 or 6 columns at a time)
  p.tn = !p.one && s.d > 128 && s.d % 24 == 0 && s.dv % 24 == 0 ? 192 : p.tm;
  int64_t fit = (int64_t)(kChunkBytes / 2) / (bh * p.skp * 4) / p.tm * p.tm;      // queries of a chunk
  if (fit < p.tm) fit = p.tm;
  const int64_t chunks = vx_cdiv(s.sq, fit);
  p.chunk = chunks == 1 ? s.sq : vx_cdiv(vx_cdiv(s.sq, chunks), p.tm) * p.tm;     // equal ones; no more than fit, a multiple of tm
  const int64_t tiles = vx_cdiv(s.sk, p.tm) * (vx_cdiv(s.dv, p.tn) + vx_cdiv(s.d, p.tn)) * bh;
  int64_t splits = 2 * cus / (tiles > 0 ? tiles : 1);
  if (splits < vx_cdiv(p.chunk, 2 * s.sk)) splits = vx_cdiv(p.chunk, 2 * s.sk);   // no workgroup much longer than those of dQ
  const int64_t most = vx_cdiv(p.chunk, 4 * bk);
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  p.span = vx_cdiv(vx_cdiv(p.chunk, splits), p.tm) * p.tm;
  p.splits = vx_cdiv(p.chunk, p.span);
  p.delta = vx_align((size_t)bh * s.sq * 4);
  p.pds = vx_align((size_t)bh * p.chunk * p.skp * 4);
  p.slab_k = vx_align((size_t)p.splits * bh * s.sk * s.d * 4);
  p.slab_v = vx_align((size_t)p.splits * bh * s.sk * s.dv * 4);
  p.live = live_bytes(s);
  p.kc = vx_align((size_t)s.b * s.hk * s.sk * s.d * e);
  p.vc = vx_align((size_t)s.b * s.hv * s.sk * s.dv * e);
  return p;
}

template <typename T, bool FAST>
int32_t bwd_chunk(const BwdArgs<T>& a, const BwdPlan& p, unsigned pds, unsigned grads, hipStream_t s) {
  const auto probs = p.one          ? attn_pds<T, 64, kPdsN, FAST, true>
                     : p.tp == 128 ? attn_pds<T, 128, kPdsN, FAST, false>
                                   : attn_pds<T, 64, kPdsN, FAST, false>;
  probs<<<pds, kTileThreads, 0, s>>>(a);
  VX_LAUNCH_CHECK();
  const auto sums = p.tm == 128 ? (p.tn == 192 ? attn_grads<T, 128, 192, FAST> : attn_grads<T, 128, 128, FAST>)
                                : (p.tn == 192 ? attn_grads<T, 64, 192, FAST> : attn_grads<T, 64, 64, FAST>);
  sums<<<grads, kTileThreads, 0, s>>>(a);
  VX_LAUNCH_CHECK();
  return VX_OK;
}

template <typename T>
int32_t bwd_impl(BwdArgs<T>& a, const Shape& sh, int32_t dtype, char* ws, hipStream_t s) {
  const BwdPlan p = bwd_plan(sh, dtype);
  const int64_t bh = sh.b * sh.h, rows = bh * sh.sq;
  a.delta = (float*)ws;
  a.p = (float*)(ws + p.delta);
  a.ds = (float*)(ws + p.delta + p.pds);
  a.slab_k = (float*)(ws + p.delta + 2 * p.pds);
  a.slab_v = (float*)(ws + p.delta + 2 * p.pds + p.slab_k);
  a.skp = (int)p.skp;
  a.bh = (int)bh;
  a.span = (int)p.span;
  a.tkp = (int)vx_cdiv(p.skp, kPdsN);
  a.tk = (int)vx_cdiv(sh.sk, p.tm);
  a.td = (int)vx_cdiv(sh.d, p.tn);
  a.tdv = (int)vx_cdiv(sh.dv, p.tn);
  char* at = ws + p.delta + 2 * p.pds + p.slab_k + p.slab_v;
  const int64_t sums = p.one ? 0 : rows;             // (attn_pds makes its own delta over one tile)
  const bool own = a.mask && sh.sk <= kOwnKeys;
  LiveArgs live{};
  GatherArgs gather{};
  int64_t head = 0;
  if (a.mask) {
    live = live_args(a, sh, at);
    a.kc = (T*)(at + p.live);
    a.vc = (T*)(at + p.live + p.kc);
    a.kc_h = sh.sk * sh.d;
    a.kc_b = sh.hk * a.kc_h;
    a.vc_h = sh.sk * sh.dv;
    a.vc_b = sh.hv * a.vc_h;
    constexpr int P = 16 / sizeof(T);
    gather.pieces_k = (int)vx_cdiv(sh.d, P);
    gather.pieces_v = (int)vx_cdiv(sh.dv, P);
    gather.items_k = sh.hk * sh.sk * gather.pieces_k;
    gather.items = gather.items_k + sh.hv * sh.sk * gather.pieces_v;
    VX_REQUIRE(vx_launchable(vx_cdiv(gather.items, 256) * sh.b, 256), "attn_bwd: too many keys");
    gather.per = (unsigned)vx_cdiv(gather.items, 256);
    head = own ? gather.per * sh.b : sh.b;
  }
  int64_t waves = vx_cdiv(sums, 4);
  if (waves > 1 << 20) waves = 1 << 20;              // (a wave then has more than one row)
  VX_REQUIRE(vx_launchable(waves + head, 256), "attn_bwd: too many keys");
  if (head + sums) {
    const auto delta = own ? attn_delta<T, true> : attn_delta<T, false>;
    delta<<<(unsigned)(waves + head), 256, 0, s>>>(a, sums, live, gather, (unsigned)head);
    VX_LAUNCH_CHECK();
  }
  if (a.mask) {
    if (!own) {
      attn_gather<T><<<(unsigned)(gather.per * sh.b), 256, 0, s>>>(a, gather);
      VX_LAUNCH_CHECK();
    }
    a.k = a.kc;
    a.k_b = a.kc_b; a.k_s = sh.d; a.k_h = a.kc_h;
    a.v = a.vc;
    a.v_b = a.vc_b; a.v_s = sh.dv; a.v_h = a.vc_h;
    a.mask = nullptr;
  }
  const bool fast = args_fast(a) && heads_fast(a.go, a.go_b, a.go_s, a.go_h, sh.dv, sizeof(T)) && p.skp < (1 << 21);
  for (int64_t q0 = 0; q0 < sh.sq; q0 += p.chunk) {
    a.q0 = (int)q0;
    a.rows = (int)(sh.sq - q0 < p.chunk ? sh.sq - q0 : p.chunk);
    a.add = q0 > 0;
    a.tq = (int)vx_cdiv(a.rows, p.tm);
    const int64_t here = vx_cdiv(a.rows, p.span);
    const int64_t nv = a.dvv ? here * bh * a.tk * a.tdv : 0, nk = a.dk ? here * bh * a.tk * a.td : 0;
    const int64_t nq = a.dq ? (int64_t)a.tq * a.td * bh : 0;
    const int64_t pds = (int64_t)a.tkp * vx_cdiv(a.rows, p.tp) * bh, grads = nv + nk + nq;
    VX_REQUIRE(vx_launchable(pds, kTileThreads) && vx_launchable(grads, kTileThreads), "attn_bwd: too many tiles");
    a.n_v = (unsigned)nv;
    a.n_k = (unsigned)nk;
    a.n_q = (unsigned)nq;
    a.tqp = (int)vx_cdiv(a.rows, p.tp);
    const int32_t rc = fast ? bwd_chunk<T, true>(a, p, (unsigned)pds, (unsigned)grads, s)
                            : bwd_chunk<T, false>(a, p, (unsigned)pds, (unsigned)grads, s);
    if (rc) return rc;
  }
  const int64_t iv = sh.b * sh.hv * sh.sk * vx_cdiv(sh.dv, 4), ik = sh.b * sh.hk * sh.sk * vx_cdiv(sh.d, 4);
  const int64_t gv = a.dvv ? vx_cdiv(iv, 256) : 0, gk = a.dk ? vx_cdiv(ik, 256) : 0;
  VX_REQUIRE(vx_launchable(gv + gk, 256), "attn_bwd: too many keys");
  if (gv + gk == 0) return VX_OK;
  attn_slab_sum<T><<<(unsigned)(gv + gk), 256, 0, s>>>(a, (int)p.splits, (unsigned)gv, iv, ik);
  VX_LAUNCH_CHECK();
  return VX_OK;
}

}  // namespace

extern "C" size_t vx_attn_fwd_workspace_bytes(const int64_t* shape, int32_t dtype) {
  if (check("attn_fwd", shape, dtype)) return 0;
  const Shape s = shape_of(shape);
  return s.b && s.sq ? fwd_bytes(s, dtype) : 0;
}

extern "C" size_t vx_attn_rest_bytes(const int64_t* shape, int32_t dtype) {
  if (check("attn_fwd", shape, dtype)) return 0;
  const Shape s = shape_of(shape);       // fp32: nothing is left behind; keys in one tile: attn_pds makes its own delta
  return dtype == VX_F32 || s.sk <= kPdsN ? 0 : (size_t)s.b * s.sq * s.h * s.dv * 2;
}

extern "C" int32_t vx_attn_fwd_rest(const void* d_q, const void* d_k, const void* d_v, const uint8_t* d_key_mask, const int64_t* shape,
                                    const int64_t* strides, float scale, void* d_out, float* d_stats, void* d_rest, int32_t dtype,
                                    void* d_workspace, size_t workspace_bytes, void* stream) {
  if (int32_t rc = check("attn_fwd", shape, dtype)) return rc;
  const Shape s = shape_of(shape);
  if (s.b == 0 || s.sq == 0) return VX_OK;
  VX_REQUIRE(strides && d_q && d_out && (s.sk == 0 || (d_k && d_v)), "attn_fwd: null pointer");
  for (int i = 0; i < 10; ++i) VX_REQUIRE(strides[i] >= 0, "attn_fwd: negative stride");
  const size_t need = fwd_bytes(s, dtype);
  if (workspace_bytes < need || (need && !d_workspace)) {
    vx_set_error("attn_fwd: workspace too small");
    return VX_ERR_WORKSPACE;
  }
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == VX_F32) {
    FwdArgs<float> a{};
    fill_args(a, s, strides, d_q, d_k, d_v, d_key_mask, scale);
    a.out = (float*)d_out;
    a.stats = (float2*)d_stats;
    return fwd_impl(a, s, dtype, (char*)d_workspace, st);
  }
  FwdArgs<__bf16> a{};
  fill_args(a, s, strides, d_q, d_k, d_v, d_key_mask, scale);
  a.out = (__bf16*)d_out;
  a.rest = (__bf16*)d_rest;
  a.stats = (float2*)d_stats;
  return fwd_impl(a, s, dtype, (char*)d_workspace, st);
}

extern "C" int32_t vx_attn_fwd(const void* d_q, const void* d_k, const void* d_v, const uint8_t* d_key_mask, const int64_t* shape,
                               const int64_t* strides, float scale, void* d_out, float* d_stats, int32_t dtype, void* d_workspace,
                               size_t workspace_bytes, void* stream) {
  return vx_attn_fwd_rest(d_q, d_k, d_v, d_key_mask, shape, strides, scale, d_out, d_stats, nullptr, dtype, d_workspace, workspace_bytes,
                          stream);
}

extern "C" size_t vx_attn_bwd_workspace_bytes(const int64_t* shape, int32_t dtype) {
  if (check("attn_bwd", shape, dtype)) return 0;
  const Shape s = shape_of(shape);
  return s.b && s.sq && s.sk ? bwd_plan(s, dtype).total() : 0;
}

template <typename T>
static int32_t attn_bwd_typed(const Shape& s, const void* d_dout, const int64_t* dout_strides, const void* d_q, const void* d_k,
                              const void* d_v, const uint8_t* d_key_mask, const int64_t* strides, const void* d_out,
                              const float* d_stats, const void* d_rest, float scale, void* d_dq, void* d_dk, void* d_dv, int32_t dtype,
                              void* ws, hipStream_t st) {
  BwdArgs<T> a{};
  fill_args(a, s, strides, d_q, d_k, d_v, d_key_mask, scale);
  a.out = (const T*)d_out;
  a.rest = (const T*)d_rest;
  a.go = (const T*)d_dout;
  a.go_b = dout_strides[0];
  a.go_s = dout_strides[1];
  a.go_h = dout_strides[2];
  a.stats = (const float2*)d_stats;
  a.dq = (T*)d_dq;
  a.dk = (T*)d_dk;
  a.dvv = (T*)d_dv;
  a.scale = scale;
  return bwd_impl(a, s, dtype, (char*)ws, st);
}

extern "C" int32_t vx_attn_bwd_rest(const void* d_dout, const int64_t* dout_strides, const void* d_q, const void* d_k, const void* d_v,
                                    const uint8_t* d_key_mask, const int64_t* shape, const int64_t* strides, const void* d_out,
                                    const float* d_stats, const void* d_rest, float scale, void* d_dq, void* d_dk, void* d_dv,
                                    int32_t dtype, void* d_workspace, size_t workspace_bytes, void* stream) {
  if (int32_t rc = check("attn_bwd", shape, dtype)) return rc;
  const Shape s = shape_of(shape);
  const hipStream_t st = (hipStream_t)stream;
  const size_t e = dtype == VX_F32 ? 4 : 2;
  if (s.b == 0 || s.sq == 0 || s.sk == 0) {          // nothing attends: zero gradients
    const size_t nq = (size_t)s.b * s.sq * s.h * s.d * e, nk = (size_t)s.b * s.sk * s.hk * s.d * e,
                 nv = (size_t)s.b * s.sk * s.hv * s.dv * e;
    if (nq && d_dq)
      if (int32_t rc = vx_fill_async(d_dq, 0, nq, st)) return rc;
    if (nk && d_dk)
      if (int32_t rc = vx_fill_async(d_dk, 0, nk, st)) return rc;
    if (nv && d_dv)
      if (int32_t rc = vx_fill_async(d_dv, 0, nv, st)) return rc;
    return VX_OK;
  }
  VX_REQUIRE(strides && dout_strides && d_dout && d_q && d_k && d_v && d_out && d_stats, "attn_bwd: null pointer");
  for (int i = 0; i < 10; ++i) VX_REQUIRE(strides[i] >= 0, "attn_bwd: negative stride");
  for (int i = 0; i < 3; ++i) VX_REQUIRE(dout_strides[i] >= 0, "attn_bwd: negative stride");
  if (workspace_bytes < bwd_plan(s, dtype).total() || !d_workspace) {
    vx_set_error("attn_bwd: workspace too small");
    return VX_ERR_WORKSPACE;
  }
  if (!d_dq && !d_dk && !d_dv) return VX_OK;
  const auto typed = dtype == VX_F32 ? attn_bwd_typed<float> : attn_bwd_typed<__bf16>;
  return typed(s, d_dout, dout_strides, d_q, d_k, d_v, d_key_mask, strides, d_out, d_stats, d_rest, scale, d_dq, d_dk, d_dv, dtype,
               d_workspace, st);
}

extern "C" int32_t vx_attn_bwd(const void* d_dout, const int64_t* dout_strides, const void* d_q, const void* d_k, const void* d_v,
                               const uint8_t* d_key_mask, const int64_t* shape, const int64_t* strides, const void* d_out,
                               const float* d_stats, float scale, void* d_dq, void* d_dk, void* d_dv, int32_t dtype,
                               void* d_workspace, size_t workspace_bytes, void* stream) {
  return vx_attn_bwd_rest(d_dout, dout_strides, d_q, d_k, d_v, d_key_mask, shape, strides, d_out, d_stats, nullptr, scale, d_dq, d_dk,
                          d_dv, dtype, d_workspace, workspace_bytes, stream);
}
