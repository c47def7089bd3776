// Attention over tokens with a sliding window and a few first tokens that stay visible ("sinks"), several heads, key / value heads
// shared by groups of query heads, sequences of different lengths; fp32 or bf16 in HBM, fp32 softmax and accumulators.
//
//   o_i = sum_j P_ij v_j,  P_ij = exp(c' q_i.k_j - lse_i) over the visible j:
//   i, j < n,  (i - left <= j <= i + right  or  j < sinks),  causal: j <= i           (a row i >= n gives zeros)
//
// All three kernels (FWD, DQ: the owner is a query; DKV: the owner is a key) have one shape.  A wavefront owns 32 tokens and holds
// their vectors as matrix-instruction operands in registers; the other side streams through LDS in double-buffered tiles of BN
// tokens that all wavefronts of the workgroup share.  Where that makes too few workgroups for the chip (SHARE), the wavefronts of a
// workgroup own the same 32 tokens instead, each streams every WV-th tile through LDS of its own, without barriers, and their partial
// results are joined in LDS at the end.
//   S^T[y][x] = sum_d Y[y][d] X[x][d]      A = rows of the tile, B = the owners: lane (l31, lhi) ends up with the owner x = l31 and
//                                          y = 32 yb + 8 (r >> 2) + (r & 3) + 4 lhi in accumulator register r of block yb -- so a
//                                          row's maximum and sum are in-lane work and one exchange with lane ^ 32
//   out^T[d][x] += sum_y Z[y][d] W[y][x]   eight registers of a block, rounded to the operand type, ARE the B operand (k position t
//                                          <-> y = 8 (t >> 2) + 4 lhi + (t & 3)); A is read transposed out of the same tile
//                                          (ds_read_b64_tr_b16 on bf16), and out keeps the owner in the lane: rescaling is in-lane
// On fp32 the same operands are 8 values a lane and a product is 8 v_mfma_f32_32x32x2_f32 (their k order differs from the bf16
// instruction's, the same way on both sides).  P and dS enter the second product on bf16 tensors as two operands, their rounding and what
// it left: o and every gradient then have the error of one rounding, 1.66e-3 of their norm (with one operand the gradients had 2.4e-3; the
// rest's products cost dq 57 -> 67 us and dk / dv 65 -> 82 us in the first case below).
// The softmax is exp2 with a running maximum that is raised only when a new logit exceeds it by 8 (P <= 256 then: no digit is lost,
// and the accumulators are rescaled once or twice a row instead of once a tile).
//
// What bounds the kernels is neither HBM nor the matrix instructions alone but the chain product -> exponential -> product of the
// few wavefronts that the registers allow, on vector instructions and LDS reads in turn.  8 sequences of 4096 tokens, 4 heads of 64, 256
// tokens of window to each side, 4 sinks (bf16; medians of a kernel trace): forward 52 us (4 wavefronts a SIMD, vector unit busy 61 %, matrix
// unit 29 %; 330 TFLOP/s of the formula's two products), dq 67 us (48 % and 30 %), the sinks' part 15 + 5 us, dk / dv 82 us (2 wavefronts a
// SIMD, 45 % and 34 %).  5 ragged sequences of 1543, 8 heads of 128 on 2, causal: 39, 48, 93 + 12 us.  2 x 1021 fp32 tokens, 4 heads of 40: 12, 14,
// 25 + 4 us.  256 tokens, 4 heads of 64: 6.3 us.  Every token of 8 x 4096, 4 heads of 64: bf16 267 us (510 TFLOP/s), 321, 479; fp32 1168 us
// (118 TFLOP/s), 1640, 2135.
#include "indm_common.h"
#pragma clang diagnostic ignored "-Winline-asm"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16;

__device__ __attribute__((aligned(16))) const unsigned zero16[4] = {0u, 0u, 0u, 0u};   // what a chunk outside a tensor reads

struct WAttnArgs {
  const void *q, *k, *v;            // [B, T, heads, D], D contiguous, 16-byte rows; strides in elements
  long qb, qt, qh, kb, kt, kh, vb, vt, vh;
  const void *o, *dO;               // dense [B, T, H, D] (backward)
  void* olo;                        // bf16: what rounding o left, rounded itself (written by the forward pass, read by the backward), or NULL
  void *out, *dq, *dk, *dv;         // dense
  float* lse;                       // [B, H, T]: log2 of the sum of exponentials, in units of the exp2 argument
  float* delta;                     // [B, H, T]: <dO, o>
  float* part;                      // sink partials [B Hk][chunks, without splits + 1][sinks][2][D]
  float* split;                     // partial dk, dv [splits][B Hk][T][2][D]
  const int* lengths;               // [B] or NULL
  int B, T, H, Hk, D, left, right, sinks, causal, tiles, chunks, splits, sunk;
  float c, scale;                   // scale * log2(e), scale
};

constexpr long MAX_STRIDE = 1 << 22;   // elements between tokens: a tile's byte offsets stay below 2^31

constexpr int pow2_ceil(int n) { return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32; }

template <typename T, int DP>
struct Geo {
  static constexpr int EPC = 16 / (int)sizeof(T);                  // elements of a 16-byte chunk
  static constexpr int CH = DP / EPC, NCH = pow2_ceil(CH);         // chunks of a row, and with padding to a power of two
  static constexpr int RB = NCH * 16;                              // bytes of a row in LDS
  static constexpr int BN = sizeof(T) == 2 ? 64 : 32, NY = BN / 32;   // streamed tokens a tile
  static constexpr int TILE = BN * RB;
  static constexpr int KK = DP / 16, DB = (DP + 31) / 32;     // 16-element steps of a product over d, blocks of 32 output elements
  // LDS address of chunk c of row r: c ^ swz(r).  16 successive rows at one chunk (the row-wise operand reads) and four
  // successive rows at one 64-byte unit (the transposed ones) then fall on different banks.
  static __device__ __forceinline__ int swz(int r) {
    return NCH == 4 ? (r >> 2) & 3 : NCH == 8 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
  }
};

// wavefronts a SIMD that the register allocation aims at (kind 0: forward, 1: dq, 2: dk / dv): 512 registers a SIMD lane over 4, 3, 2 or
// 1, so that nothing in a loop spills (the compiler reports 12 bytes of scratch for the forward kernel of bf16 heads of 49 to 64, none for any
// other).  bf16 dk / dv of heads of more than 96: 85 to 93 registers spill at two wavefronts (8 x 4096 tokens, 4 heads of 128: 267 us, at one
// 195 us).  Workgroups that share an owner block fill a compute unit's LDS: one wavefront a SIMD.
constexpr int waves_per_simd(int size, int DP, int kind, bool share) {
  if (share) return 1;
  if (size == 2) return DP <= 64 ? (kind == 0 ? 4 : kind == 1 ? 3 : 2) : DP > 96 && kind == 2 ? 1 : 2;
  return DP <= 32 ? 3 : DP <= 64 ? (kind == 0 ? 3 : 2) : DP <= 96 && kind == 0 ? 2 : 1;
}
// wavefronts of a workgroup that shares an owner block: each streams tiles of its own, 128 KB of LDS together
template <typename T, int DP> constexpr int share_waves() { return Geo<T, DP>::TILE <= 8192 ? 4 : 2; }

template <typename T> struct Op;
template <> struct Op<u16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag zero() {
    const u32x4 z = {0u, 0u, 0u, 0u};
    return __builtin_bit_cast(frag, z);
  }
  static __device__ __forceinline__ frag global(const u16* p) { return *(const bf16x8*)p; }
  static __device__ __forceinline__ frag pack(const f32x16& s, int o) {
    return indm_pack_bf16x8(s[o], s[o + 1], s[o + 2], s[o + 3], s[o + 4], s[o + 5], s[o + 6], s[o + 7]);
  }
  static __device__ __forceinline__ frag pack_rest(const f32x16& s, const frag& w, int o) {   // what pack's rounding left
    const u32x4 u = __builtin_bit_cast(u32x4, w);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = s[o + 2 * i] - __uint_as_float(u[i] << 16);
      v[2 * i + 1] = s[o + 2 * i + 1] - __uint_as_float(u[i] & 0xffff0000u);
    }
    return indm_pack_bf16x8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
  }
  static __device__ __forceinline__ float get(const frag& f, int i) { return (float)f[i]; }
};
struct f32frag {
  f32x4 a, b;
};
template <> struct Op<float> {
  typedef f32frag frag;
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.a[i], b.a[i], c, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.b[i], b.b[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ frag zero() {
    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
    return {z, z};
  }
  static __device__ __forceinline__ frag global(const float* p) { return {*(const f32x4*)p, *(const f32x4*)(p + 4)}; }
  static __device__ __forceinline__ frag pack(const f32x16& s, int o) {
    const f32x4 a = {s[o], s[o + 1], s[o + 2], s[o + 3]}, b = {s[o + 4], s[o + 5], s[o + 6], s[o + 7]};
    return {a, b};
  }
  static __device__ __forceinline__ float get(const frag& f, int i) { return i < 4 ? f.a[i] : f.b[i - 4]; }
};

template <typename T> using Frag = typename Op<T>::frag;

// value of the other half of the wavefront combined with this one's: x over lanes l31 and l31 + 32
__device__ __forceinline__ float half_max(float x) {
  const unsigned u = __float_as_uint(x);
  const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(u, u, false, false));
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const unsigned u = __float_as_uint(x);
  const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(u, u, false, false));
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// the lane's places in a tile, computed once
template <typename T, int DP>
struct Lane {
  using G = Geo<T, DP>;
  int l31, lhi, row, tr0, tr1, x, t0, t1;
  __device__ __forceinline__ Lane(int lane) {
    l31 = lane & 31;
    lhi = lane >> 5;
    row = l31 * G::RB;                       // row-wise operand: row l31, chunk (.. + lhi) ^ x
    x = G::swz(l31);
    if constexpr (sizeof(T) == 2) {
      const int jj = (lane & 15) >> 2, g1 = (lane >> 4) & 1, c4 = lane & 3, r = 4 * lhi + jj;
      tr0 = r * G::RB + (c4 & 1) * 8;        // transposed operand: rows r and r + 8 of a 16-row group
      tr1 = tr0 + 8 * G::RB;
      t0 = (2 * g1 + (c4 >> 1)) ^ G::swz(r);
      t1 = (2 * g1 + (c4 >> 1)) ^ G::swz(r + 8);
    } else {
      tr0 = 4 * lhi * G::RB + (l31 & 3) * 4;
      tr1 = t0 = t1 = 0;
    }
  }
  // elements 16 kk + 8 lhi .. + 7 of row 32 yb + l31
  __device__ __forceinline__ typename Op<T>::frag rowwise(const char* tile, int yb, int kk) const {
    const char* p = tile + row + yb * 32 * G::RB;
    if constexpr (sizeof(T) == 2) {
      return *(const bf16x8*)(p + (((2 * kk + lhi) ^ x) << 4));
    } else {
      return {*(const f32x4*)(p + (((4 * kk + 2 * lhi) ^ x) << 4)), *(const f32x4*)(p + (((4 * kk + 2 * lhi + 1) ^ x) << 4))};
    }
  }
  // element d = 32 db + l31 of the eight rows r0 + 8 (t >> 2) + 4 lhi + (t & 3), r0 a multiple of 16
  __device__ __forceinline__ typename Op<T>::frag transposed(const char* tile, int r0, int db) const {
    if constexpr (sizeof(T) == 2) {
      const char* p = tile + r0 * G::RB;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(p + tr0 + (((db * 4) ^ t0) << 4)));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(p + tr1 + (((db * 4) ^ t1) << 4)));
      const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(bf16x8, v);
    } else {
      const char* p = tile + r0 * G::RB + tr0;
      const int chunk = db * 8 + (l31 >> 2);
      f32frag f;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int r = 8 * (t >> 2) + (t & 3);
        const float v = *(const float*)(p + r * G::RB + ((chunk ^ G::swz(r + 4 * lhi)) << 4));
        if (t < 4) f.a[t] = v; else f.b[t - 4] = v;
      }
      return f;
    }
  }
};

// out^T += Z^T W of 32 streamed tokens (rows row0 .. of the tile).  On bf16 W goes in as two operands, its rounding and what that left: W
// then is off by 2^-16 of itself, and the result by its own rounding alone.
template <typename T, int DP>
__device__ __forceinline__ void gather(const Lane<T, DP>& at, const char* tile, int row0, const f32x16& W, f32x16 (&out)[Geo<T, DP>::DB]) {
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const Frag<T> w = Op<T>::pack(W, 8 * a);
    if constexpr (sizeof(T) == 2) {
      const Frag<T> rest = Op<T>::pack_rest(W, w, 8 * a);
#pragma unroll
      for (int d = 0; d < Geo<T, DP>::DB; ++d) {
        const Frag<T> z = at.transposed(tile, row0 + 16 * a, d);
        out[d] = Op<T>::mma(z, rest, Op<T>::mma(z, w, out[d]));
      }
    } else {
#pragma unroll
      for (int d = 0; d < Geo<T, DP>::DB; ++d) out[d] = Op<T>::mma(at.transposed(tile, row0 + 16 * a, d), w, out[d]);
    }
  }
}

// rows first .. first + BN - 1 of a head -> a tile in LDS, by direct copies of 16 bytes a lane (1 KB a wave-instruction, the swizzle is
// on the source side).  A whole tile of whole rows needs no vector arithmetic in the loop: a scalar base plus the lane's byte offsets,
// which are computed once (the swizzle repeats every 16 rows: PER of them).  Otherwise rows from n on and chunks from D on read
// zeros: what lies behind a sequence never enters a product.
template <typename T, int DP, int WV>
struct Stager {
  using G = Geo<T, DP>;
  static constexpr int COPIES = G::BN * G::NCH / 64, N = (COPIES + WV - 1) / WV;
  static constexpr int R = WV * 64 / G::NCH;                  // rows from one of a wavefront's copies to its next
  static constexpr int PER = R >= 16 ? 1 : 16 / R < N ? 16 / R : N;
  unsigned off[PER];
  __device__ __forceinline__ Stager(long stride, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int slot = (wave + i * WV) * 64 + lane, r = slot / G::NCH, c = (slot % G::NCH) ^ G::swz(r);
      off[i] = (unsigned)(r * (int)stride + c * G::EPC) * (unsigned)sizeof(T);   // (the host keeps strides up to 2^22 elements)
    }
  }
  __device__ __forceinline__ void fetch(char* tile, const T* src, long stride, int first, int n, int D, int wave, int lane) const {
    const bool whole = first + G::BN <= n && D == DP && G::CH == G::NCH;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int w = wave + i * WV;
      if (COPIES % WV == 0 || w < COPIES) {
        char* dst = tile + w * 1024;
        const char* s = (const char*)(src + (long)(first + i / PER * (PER * R)) * stride) + off[i % PER];
        if (!whole) {
          const int slot = w * 64 + lane, r = slot / G::NCH, c = (slot % G::NCH) ^ G::swz(r);
          if (!(first + r < n && c * G::EPC < D)) s = (const char*)zero16;
        }
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)s,
                                         (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
      }
    }
  }
};
// this wavefront's copies have landed -- and, where a workgroup shares its tiles, everybody's
template <bool SHARE>
__device__ __forceinline__ void staged() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  if constexpr (!SHARE) __syncthreads();
}

// the owner's row as operands (rows from n on: zeros)
template <typename T, int DP>
__device__ __forceinline__ void load_owner(const T* row, bool live, int D, int lhi, Frag<T> (&f)[Geo<T, DP>::KK]) {
#pragma unroll
  for (int kk = 0; kk < Geo<T, DP>::KK; ++kk)
    f[kk] = live && 16 * kk + 8 * lhi < D ? Op<T>::global(row + 16 * kk + 8 * lhi) : Op<T>::zero();
}

// half a block of out^T -- accumulator registers 8 half .. + 7, elements 32 db + 16 half .. + 15 of the owner's row -- times f: 16
// bytes a lane and store.  (bf16: the halves of the wavefront trade, so that lane l31 holds elements 0 .. 7 and lane l31 + 32
// elements 8 .. 15.)
template <typename T>
__device__ __forceinline__ void store_half(T* row, const float (&a)[8], float f, bool live, int d0, int D, int lhi) {
  if constexpr (sizeof(T) == 2) {
    unsigned w[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x2 v = {a[4 * h + 2 * e] * f, a[4 * h + 2 * e + 1] * f};
        w[h][e] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
      }
    const u32x2 s0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false));
    const u32x2 s1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false));
    const u32x4 o = {s0[0], s1[0], s0[1], s1[1]};
    const int d = d0 + 8 * lhi;
    if (live && d < D) *(u32x4*)(row + d) = o;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 o = {a[4 * h] * f, a[4 * h + 1] * f, a[4 * h + 2] * f, a[4 * h + 3] * f};
      const int d = d0 + 8 * h + 4 * lhi;
      if (live && d < D) *(f32x4*)(row + d) = o;
    }
  }
}
template <int DB>
__device__ __forceinline__ void half_of(const f32x16 (&acc)[DB], int u, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = acc[u >> 1][8 * (u & 1) + e];
}

// Where the wavefronts of a workgroup shared an owner block: their accumulators go to LDS (a wavefront's N vectors of four registers,
// [vector][lane]), and each wavefront adds up some of the halves, over the wavefronts in order.
template <int WV, int N>
struct Join {
  float* red;
  int lane;
  template <int DB>
  __device__ __forceinline__ void leave(const f32x16 (&acc)[DB], int wave, int first) const {
#pragma unroll
    for (int v = 0; v < 4 * DB; ++v) {
      const f32x4 w = {acc[v >> 2][4 * (v & 3)], acc[v >> 2][4 * (v & 3) + 1], acc[v >> 2][4 * (v & 3) + 2], acc[v >> 2][4 * (v & 3) + 3]};
      *(f32x4*)(red + ((wave * N + first + v) * 64 + lane) * 4) = w;
    }
  }
  __device__ __forceinline__ void half(int u, const float (&f)[WV], float (&v)[8]) const {   // sum of f[w] times wavefront w's half u
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
    for (int w = 0; w < WV; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 a = *(const f32x4*)(red + ((w * N + 2 * u + h) * 64 + lane) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] = __builtin_fmaf(a[e], f[w], v[4 * h + e]);
      }
  }
};

// workgroup -> work item, so that neighbouring items (which share most of their tiles) run on one XCD's L2.  (Items run over a head's
// blocks, then the sequences, then the heads: every XCD gets all sequences, whatever their lengths.  Five sequences, one of them empty,
// 1543 x 8 heads of 128: forward 44 -> 39 us, dk / dv 122 -> 94 us against all heads of a sequence together.)
__device__ __forceinline__ int xcd_item(int id, int total) {
  const int x = id & 7, per = total >> 3, rem = total & 7;
  return x * per + (x < rem ? x : rem) + (id >> 3);
}

__device__ __forceinline__ int seq_len(const WAttnArgs& p, int b) {
  if (p.lengths == nullptr) return p.T;
  const int n = p.lengths[b];
  return n < 0 ? 0 : n < p.T ? n : p.T;
}

// tiles of keys that queries q0 .. q1 of a sequence of n see: [0, ns) and [t0, t1]
struct KeyTiles {
  int ns, t0, count;
};
__device__ __forceinline__ KeyTiles key_tiles(const WAttnArgs& p, int q0, int q1, int n, int BN) {
  if (q0 >= n) return {0, 0, 0};
  if (q1 > n - 1) q1 = n - 1;
  int lo = q0 - p.left, hi = p.causal ? q1 : q1 + p.right;
  lo = lo < 0 ? 0 : lo;
  hi = hi > n - 1 ? n - 1 : hi;
  int s = p.sinks < n ? p.sinks : n;
  if (p.causal && s > q1 + 1) s = q1 + 1;
  const int st = (s + BN - 1) / BN;
  int t0 = lo / BN, t1 = hi / BN;
  if (st >= t0) {
    t0 = s > 0 ? 0 : t0;
    if (st - 1 > t1) t1 = st - 1;
    return {0, t0, t1 - t0 + 1};
  }
  return {st, t0, st + t1 - t0 + 1};
}

// ---------------------------------------------------------------------------------------------- owner = queries: forward, dq
template <typename T, int DP, int WV, bool SHARE, bool BWD>
__global__ __launch_bounds__(WV * 64, waves_per_simd(sizeof(T), DP, BWD ? 1 : 0, SHARE)) void wattn_query_kernel(WAttnArgs p) {
  using G = Geo<T, DP>;
  using O = Op<T>;
  typedef typename O::frag frag;
  constexpr int OWN = SHARE ? 32 : WV * 32, STEP = SHARE ? WV : 1;
  extern __shared__ __attribute__((aligned(16))) char smem_all[];   // [2 buffers][K tile, V tile], SHARE: for each wavefront
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Lane<T, DP> at(lane);
  const int item = xcd_item(blockIdx.x, gridDim.x);
  const int tile = item % p.tiles, bh = item / p.tiles, h = bh / p.B, b = bh % p.B;
  const int n = seq_len(p, b);
  char* smem = smem_all + (SHARE ? wave * 4 * G::TILE : 0);
  const int q0 = tile * OWN, qw = q0 + (SHARE ? 0 : wave * 32), i = qw + at.l31;
  const int hk = h / (p.H / p.Hk);
  const T* K = (const T*)p.k + b * p.kb + hk * p.kh;
  const T* V = (const T*)p.v + b * p.vb + hk * p.vh;
  const long orow = (((long)b * p.T + i) * p.H + h) * p.D, srow = ((long)b * p.H + h) * p.T + i;
  const bool live = i < n;
  const bool wanted = !BWD || p.dq != nullptr;   // (dq not wanted: <dO, o> alone, for the other kernels)
  const KeyTiles kt = key_tiles(p, q0, q0 + OWN - 1, wanted ? n : 0, G::BN);
  auto first_of = [&](int it) { return (it < kt.ns ? it : kt.t0 + it - kt.ns) * G::BN; };
  const int swave = SHARE ? 0 : wave, it0 = SHARE ? wave : 0;
  const Stager<T, DP, SHARE ? 1 : WV> ks(p.kt, swave, lane), vs(p.vt, swave, lane);
  auto fetch = [&](int it, int side) {
    char* buf = smem + side * 2 * G::TILE;
    ks.fetch(buf, K, p.kt, first_of(it), n, p.D, swave, lane);
    vs.fetch(buf + G::TILE, V, p.vt, first_of(it), n, p.D, swave, lane);
  };
  if (it0 < kt.count) fetch(it0, 0);

  frag qf[G::KK], df[BWD ? G::KK : 1];
  load_owner<T, DP>((const T*)p.q + b * p.qb + (long)i * p.qt + h * p.qh, live, p.D, at.lhi, qf);
  float lse = INFINITY, delta = 0.f;
  if constexpr (BWD) {
    load_owner<T, DP>((const T*)p.dO + orow, live, p.D, at.lhi, df);
    frag of[G::KK];
    load_owner<T, DP>((const T*)p.o + orow, live, p.D, at.lhi, of);
#pragma unroll
    for (int kk = 0; kk < G::KK; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += O::get(df[kk], e) * O::get(of[kk], e);
    if (sizeof(T) == 2 && p.olo != nullptr) {
      load_owner<T, DP>((const T*)p.olo + orow, live, p.D, at.lhi, of);
#pragma unroll
      for (int kk = 0; kk < G::KK; ++kk)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta += O::get(df[kk], e) * O::get(of[kk], e);
    }
    delta = half_sum(delta);
    if (live) lse = p.lse[srow];
    if (i < p.T && at.lhi == 0 && (!SHARE || wave == 0)) p.delta[srow] = delta;
  }
  // the lane's visible keys: lo .. lo + span, and those below sk (a row behind the sequence: none)
  int lo = i - p.left, hi = p.causal ? i : i + p.right, sk = p.sinks;
  if (hi > n - 1) hi = n - 1;
  if (p.causal && sk > i + 1) sk = i + 1;
  if (sk > n) sk = n;
  unsigned span = (unsigned)(hi - lo);
  if (!live) {
    lo = 0x7fffffff;
    span = 0;
    sk = 0;
  }

  f32x16 acc[G::DB];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  float m = -INFINITY, sum = 0.f;   // running maximum in use (units of the exp2 argument), this lane's half of the sum
  const int qa = qw, qb = qw + 31 < n - 1 ? qw + 31 : n - 1;

  if (it0 < kt.count) staged<SHARE>();
  for (int it = it0, side = 0; it < kt.count; it += STEP, side ^= 1) {
    if (it + STEP < kt.count) fetch(it + STEP, side ^ 1);
    const char* kb = smem + side * 2 * G::TILE;
    const char* vb = kb + G::TILE;
#pragma unroll
    for (int y = 0; y < G::NY; ++y) {
      const int k0 = first_of(it) + 32 * y, k1 = k0 + 31;
      // (wave-uniform) does any of this wavefront's queries see any of these 32 keys?  all of all?
      const bool any = qa < n && k0 < n && (k0 < p.sinks || (k1 >= qa - p.left && (p.causal || k0 <= qb + p.right))) && (!p.causal || k0 <= qb);
      const bool all = qa + 31 < n && k1 < n && (k1 < p.sinks || (k0 >= qa + 31 - p.left && (p.causal || k1 <= qa + p.right))) && (!p.causal || k1 <= qa);
      if (!any) continue;
      f32x16 S;
#pragma unroll
      for (int r = 0; r < 16; ++r) S[r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < G::KK; ++kk) S = O::mma(at.rowwise(kb, y, kk), qf[kk], S);
      if (!all) {
        const unsigned from = (unsigned)(k0 + 4 * at.lhi - lo);
        if (k0 < p.sinks) {
          const int left = sk - k0 - 4 * at.lhi;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = 8 * (r >> 2) + (r & 3);
            S[r] = from + j <= span || j < left ? S[r] : -INFINITY;
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) S[r] = from + 8 * (r >> 2) + (r & 3) <= span ? S[r] : -INFINITY;
        }
      }
      if constexpr (!BWD) {
        float top = S[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, S[r]);
        top = half_max(top) * p.c;
        if (__any(top > m + 8.f)) {   // (-inf + 8 = -inf: the first visible key always raises it)
          asm volatile("" ::: "memory");   // (keeps the rescaling behind the branch)
          const float up = fmaxf(m, top);
          const float f = up > -INFINITY ? __builtin_amdgcn_exp2f(m - up) : 1.f;
          m = up;
          sum *= f;
#pragma unroll
          for (int d = 0; d < G::DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= f;
        }
        const float mm = m > -INFINITY ? m : 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          S[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r], p.c, -mm));
          sum += S[r];
        }
      } else {
        f32x16 dP;
#pragma unroll
        for (int r = 0; r < 16; ++r) dP[r] = 0.f;
#pragma unroll
        for (int kk = 0; kk < G::KK; ++kk) dP = O::mma(at.rowwise(vb, y, kk), df[kk], dP);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          S[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r], p.c, -lse)) * (dP[r] - delta);   // dS / scale
      }
      gather<T, DP>(at, BWD ? kb : vb, 32 * y, S, acc);
    }
    staged<SHARE>();
  }

  if (!wanted) return;
  if constexpr (!BWD) sum = half_sum(sum);
  float inv = sum > 0.f ? 1.f / sum : 0.f;
  auto emit = [&](int u, float (&v)[8]) {   // a half of the result, before the division by the sum
    if (!live) {   // (also where a visible key's values were infinite: 0 times that is not 0)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    if constexpr (BWD) {
      store_half<T>((T*)p.dq + orow, v, p.scale, i < p.T, 16 * u, p.D, at.lhi);
    } else {
      store_half<T>((T*)p.out + orow, v, inv, i < p.T, 16 * u, p.D, at.lhi);
      if (sizeof(T) == 2 && p.olo != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = v[e] * inv;
          v[e] = x - (float)(__bf16)x;
        }
        store_half<T>((T*)p.olo + orow, v, 1.f, i < p.T, 16 * u, p.D, at.lhi);
      }
    }
  };
  if constexpr (SHARE) {
    const Join<WV, 4 * G::DB> join = {(float*)smem_all, lane};
    float2* stats = (float2*)(smem_all + WV * 4 * G::DB * 1024);
    __syncthreads();
    join.leave(acc, wave, 0);
    if constexpr (!BWD) stats[wave * 64 + lane] = make_float2(m, sum);
    __syncthreads();
    float f[WV];
#pragma unroll
    for (int w = 0; w < WV; ++w) f[w] = 1.f;
    if constexpr (!BWD) {
      m = -INFINITY;
      sum = 0.f;
#pragma unroll
      for (int w = 0; w < WV; ++w) m = fmaxf(m, stats[w * 64 + lane].x);
#pragma unroll
      for (int w = 0; w < WV; ++w) {
        const float2 s = stats[w * 64 + lane];
        f[w] = m > -INFINITY ? __builtin_amdgcn_exp2f(s.x - m) : 1.f;
        sum += s.y * f[w];
      }
      inv = sum > 0.f ? 1.f / sum : 0.f;
    }
#pragma unroll
    for (int u = wave; u < 2 * G::DB; u += WV) {
      float v[8];
      join.half(u, f, v);
      emit(u, v);
    }
  } else {
#pragma unroll
    for (int u = 0; u < 2 * G::DB; ++u) {
      float v[8];
      half_of(acc, u, v);
      emit(u, v);
    }
  }
  if (!BWD && p.lse != nullptr && i < p.T && at.lhi == 0 && (!SHARE || wave == 0)) p.lse[srow] = live ? m + __log2f(sum) : INFINITY;
}

// ---------------------------------------------------------------------------------------------- owner = keys: dk, dv
// The queries of every head of the group stream past the key.  There are two kinds of workgroups: the last p.sunk ones gather what the
// sink keys get from queries whose window they are outside of -- a few keys against all queries, shared by p.chunks workgroups a block of
// them --, the others the window's part of all keys (SPLIT: where there are few key blocks, each one's queries shared by p.splits
// workgroups).  What several workgroups contribute to goes to fp32 partial sums that a last kernel adds up in order (no atomics).
// (WHO spares the launches of one kind the other's tests: 8 x 4096 tokens, 4 heads of 64, window 256 + 256 without sinks: 79 instead of 83 us.)
enum { KEYS = 1, SINKS = 2, BOTH = 3 };
template <typename T, int DP, int WV, bool SHARE, bool SPLIT, int WHO>
__global__ __launch_bounds__(WV * 64, waves_per_simd(sizeof(T), DP, 2, SHARE)) void wattn_key_kernel(WAttnArgs p) {
  using G = Geo<T, DP>;
  using O = Op<T>;
  typedef typename O::frag frag;
  constexpr int OWN = SHARE ? 32 : WV * 32, STEP = SHARE ? WV : 1, BUF = 2 * G::TILE + 2 * G::BN * (int)sizeof(float);
  extern __shared__ __attribute__((aligned(16))) char smem_all[];   // [2 buffers][Q tile, dO tile, lse, delta], SHARE: for each wavefront
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Lane<T, DP> at(lane);
  const int blocks = gridDim.x - p.sunk;
  const bool sink = WHO == SINKS || (WHO == BOTH && (int)blockIdx.x >= blocks);
  const int item = sink ? xcd_item(blockIdx.x - blocks, p.sunk) : xcd_item(blockIdx.x, blocks);
  const int shares = sink ? p.chunks : SPLIT ? p.splits : 1, per = (sink ? (p.sinks + OWN - 1) / OWN : p.tiles) * shares;
  const int hk = item / per / p.B, b = item / per % p.B, bh = b * p.Hk + hk;
  const int share = item % per % shares, tile = item % per / shares;
  const int n = seq_len(p, b), group = p.H / p.Hk;
  char* smem = smem_all + (SHARE ? wave * 2 * BUF : 0);
  const int j0 = tile * OWN, jw = j0 + (SHARE ? 0 : wave * 32), j = jw + at.l31;
  const bool live = j < n;
  // tiles of queries: i0 .. i1 of each head of the group, one after the other, of which this workgroup takes its share
  int i0, i1;
  if (sink) {
    i0 = p.causal ? j0 : 0;
    i1 = n - 1;
  } else {
    i0 = p.causal ? j0 : j0 - p.right;
    i1 = j0 + OWN - 1 + p.left;
    i0 = i0 < 0 ? 0 : i0;
    i1 = i1 > n - 1 ? n - 1 : i1;
  }
  const int t0 = i0 / G::BN, nt = j0 < n && i1 >= i0 ? i1 / G::BN - t0 + 1 : 0;
  const int all_tiles = nt * group, to = (int)((long)all_tiles * (share + 1) / shares);
  const int from = (int)((long)all_tiles * share / shares) + (SHARE ? wave : 0), swave = SHARE ? 0 : wave;
  const Stager<T, DP, SHARE ? 1 : WV> qs(p.qt, swave, lane), ds((long)p.H * p.D, swave, lane);
  float hold[2];
  auto fetch = [&](int it, int side) {
    const int h = hk * group + it / nt, first = (t0 + it % nt) * G::BN;
    char* buf = smem + side * BUF;
    qs.fetch(buf, (const T*)p.q + b * p.qb + h * p.qh, p.qt, first, n, p.D, swave, lane);
    ds.fetch(buf + G::TILE, (const T*)p.dO + ((long)b * p.T * p.H + h) * p.D, (long)p.H * p.D, first, n, p.D, swave, lane);
    const int i = first + lane;
    if (swave == 0 && lane < G::BN) {
      const long s = ((long)b * p.H + h) * p.T + i;
      hold[0] = i < n ? p.lse[s] : INFINITY;
      hold[1] = i < n ? p.delta[s] : 0.f;
    }
  };
  auto put = [&](int side) {   // (the row statistics go through registers: written once the tile's reads are on their way)
    if (swave == 0 && lane < G::BN) {
      float* st = (float*)(smem + side * BUF + 2 * G::TILE);
      st[lane] = hold[0];
      st[G::BN + lane] = hold[1];
    }
  };
  if (from < to) fetch(from, 0);

  frag kf[G::KK], vf[G::KK];
  load_owner<T, DP>((const T*)p.k + b * p.kb + (long)j * p.kt + hk * p.kh, live, p.D, at.lhi, kf);
  load_owner<T, DP>((const T*)p.v + b * p.vb + (long)j * p.vt + hk * p.vh, live, p.D, at.lhi, vf);
  // the lane's queries.  window: lo .. hi.  sinks: up to last, outside of lo .. hi
  int lo = p.causal ? j : j - p.right, hi = j + p.left, last = n - 1;
  if (sink) {
    if (p.causal) lo = -(1 << 30);
    if (j >= p.sinks || !live) last = -1;
  } else {
    if (hi > n - 1) hi = n - 1;
    if (!live) {
      lo = 0x7fffffff;
      hi = lo;
    }
  }
  const unsigned span = (unsigned)(hi - lo);

  f32x16 dk[G::DB], dv[G::DB];
#pragma unroll
  for (int d = 0; d < G::DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.f;

  if (from < to) {
    put(0);
    staged<SHARE>();
  }
  for (int it = from, side = 0; it < to; it += STEP, side ^= 1) {
    if (it + STEP < to) fetch(it + STEP, side ^ 1);
    const char* qb = smem + side * BUF;
    const char* db = qb + G::TILE;
    const float* st = (const float*)(db + G::TILE);
    const int first = (t0 + it % nt) * G::BN;
#pragma unroll
    for (int y = 0; y < G::NY; ++y) {
      const int ia = first + 32 * y, ib = ia + 31;   // (wave-uniform tests, as in the other kernel)
      bool any, all;
      if (sink) {
        any = jw < p.sinks && jw < n && ia < n && (ib > jw + p.left || (!p.causal && ia < jw + 31 - p.right));
        all = false;
      } else {
        any = jw < n && ia < n && ia <= jw + 31 + p.left && ib >= (p.causal ? jw : jw - p.right);
        all = jw + 31 < n && ib < n && ib <= jw + p.left && ia >= (p.causal ? jw + 31 : jw + 31 - p.right);
      }
      if (!any) continue;
      f32x16 P, dP;
#pragma unroll
      for (int r = 0; r < 16; ++r) P[r] = dP[r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < G::KK; ++kk) P = O::mma(at.rowwise(qb, y, kk), kf[kk], P);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 l4 = *(const f32x4*)(st + 32 * y + 8 * a + 4 * at.lhi);
#pragma unroll
        for (int e = 0; e < 4; ++e) P[4 * a + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(P[4 * a + e], p.c, -l4[e]));
      }
      if (!all) {
        asm volatile("" ::: "memory");   // (keeps the masks behind the branch)
        const unsigned at0 = (unsigned)(ia + 4 * at.lhi - lo);
        if (sink) {
          const int room = last - ia - 4 * at.lhi;
#pragma unroll
          for (int r = 0; r < 16; ++r) P[r] = 8 * (r >> 2) + (r & 3) <= room && at0 + 8 * (r >> 2) + (r & 3) > span ? P[r] : 0.f;
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) P[r] = at0 + 8 * (r >> 2) + (r & 3) <= span ? P[r] : 0.f;
        }
      }
      gather<T, DP>(at, db, 32 * y, P, dv);
#pragma unroll
      for (int kk = 0; kk < G::KK; ++kk) dP = O::mma(at.rowwise(db, y, kk), vf[kk], dP);
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const f32x4 d4 = *(const f32x4*)(st + G::BN + 32 * y + 8 * a + 4 * at.lhi);
#pragma unroll
        for (int e = 0; e < 4; ++e) P[4 * a + e] *= dP[4 * a + e] - d4[e];
      }
      gather<T, DP>(at, qb, 32 * y, P, dk);
    }
    if (it + STEP < to) put(side ^ 1);
    staged<SHARE>();
  }
  // a sink's partial sums: the chunks', and without splits one more from the window
  float* part = p.part + (((long)bh * (p.chunks + (SPLIT ? 0 : 1)) + (sink ? share : p.chunks)) * p.sinks + j) * 2 * p.D;
  const bool sunk = p.chunks > 0 && jw < p.sinks, ends = jw + 31 >= n;   // (wave-uniform)
  auto emit = [&](int u, float (&v)[8]) {   // a half: of dk, then of dv
    const bool first = u < 2 * G::DB;
    const int d0 = 16 * (first ? u : u - 2 * G::DB), at0 = first ? 0 : p.D;
    if (sink) {
      store_half<float>(part + at0, v, 1.f, j < p.sinks, d0, p.D, at.lhi);
    } else if constexpr (SPLIT) {
      store_half<float>(p.split + ((((long)share * p.B * p.Hk + bh) * p.T + j) * 2) * p.D + at0, v, 1.f, live, d0, p.D, at.lhi);
    } else {
      if (ends && !live) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
      if (sunk) store_half<float>(part + at0, v, 1.f, j < p.sinks, d0, p.D, at.lhi);
      store_half<T>((T*)(first ? p.dk : p.dv) + (((long)b * p.T + j) * p.Hk + hk) * p.D, v, first ? p.scale : 1.f,
                    j < p.T && !(sunk && j < p.sinks), d0, p.D, at.lhi);
    }
  };
  if constexpr (SHARE) {
    const Join<WV, 8 * G::DB> join = {(float*)smem_all, lane};
    __syncthreads();
    join.leave(dk, wave, 0);
    join.leave(dv, wave, 4 * G::DB);
    __syncthreads();
    float f[WV];
#pragma unroll
    for (int w = 0; w < WV; ++w) f[w] = 1.f;
#pragma unroll
    for (int u = wave; u < 4 * G::DB; u += WV) {
      float v[8];
      join.half(u, f, v);
      emit(u, v);
    }
  } else {
#pragma unroll
    for (int u = 0; u < 4 * G::DB; ++u) {
      float v[8];
      if (u < 2 * G::DB) half_of(dk, u, v);
      else half_of(dv, u - 2 * G::DB, v);
      emit(u, v);
    }
  }
}

// dk, dv of the sinks: their partial sums in order (without splits).  A workgroup's lanes own 64 of the n = sinks x 2 D values of a
// (sequence, key head), its wavefronts a sixteenth of the partial sums each.
template <typename T>
__global__ __launch_bounds__(1024) void wattn_sinks_kernel(WAttnArgs p) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slots = p.chunks + 1;
  const long n = (long)p.sinks * 2 * p.D, cols = (n + 63) / 64, groups = (long)p.B * p.Hk * cols;
  for (long g = blockIdx.x; g < groups; g += gridDim.x) {
    const long bh = g / cols, col = (g - bh * cols) * 64 + lane;
    const float* src = p.part + bh * slots * n + col;
    float s = 0.f;
    if (col < n) {
#pragma unroll 4
      for (int c = slots * wave / 16; c < slots * (wave + 1) / 16; ++c) s += src[c * n];
    }
    sh[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < n) {
      s = 0.f;
#pragma unroll
      for (int w = 0; w < 16; ++w) s += sh[w][lane];
      const long jw = col / p.D, j = jw >> 1, b = bh / p.Hk, hk = bh - b * p.Hk;
      if (j >= seq_len(p, (int)b)) s = 0.f;
      T* out = (T*)(jw & 1 ? p.dv : p.dk) + ((b * p.T + j) * p.Hk + hk) * p.D + (col - jw * p.D);
      if (!(jw & 1)) s *= p.scale;
      if constexpr (sizeof(T) == 2) *out = __builtin_bit_cast(u16, (__bf16)s);
      else *out = s;
    }
    __syncthreads();
  }
}

// dk, dv = the splits' partial sums, in order, and the sinks' -- four elements a thread
template <typename T>
__global__ __launch_bounds__(256) void wattn_sum_kernel(WAttnArgs p) {
  const int d4 = p.D / 4;
  const long total = (long)p.B * p.T * p.Hk * 2 * d4;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const int d = (int)(i % d4) * 4;
    const long row = i / d4;                 // ((b T + j) Hk + hk) 2 + which
    const int which = (int)(row & 1);
    const long k = row >> 1, hk = k % p.Hk, bj = k / p.Hk, b = bj / p.T;
    const int j = (int)(bj - b * p.T);
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (j < seq_len(p, (int)b)) {
      const float* src = p.split + (((b * p.Hk + hk) * p.T + j) * 2 + which) * p.D + d;
      for (int c = 0; c < p.splits; ++c) s += *(const f32x4*)(src + (long)c * p.B * p.Hk * p.T * 2 * p.D);
      if (j < p.sinks) {
        const float* part = p.part + (((b * p.Hk + hk) * p.chunks * p.sinks + j) * 2 + which) * p.D + d;
#pragma unroll 4
        for (int c = 0; c < p.chunks; ++c) s += *(const f32x4*)(part + (long)c * p.sinks * 2 * p.D);
      }
      if (which == 0) s *= p.scale;
    }
    T* out = (T*)(which == 0 ? p.dk : p.dv) + k * p.D + d;
    if constexpr (sizeof(T) == 2) {
      const f32x2 a = {s[0], s[1]}, c = {s[2], s[3]};
      const u32x2 w = {__builtin_bit_cast(unsigned, __builtin_convertvector(a, bf16x2)), __builtin_bit_cast(unsigned, __builtin_convertvector(c, bf16x2))};
      *(u32x2*)out = w;
    } else {
      *(f32x4*)out = s;
    }
  }
}

// ---------------------------------------------------------------------------------------------- host
template <auto Kernel>
int launch(const WAttnArgs& p, long groups, int threads, size_t lds, hipStream_t st) {
  if (groups > 0x7fffffffL) return INDM_E_SHAPE;
  if (indm_lds_optin<Kernel>(lds) != INDM_OK) return INDM_E_LAUNCH;
  hipLaunchKernelGGL((*Kernel), dim3((unsigned)groups), dim3(threads), lds, st, p);
  return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
}

template <typename T, int DP, bool SHARE, bool BWD>
int run_query(WAttnArgs p, hipStream_t st) {
  constexpr int WV = SHARE ? share_waves<T, DP>() : 4;
  p.tiles = cdiv(p.T, SHARE ? 32 : WV * 32);
  return launch<wattn_query_kernel<T, DP, WV, SHARE, BWD>>(p, (long)p.tiles * p.H * p.B, WV * 64,
                                                           (SHARE ? WV : 1) * 4 * (size_t)Geo<T, DP>::TILE, st);
}
// the window's part of all keys, the sinks' from all queries, or both
template <typename T, int DP, bool SHARE, bool SPLIT, int WHO>
int run_key(WAttnArgs p, hipStream_t st) {
  using G = Geo<T, DP>;
  constexpr int WV = SHARE ? share_waves<T, DP>() : 4, OWN = SHARE ? 32 : WV * 32;
  p.tiles = cdiv(p.T, OWN);
  const long heads = (long)p.Hk * p.B, sunk = WHO & SINKS ? cdiv(p.sinks, OWN) * p.chunks * heads : 0;
  if (sunk > 0x7fffffffL) return INDM_E_SHAPE;
  p.sunk = (int)sunk;
  return launch<wattn_key_kernel<T, DP, WV, SHARE, SPLIT, WHO>>(p, sunk + (WHO & KEYS ? (long)p.tiles * (SPLIT ? p.splits : 1) * heads : 0), WV * 64,
                                                                (SHARE ? WV : 1) * 2 * (2 * (size_t)G::TILE + 2 * G::BN * sizeof(float)), st);
}
template <typename T>
int run_sinks(const WAttnArgs& p, hipStream_t st) {
  const long groups = (long)p.B * p.Hk * (((long)p.sinks * 2 * p.D + 63) / 64);
  hipLaunchKernelGGL(wattn_sinks_kernel<T>, dim3((unsigned)(groups < 1 << 20 ? groups : 1 << 20)), dim3(1024), 0, st, p);
  return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
}
template <typename T>
int run_sum(const WAttnArgs& p, hipStream_t st) {
  hipLaunchKernelGGL(wattn_sum_kernel<T>, dim3(ew_grid((long)p.B * p.T * p.Hk * 2 * (p.D / 4), 256)), dim3(256), 0, st, p);
  return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
}

// Up to this many workgroups of four owner blocks, four times as many that share one each do better: half of the compute units would
// idle, and a shared block takes a quarter of the time (2 x 1021 fp32 tokens, 4 heads of 40, 64 workgroups of four: forward 26 us, shared
// 12 us).
constexpr long SHARE_BELOW = 128;
// How the work is laid out, from the sizes alone (the scratch is sized by the same rules).
struct Plan {
  int chunks, splits;   // workgroups that share a sink block's queries (0: the sinks reach nothing), and a key block's
  bool share;           // a key block's wavefronts share 32 keys
  bool apart;           // the sinks' workgroups are a launch of their own (and share 32 keys)
};
inline Plan plan_keys(int tile, int B, int T, int H, int Hk, int left, int right, int sinks, int causal) {
  Plan r = {0, 1, false, false};
  // few key blocks: share each one's queries among workgroups, as long as that leaves each about four tiles of 64 (of all heads of the group)
  const long blocks = (long)cdiv(T, 128) * Hk * B, group = H / Hk;
  const long reach = (long)(left < T ? left : T) + (causal ? 0 : (right < T ? right : T)) + 128, span = reach < T ? reach : T;
  if (blocks < 384) {
    const long tiles = group * cdiv(span, 64);
    long s = (512 + blocks - 1) / blocks;
    if (s > tiles / 4) s = tiles / 4;
    r.splits = s < 1 ? 1 : (int)s;
    r.share = blocks * r.splits <= SHARE_BELOW;
  }
  // Do the sinks reach queries outside of the window?  Then all queries of a block of them are shared by so many workgroups that a
  // wavefront which streams by itself has one tile and a workgroup that streams together eight, up to one or two a compute unit: 256
  // partial sums of 32 sinks or 512 of 128, 8 or 64 MB at 128 entries.  More blocks of sinks than that have one workgroup each, and the
  // partial sums then are as large as two fp32 copies of the sinks' dk and dv (one, where key blocks are split).  Where the key blocks
  // leave the chip room, these workgroups follow them in the same launch (the sinks' and the keys' part and the last sums: 5 x 1543
  // tokens, 8 heads of 128 on 2: 106 us together, 120 apart; 2 x 1021 fp32 tokens, 4 heads of 40: 29 us either way, a launch less); where
  // they fill it, it is a launch before (8 x 4096 tokens, 4 heads of 64: 103 us apart, 109 together).
  if (sinks > 0 && (T - 1 > left || (!causal && sinks - 1 > right))) {
    r.apart = r.splits == 1 && !r.share;
    const bool alone = r.share || r.apart;
    const long rows = (long)B * Hk * cdiv(sinks, alone ? 32 : 128), tiles = group * cdiv(T, tile), mine = alone ? 4 : 8, most = alone ? 256 : 512;
    long c = (tiles + mine - 1) / mine;
    if (c > most / rows) c = most / rows;
    r.chunks = (int)(c < 1 ? 1 : c);
  }
  return r;
}
inline long part_floats(const Plan& plan, int B, int Hk, int sinks, int D) {
  return plan.chunks == 0 ? 0 : (long)B * Hk * (plan.chunks + (plan.splits > 1 ? 0 : 1)) * sinks * 2 * D;
}
inline bool share_queries(int B, int T, int H) { return (long)cdiv(T, 128) * H * B <= SHARE_BELOW; }

#define WA_DISPATCH(CALL)                 \
  if (p.D <= 32) return CALL(32);         \
  if (p.D <= 48) return CALL(48);         \
  if (p.D <= 64) return CALL(64);         \
  if (p.D <= 80) return CALL(80);         \
  if (p.D <= 96) return CALL(96);         \
  return CALL(128);

template <typename T>
int check(const WAttnArgs& p, const long* strides) {
  if (p.B < 0 || p.T < 0 || p.T > (1 << 28) || p.H <= 0 || p.Hk <= 0 || p.H % p.Hk || p.D <= 0 || p.D > 128 || p.D % 8) return INDM_E_SHAPE;
  if (p.left < 0 || p.right < 0 || p.sinks < 0 || strides == nullptr || !(p.scale > 0.f && p.scale < 2e38f)) return INDM_E_ARG;   // (p.c is finite)
  if (p.B == 0 || p.T == 0) return INDM_OK;
  if (p.q == nullptr || p.k == nullptr || p.v == nullptr || (((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) & 15)) return INDM_E_ARG;
  for (int i = 0; i < 9; ++i)
    if (strides[i] < 0 || strides[i] % (16 / (long)sizeof(T))) return INDM_E_ARG;
  if (p.qt > MAX_STRIDE || p.kt > MAX_STRIDE || p.vt > MAX_STRIDE || (long)p.H * p.D > MAX_STRIDE) return INDM_E_SHAPE;
  return 1;
}
WAttnArgs pack_args(const void* q, const void* k, const void* v, const long* s, const int* lengths, int B, int T, int H, int Hk, int D,
                    int left, int right, int sinks, int causal, float scale) {
  WAttnArgs p = {};
  p.q = q; p.k = k; p.v = v; p.lengths = lengths;
  if (s != nullptr) {
    p.qb = s[0]; p.qt = s[1]; p.qh = s[2]; p.kb = s[3]; p.kt = s[4]; p.kh = s[5]; p.vb = s[6]; p.vt = s[7]; p.vh = s[8];
  }
  p.B = B; p.T = T; p.H = H; p.Hk = Hk; p.D = D; p.causal = causal != 0;
  p.left = left < T ? left : T; p.right = right < T ? right : T; p.sinks = sinks < T ? sinks : T;   // (no further than T: no overflow)
  p.scale = scale; p.c = scale * 1.44269504088896340736f;
  return p;
}

template <typename T>
int fwd(WAttnArgs p, const long* strides, void* o, void* olo, float* lse, hipStream_t st) {
  const int r = check<T>(p, strides);
  if (r <= 0) return r;
  if (o == nullptr || (((uintptr_t)o | (uintptr_t)olo) & 15)) return INDM_E_ARG;
  p.out = o; p.olo = olo; p.lse = lse;
#define WA_FWD(DP) (share_queries(p.B, p.T, p.H) ? run_query<T, DP, true, false>(p, st) : run_query<T, DP, false, false>(p, st))
  WA_DISPATCH(WA_FWD)
}

template <typename T, int DP>
int bwd_dp(const WAttnArgs& p, const Plan& plan, hipStream_t st) {
  int r = share_queries(p.B, p.T, p.H) ? run_query<T, DP, true, true>(p, st) : run_query<T, DP, false, true>(p, st);   // dq; delta for the others
  const bool sinks = p.chunks > 0;
  if (r != INDM_OK || p.dk == nullptr) return r;
  if (sinks && plan.apart) r = run_key<T, DP, true, false, SINKS>(p, st);
  if (r == INDM_OK)
    r = p.splits > 1 ? (plan.share ? run_key<T, DP, true, true, BOTH>(p, st) : run_key<T, DP, false, true, BOTH>(p, st))
                     : (plan.share ? run_key<T, DP, true, false, BOTH>(p, st) : run_key<T, DP, false, false, KEYS>(p, st));
  if (r == INDM_OK && p.splits > 1) r = run_sum<T>(p, st);
  else if (r == INDM_OK && sinks) r = run_sinks<T>(p, st);
  return r;
}
template <typename T>
int bwd(WAttnArgs p, const long* strides, const void* o, const void* olo, const void* dO, const float* lse, void* dq, void* dk, void* dv, float* ws,
        hipStream_t st) {
  const int r = check<T>(p, strides);
  if (r <= 0) return r;
  if ((dk == nullptr) != (dv == nullptr)) return INDM_E_ARG;
  if (dq == nullptr && dk == nullptr) return INDM_OK;
  if (o == nullptr || dO == nullptr || lse == nullptr || ws == nullptr ||
      (((uintptr_t)o | (uintptr_t)olo | (uintptr_t)dO | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)ws) & 15)) return INDM_E_ARG;
  p.o = o; p.olo = const_cast<void*>(olo); p.dO = dO; p.lse = const_cast<float*>(lse); p.dq = dq; p.dk = dk; p.dv = dv;
  p.delta = ws;
  const Plan plan = plan_keys(Geo<T, 32>::BN, p.B, p.T, p.H, p.Hk, p.left, p.right, p.sinks, p.causal);
  p.chunks = plan.chunks;
  p.splits = plan.splits;
  p.part = ws + ((long)p.B * p.H * p.T + 3) / 4 * 4;
  p.split = p.part + part_floats(plan, p.B, p.Hk, p.sinks, p.D);
#define WA_BWD(DP) bwd_dp<T, DP>(p, plan, st)
  WA_DISPATCH(WA_BWD)
}

}  // namespace

INDM_API int indm_wattn_fwd_f32(const float* q, const float* k, const float* v, const long* strides, float* o, void*, float* lse,
                                const int* lengths, int B, int T, int H, int Hk, int D, int left, int right, int sinks, int causal,
                                float scale, void* stream) {
  return fwd<float>(pack_args(q, k, v, strides, lengths, B, T, H, Hk, D, left, right, sinks, causal, scale), strides, o, nullptr, lse,
                    (hipStream_t)stream);
}
INDM_API int indm_wattn_fwd_bf16(const void* q, const void* k, const void* v, const long* strides, void* o, void* o_lo, float* lse,
                                 const int* lengths, int B, int T, int H, int Hk, int D, int left, int right, int sinks, int causal,
                                 float scale, void* stream) {
  return fwd<u16>(pack_args(q, k, v, strides, lengths, B, T, H, Hk, D, left, right, sinks, causal, scale), strides, o, o_lo, lse,
                  (hipStream_t)stream);
}

INDM_API long indm_wattn_bwd_ws_floats(int B, int T, int H, int Hk, int D, int left, int right, int sinks, int causal) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0 || left < 0 || right < 0 || sinks < 0) return 0;
  sinks = sinks < T ? sinks : T;
  left = left < T ? left : T;
  right = right < T ? right : T;
  long most = 0;
  for (int tile = 32; tile <= 64; tile *= 2) {   // (whichever type needs more)
    const Plan plan = plan_keys(tile, B, T, H, Hk, left, right, sinks, causal != 0);
    const long n = part_floats(plan, B, Hk, sinks, D) + (plan.splits > 1 ? (long)plan.splits * B * Hk * T * 2 * D : 0);
    most = n > most ? n : most;
  }
  return ((long)B * H * T + 3) / 4 * 4 + most;
}
INDM_API int indm_wattn_bwd_f32(const float* q, const float* k, const float* v, const long* strides, const float* o, const void*,
                                const float* dO, const float* lse, const int* lengths, float* dq, float* dk, float* dv, float* ws, int B, int T, int H,
                                int Hk, int D, int left, int right, int sinks, int causal, float scale, void* stream) {
  return bwd<float>(pack_args(q, k, v, strides, lengths, B, T, H, Hk, D, left, right, sinks, causal, scale), strides, o, nullptr, dO, lse, dq,
                    dk, dv, ws, (hipStream_t)stream);
}
INDM_API int indm_wattn_bwd_bf16(const void* q, const void* k, const void* v, const long* strides, const void* o, const void* o_lo,
                                 const void* dO, const float* lse, const int* lengths, void* dq, void* dk, void* dv, float* ws, int B, int T, int H,
                                 int Hk, int D, int left, int right, int sinks, int causal, float scale, void* stream) {
  return bwd<u16>(pack_args(q, k, v, strides, lengths, B, T, H, Hk, D, left, right, sinks, causal, scale), strides, o, o_lo, dO, lse, dq, dk,
                  dv, ws, (hipStream_t)stream);
}

INDM_API int indm_wattn_layout(int elem_bytes, int B, int T, int H, int Hk, int D, int left, int right, int sinks, int causal) {
  if (B <= 0 || T <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0 || left < 0 || right < 0 || sinks < 0 || (elem_bytes != 2 && elem_bytes != 4)) return INDM_E_SHAPE;
  const Plan plan = plan_keys(elem_bytes == 2 ? Geo<u16, 32>::BN : Geo<float, 32>::BN, B, T, H, Hk, left < T ? left : T, right < T ? right : T,
                              sinks < T ? sinks : T, causal != 0);
  return (share_queries(B, T, H) ? 1 : 0) | (plan.share ? 2 : 0) | (plan.apart ? 4 : 0) | plan.splits << 4 | plan.chunks << 16;
}
