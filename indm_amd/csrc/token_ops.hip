// Row- and element-wise operators of a block over tokens ([..., C] rows, C contiguous), fp32 or bf16 in HBM, fp32 arithmetic:
//   * layer norm forward / backward with the reduction of the weight's and the bias' gradient
//   * dropout from a Philox counter: the mask is a function of (seed, element), never stored
//   * rotary positions over several axes
// All three are HBM-bound: every tensor is read once and written once, in 16-byte accesses.  A row (or a tensor) need not start
// on 16 bytes: the vector types below carry their element's alignment, gfx950 takes such an access as one instruction, and only
// the last partial vector of a row goes element by element.
#include "indm_common.h"

namespace {

typedef unsigned u32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x2t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ unsigned short to_bits16(float v) {
  const __bf16 h = (__bf16)v;   // round to nearest even
  return __builtin_bit_cast(unsigned short, h);
}

// V elements of type T (16 bytes) <-> V floats
template <typename T> struct Row;
template <> struct Row<float> {
  static constexpr int V = 4;
  typedef u32x4a4 raw;
  static __device__ __forceinline__ raw load(const float* p) { return *(const u32x4a4*)p; }
  static __device__ __forceinline__ void unpack(const raw& w, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    raw w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
    *(u32x4a4*)p = w;
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <> struct Row<unsigned short> {   // bf16
  static constexpr int V = 8;
  typedef u32x4a2 raw;
  static __device__ __forceinline__ raw load(const unsigned short* p) { return *(const u32x4a2*)p; }
  static __device__ __forceinline__ void unpack(const raw& w, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(unsigned short* p, const float (&v)[8]) {
    const indm_bf16x8 h = indm_pack_bf16x8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
    *(u32x4a2*)p = __builtin_bit_cast(u32x4a2, h);
  }
  static __device__ __forceinline__ float get(const unsigned short* p) { return __uint_as_float((unsigned)*p << 16); }
  static __device__ __forceinline__ void put(unsigned short* p, float v) { *p = to_bits16(v); }
};

// the vector at p, of which n elements (any n) exist; the others read as 0
template <typename T>
__device__ __forceinline__ void load_part(const T* p, int n, float (&v)[Row<T>::V]) {
  if (n >= Row<T>::V) {
    Row<T>::unpack(Row<T>::load(p), v);
  } else {
#pragma unroll
    for (int i = 0; i < Row<T>::V; ++i) v[i] = i < n ? Row<T>::get(p + i) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_part(T* p, int n, const float (&v)[Row<T>::V]) {
  if (n >= Row<T>::V) {
    Row<T>::store(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < Row<T>::V; ++i)
      if (i < n) Row<T>::put(p + i, v[i]);
  }
}
// V fp32 parameters
template <int V>
__device__ __forceinline__ void load_param(const float* p, int n, float fill, float (&v)[V]) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = fill;
  } else if (n >= V) {
#pragma unroll
    for (int h = 0; h < V; h += 4) {
      const u32x4a4 w = *(const u32x4a4*)(p + h);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[h + i] = __uint_as_float(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}

// ------------------------------------------------------------------------------------------------ layer norm
// A team of L lanes owns a row and keeps it in registers (NV vectors a lane), so the statistics are the two-pass ones -- the
// mean, then the sum of squared differences from it -- and x is read from HBM once.  L < 64: several rows a wavefront.
// Sum over the team; every lane gets it.  L > 64: the team is the whole workgroup.
template <int L>
__device__ __forceinline__ float team_sum(float v, float* sh) {
  if constexpr (L <= 64) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
  } else {
    return block_sum(v, sh);
  }
}

// y = (x - mean) rstd gamma + beta;  R rows of C, x's rows ldx elements apart.  RPT rows a team at once: their loads are all in
// flight together and gamma / beta are fetched once for all of them.
template <typename T, int L, int NV, int RPT>
__global__ __launch_bounds__(L > 256 ? L : 256) void layernorm_fwd_kernel(const T* __restrict__ x, long ldx,
                                                                           const float* __restrict__ gamma,
                                                                           const float* __restrict__ beta, T* __restrict__ y,
                                                                           float* __restrict__ mean, float* __restrict__ rstd,
                                                                           long R, int C, float eps) {
  constexpr int V = Row<T>::V, TEAMS = L > 256 ? 1 : 256 / L;
  __shared__ float sh[16];
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const long r0 = (long)blockIdx.x * (TEAMS * RPT) + team;
  float v[RPT][NV][V];
#pragma unroll
  for (int k = 0; k < RPT; ++k) {
    const long r = r0 + k * TEAMS;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * V;
      load_part<T>(x + r * ldx + c, r < R ? C - c : 0, v[k][j]);
    }
  }
  float m[RPT], rs[RPT];
  const float inv = 1.f / (float)C;
#pragma unroll
  for (int k = 0; k < RPT; ++k) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s += v[k][j][i];
    m[k] = team_sum<L>(s, sh) * inv;
  }
#pragma unroll
  for (int k = 0; k < RPT; ++k) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int n = C - (j * L + lane) * V;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][j][i] -= m[k];
        s += i < n ? v[k][j][i] * v[k][j][i] : 0.f;
      }
    }
    rs[k] = 1.f / sqrtf(team_sum<L>(s, sh) * inv + eps);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * L + lane) * V, n = C - c;
    float g[V], b[V];
    load_param<V>(gamma == nullptr ? nullptr : gamma + c, n, 1.f, g);
    load_param<V>(beta == nullptr ? nullptr : beta + c, n, 0.f, b);
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const long r = r0 + k * TEAMS;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = v[k][j][i] * rs[k] * g[i] + b[i];
      store_part<T>(y + r * C + c, r < R ? n : 0, o);
    }
  }
  if (mean != nullptr && lane == 0) {
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const long r = r0 + k * TEAMS;
      if (r < R) {
        mean[r] = m[k];
        rstd[r] = rs[k];
      }
    }
  }
}

// dx = rstd (h - mean(h) - xh mean(h xh)),  h = dy gamma,  xh = (x - mean) rstd;  per-workgroup partial sums of
// dgamma = sum dy xh and dbeta = sum dy in registers over the workgroup's rows, folded over its teams in a fixed order and
// written to part[workgroup][2][C] (layernorm_param_kernel adds those up: no atomics, the same bits every time).
template <typename T, int L, int NV>
__global__ __launch_bounds__(L > 256 ? L : 256) void layernorm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                           long ldx, const float* __restrict__ gamma,
                                                                           const float* __restrict__ mean,
                                                                           const float* __restrict__ rstd, T* __restrict__ dx,
                                                                           float* __restrict__ part, long R, int C) {
  constexpr int V = Row<T>::V, TEAMS = L > 256 ? 1 : 256 / L;
  extern __shared__ float fold[];   // [2][C] when part is wanted and several teams share the workgroup
  __shared__ float sh[16];
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const float inv = 1.f / (float)C;
  float g[NV][V], dg[NV][V], db[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * L + lane) * V;
    load_param<V>(gamma == nullptr ? nullptr : gamma + c, C - c, 1.f, g[j]);
#pragma unroll
    for (int i = 0; i < V; ++i) dg[j][i] = db[j][i] = 0.f;
  }
  const long step = (long)gridDim.x * TEAMS;
  // (the loop's trip count is the same for every team of a workgroup: team_sum's barriers are reached by all)
  for (long rb = (long)blockIdx.x * TEAMS; rb < R; rb += step) {
    const long r = rb + team;
    const bool live = r < R;
    float d[NV][V], xh[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * V;
      load_part<T>(x + r * ldx + c, live ? C - c : 0, xh[j]);
      load_part<T>(dy + r * C + c, live ? C - c : 0, d[j]);
    }
    const float m = live ? mean[r] : 0.f, rs = live ? rstd[r] : 0.f;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        xh[j][i] = (xh[j][i] - m) * rs;   // (places behind the row have d = 0: they add nothing below)
        const float h = d[j][i] * g[j][i];
        dg[j][i] += d[j][i] * xh[j][i];
        db[j][i] += d[j][i];
        s1 += h;
        s2 += h * xh[j][i];
      }
    s1 = team_sum<L>(s1, sh) * inv;
    s2 = team_sum<L>(s2, sh) * inv;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * V;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = rs * (d[j][i] * g[j][i] - s1 - xh[j][i] * s2);
      store_part<T>(dx + r * C + c, live ? C - c : 0, o);
    }
  }
  if (part == nullptr) return;
  float* out = part + (long)blockIdx.x * 2 * C;
  if constexpr (TEAMS == 1) {   // one row at a time: each column has its one owner
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * L + lane) * V;
#pragma unroll
      for (int h = 0; h < V; h += 4) {
        const float a[4] = {dg[j][h], dg[j][h + 1], dg[j][h + 2], dg[j][h + 3]};
        const float b[4] = {db[j][h], db[j][h + 1], db[j][h + 2], db[j][h + 3]};
        store_part<float>(out + c + h, C - c - h, a);
        store_part<float>(out + C + c + h, C - c - h, b);
      }
    }
    return;
  }
  for (int t = 0; t < TEAMS; ++t) {
    if (team == t) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = (j * L + lane) * V + i;
          if (c < C) {
            fold[c] = t == 0 ? dg[j][i] : fold[c] + dg[j][i];
            fold[C + c] = t == 0 ? db[j][i] : fold[C + c] + db[j][i];
          }
        }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < 2 * C; c += blockDim.x) out[c] = fold[c];
}

// out[c] = sum over the nb workgroups of part[b][c], c < 2 C (dgamma | dbeta): 32 columns x 32 runs of workgroups
__global__ __launch_bounds__(1024) void layernorm_param_kernel(const float* __restrict__ part, float* __restrict__ dgamma,
                                                                float* __restrict__ dbeta, int nb, int C) {
  __shared__ float sh[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < 2 * C) {
#pragma unroll 8
    for (int b = ty; b < nb; b += 32) s += part[(long)b * 2 * C + c];
  }
  sh[ty][tx] = s;
  __syncthreads();
  s = sh[tx][ty];   // lane tx of row ty: the partial sum of run tx of column ty
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  const int co = blockIdx.x * 32 + ty;
  if (tx == 0 && co < 2 * C) {
    float* out = co < C ? dgamma : dbeta;
    if (out != nullptr) out[co < C ? co : co - C] = s;
  }
}

template <typename T> constexpr int ln_max_c() { return 4096 * Row<T>::V; }   // 1024 lanes x 4 vectors

// teams (rows in flight) of a workgroup for rows of C elements, V a vector
inline int ln_teams(int C, int V) {
  const int n = cdiv(C, V);
  return n <= 16 ? 16 : n <= 32 ? 8 : n <= 256 ? 4 : 1;
}
// workgroups of the backward pass: enough to fill the chip, but no more than keeps the partial sums small next to the rows
inline int ln_bwd_blocks(long R, int C, int V) {
  const int teams = ln_teams(C, V);
  const long rows = (R + teams - 1) / teams;
  long nb = rows / 4;
  if (nb > 1024) nb = 1024;
  if (nb < 256) nb = 256;
  return (int)(nb < rows ? nb : rows);
}

template <typename T, int L, int NV>
int launch_ln_fwd(const T* x, long ldx, const float* gamma, const float* beta, T* y, float* mean, float* rstd, long R, int C,
                  float eps, hipStream_t st) {
  constexpr int BLOCK = L > 256 ? L : 256, TEAMS = BLOCK / L, RPT = NV == 1 ? 4 : NV == 2 && L <= 256 ? 2 : 1;
  if (RPT > 1 && R >= 512L * TEAMS * RPT) {
    const long nb = (R + TEAMS * RPT - 1) / (TEAMS * RPT);
    if (nb > 0x7fffffffL) return INDM_E_SHAPE;
    hipLaunchKernelGGL((layernorm_fwd_kernel<T, L, NV, RPT>), dim3((unsigned)nb), dim3(BLOCK), 0, st, x, ldx, gamma, beta, y, mean,
                       rstd, R, C, eps);
  } else {
    const long nb = (R + TEAMS - 1) / TEAMS;
    if (nb > 0x7fffffffL) return INDM_E_SHAPE;
    hipLaunchKernelGGL((layernorm_fwd_kernel<T, L, NV, 1>), dim3((unsigned)nb), dim3(BLOCK), 0, st, x, ldx, gamma, beta, y, mean,
                       rstd, R, C, eps);
  }
  return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
}

template <typename T, int L, int NV>
int launch_ln_bwd(const T* dy, const T* x, long ldx, const float* gamma, const float* mean, const float* rstd, T* dx, float* dgamma,
                  float* dbeta, float* part, long R, int C, hipStream_t st) {
  constexpr int BLOCK = L > 256 ? L : 256;
  const int nb = ln_bwd_blocks(R, C, Row<T>::V);
  const bool params = dgamma != nullptr || dbeta != nullptr;
  const size_t lds = params && L < 256 ? 2 * (size_t)C * sizeof(float) : 0;   // (at most 2 x 2048 floats: four teams of 64 lanes)
  hipLaunchKernelGGL((layernorm_bwd_kernel<T, L, NV>), dim3(nb), dim3(BLOCK), lds, st, dy, x, ldx, gamma, mean, rstd, dx,
                     params ? part : nullptr, R, C);
  if (hipGetLastError() != hipSuccess) return INDM_E_LAUNCH;
  if (params) {
    hipLaunchKernelGGL(layernorm_param_kernel, dim3(cdiv(2L * C, 32)), dim3(1024), 0, st, part, dgamma, dbeta, nb, C);
    if (hipGetLastError() != hipSuccess) return INDM_E_LAUNCH;
  }
  return INDM_OK;
}

// the team and its vectors a lane: the fewest lanes that hold the row (ln_teams follows the same steps)
#define LN_DISPATCH(CALL)                                  \
  const int n = cdiv(C, Row<T>::V);                        \
  if (n <= 16) return CALL(16, 1);                         \
  if (n <= 32) return CALL(32, 1);                         \
  if (n <= 64) return CALL(64, 1);                         \
  if (n <= 128) return CALL(64, 2);                        \
  if (n <= 256) return CALL(64, 4);                        \
  if (n <= 512) return CALL(256, 2);                       \
  if (n <= 1024) return CALL(256, 4);                      \
  if (n <= 2048) return CALL(1024, 2);                     \
  return CALL(1024, 4);

template <typename T>
int ln_fwd(const T* x, long ldx, const float* gamma, const float* beta, T* y, float* mean, float* rstd, long R, int C, float eps,
           hipStream_t st) {
  if (R < 0 || C <= 0 || C > ln_max_c<T>() || ldx < 0) return INDM_E_SHAPE;
  if ((mean == nullptr) != (rstd == nullptr)) return INDM_E_ARG;
  if (R == 0) return INDM_OK;
  if (x == nullptr || y == nullptr) return INDM_E_ARG;
#define LN_FWD(L, NV) launch_ln_fwd<T, L, NV>(x, ldx, gamma, beta, y, mean, rstd, R, C, eps, st)
  LN_DISPATCH(LN_FWD)
#undef LN_FWD
}

template <typename T>
int ln_bwd(const T* dy, const T* x, long ldx, const float* gamma, const float* mean, const float* rstd, T* dx, float* dgamma,
           float* dbeta, float* ws, long R, int C, hipStream_t st) {
  if (R < 0 || C <= 0 || C > ln_max_c<T>() || ldx < 0) return INDM_E_SHAPE;
  if (R == 0) {   // the gradients of no rows are zeros
    if (dgamma == nullptr && dbeta == nullptr) return INDM_OK;
    hipLaunchKernelGGL(layernorm_param_kernel, dim3(cdiv(2L * C, 32)), dim3(1024), 0, st, ws, dgamma, dbeta, 0, C);
    return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
  }
  if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr || dx == nullptr) return INDM_E_ARG;
  if ((dgamma != nullptr || dbeta != nullptr) && ws == nullptr) return INDM_E_ARG;
#define LN_BWD(L, NV) launch_ln_bwd<T, L, NV>(dy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, ws, R, C, st)
  LN_DISPATCH(LN_BWD)
#undef LN_BWD
}

// ------------------------------------------------------------------------------------------------ dropout
// factors of the 4 elements of flat quad idx4: the mask of the fused GroupNorm + dropout (norm_act.hip: same seed, same mask)
__device__ __forceinline__ void keep4(uint64_t seed, uint64_t idx4, float p, bool (&k)[4]) {
  const uint4 r = philox4x32(make_uint2((uint32_t)seed, (uint32_t)(seed >> 32)),
                             make_uint4((uint32_t)idx4, (uint32_t)(idx4 >> 32), 0u, 0u));
  k[0] = u32_to_unit(r.x) > p;
  k[1] = u32_to_unit(r.y) > p;
  k[2] = u32_to_unit(r.z) > p;
  k[3] = u32_to_unit(r.w) > p;
}

// y = (res) + keep x / (1 - p).  A dropped element is 0 whatever x holds there (also an infinity or a NaN).
template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, T* y, long n,   // (y may be x or res)
                                                      float p, float factor, uint64_t seed, const uint64_t* seed_dev) {
  constexpr int V = Row<T>::V;
  if (seed_dev) seed += *seed_dev;
  const long nv = (n + V - 1) / V;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < nv; i += (long)gridDim.x * 256) {
    const long at = i * V;
    const int left = n - at < V ? (int)(n - at) : V;
    float v[V], w[V], o[V];
    load_part<T>(x + at, left, v);
    if constexpr (RES) load_part<T>(res + at, left, w);
#pragma unroll
    for (int h = 0; h < V; h += 4) {
      bool k[4];
      keep4(seed, (uint64_t)i * (V / 4) + h / 4, p, k);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[h + e] = k[e] ? v[h + e] * factor : 0.f;
        if constexpr (RES) o[h + e] += w[h + e];
      }
    }
    store_part<T>(y + at, left, o);
  }
}

template <typename T>
int dropout(const T* x, const T* res, T* y, long n, float p, uint64_t seed, const uint64_t* seed_dev, hipStream_t st) {
  if (n < 0) return INDM_E_SHAPE;
  if (!(p >= 0.f && p <= 1.f)) return INDM_E_ARG;
  if (n == 0) return INDM_OK;
  if (x == nullptr || y == nullptr) return INDM_E_ARG;
  const float factor = p < 1.f ? 1.f / (1.f - p) : 0.f;   // p = 1 drops every element (no uniform of (0, 1] is larger)
  const int grid = ew_grid((n + Row<T>::V - 1) / Row<T>::V, 256);
  if (res != nullptr)
    hipLaunchKernelGGL((dropout_kernel<T, true>), dim3(grid), dim3(256), 0, st, x, res, y, n, p, factor, seed, seed_dev);
  else
    hipLaunchKernelGGL((dropout_kernel<T, false>), dim3(grid), dim3(256), 0, st, x, res, y, n, p, factor, seed, seed_dev);
  return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
}

// ------------------------------------------------------------------------------------------------ rotary positions
// A head's first sum(sections) entries are rotated in pairs (a, b) -> (a cos - b sin, b cos + a sin) by the angle
// pos[token][axis of the pair's section] * freqs[pair]; the rest passes through.  A pair of a section of n entries at offset o is
// (o + j, o + n/2 + j), or (o + 2 j, o + 2 j + 1) when interleaved.  The angle is formed and reduced to a quadrant in 64 bits
// (a far position times a frequency needs more than fp32's 24 bits), its sine and cosine on [-pi/4, pi/4] in fp32.
// A thread owns one vector (V entries) of a token's heads: it computes their sines once and applies them to HPT heads of q and k.
constexpr int ROT_AXES = 8;

struct RotArgs {
  const void* x[2];   // q, k: [B, T, heads, D] with these strides (elements), D contiguous
  void* y[2];         // the same, contiguous
  long sb[2], st[2], sh[2];
  int heads[2];
  const void* pos;    // [T, A] or [B, T, A]
  long pos_sb;        // 0: shared by the batch
  const double* freqs;
  long B, T;
  int D, axes, hpt, hchunks;
  int end[ROT_AXES];  // end offset of each section
  float sign;         // -1: the inverse rotation (the backward pass)
};

template <typename T, typename P, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs a) {
  constexpr int V = Row<T>::V;
  const int nvec = (a.D + V - 1) / V;
  const long per = (long)nvec * a.hchunks;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.B * a.T * per) return;
  const long tok = i / per;
  const int rest = (int)(i - tok * per);
  const int hc = rest / nvec, d0 = (rest - hc * nvec) * V;
  const long b = tok / a.T, t = tok - b * a.T;
  const int left = a.D - d0 < V ? a.D - d0 : V;
  const P* pos = (const P*)a.pos + b * a.pos_sb + t * a.axes;

  float c[V], s[V];
  int mate[V];        // offset of the pair's other entry, 0: passes through
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int d = d0 + e;
    int ax = -1, start = 0, from = 0, size = 0;
    for (int k = 0; k < a.axes; ++k) {
      if (ax < 0 && d < a.end[k]) {
        ax = k;
        start = from;
        size = a.end[k] - from;
      }
      from = a.end[k];
    }
    c[e] = 1.f;
    s[e] = 0.f;
    mate[e] = 0;
    if (ax >= 0 && e < left) {
      const int in = d - start, half = size / 2;
      const bool second = INTER ? (in & 1) : in >= half;
      const int j = INTER ? in >> 1 : second ? in - half : in;
      mate[e] = INTER ? (second ? -1 : 1) : second ? -half : half;
      const double quarter = (double)pos[ax] * a.freqs[start / 2 + j] * 0.63661977236758134308;   // angle in units of pi / 2
      const double q = __builtin_rint(quarter);
      float sn, cs;
      indm_sincos_quadrant((float)((quarter - q) * 1.57079632679489661923), (int)(q - 4.0 * __builtin_floor(q * 0.25)), sn, cs);
      c[e] = cs;
      s[e] = (second ? sn : -sn) * a.sign;
    }
  }
  // the mates of a whole vector are a whole vector when all lie equally far: one more (cached) vector load
  bool same = left == V;
#pragma unroll
  for (int e = 1; e < V; ++e) same = same && mate[e] == mate[0];

  const int total = a.heads[0] + a.heads[1];
  const int h0 = hc * a.hpt, h1 = h0 + a.hpt < total ? h0 + a.hpt : total;
#pragma unroll 4
  for (int hh = h0; hh < h1; ++hh) {
    const int w = hh < a.heads[0] ? 0 : 1;
    const int h = w == 0 ? hh : hh - a.heads[0];
    const T* x = (const T*)a.x[w] + b * a.sb[w] + t * a.st[w] + h * a.sh[w] + d0;
    T* y = (T*)a.y[w] + ((b * a.T + t) * a.heads[w] + h) * a.D + d0;
    float v[V], o[V];
    load_part<T>(x, left, v);
    if constexpr (INTER) {   // the sections are even: both entries of a pair are in this vector
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = mate[e] == 0 ? v[e] : v[e] * c[e] + v[e ^ 1] * s[e];
    } else if (same) {
      if (mate[0] == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = v[e];
      } else {
        float u[V];
        Row<T>::unpack(Row<T>::load(x + mate[0]), u);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = v[e] * c[e] + u[e] * s[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = mate[e] == 0 ? v[e] : v[e] * c[e] + Row<T>::get(x + e + mate[e]) * s[e];
    }
    store_part<T>(y, left, o);
  }
}

template <typename T>
int rotary(const T* q, const T* k, T* yq, T* yk, const long* strides, int B, long Tn, int H, int Hk, int D, const void* pos,
           int pos_type, long pos_sb, const double* freqs, const int* sections, int axes, int interleaved, int inverse,
           hipStream_t st) {
  if (B < 0 || Tn < 0 || H < 0 || Hk < 0 || D <= 0 || axes <= 0 || axes > ROT_AXES) return INDM_E_SHAPE;
  if (strides == nullptr || sections == nullptr || pos_type < 0 || pos_type > 2) return INDM_E_ARG;
  RotArgs a = {};
  int at = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] <= 0 || (sections[i] & 1) || sections[i] > D - at) return INDM_E_SHAPE;
    a.end[i] = at += sections[i];
  }
  if (B == 0 || Tn == 0 || H + Hk == 0) return INDM_OK;
  if ((H > 0 && (q == nullptr || yq == nullptr)) || (Hk > 0 && (k == nullptr || yk == nullptr)) || pos == nullptr || freqs == nullptr)
    return INDM_E_ARG;
  a.x[0] = q; a.x[1] = k; a.y[0] = yq; a.y[1] = yk;
  for (int w = 0; w < 2; ++w) {
    a.sb[w] = strides[3 * w]; a.st[w] = strides[3 * w + 1]; a.sh[w] = strides[3 * w + 2];
  }
  a.heads[0] = H; a.heads[1] = Hk;
  a.pos = pos; a.pos_sb = pos_sb; a.freqs = freqs; a.B = B; a.T = Tn; a.D = D; a.axes = axes;
  a.sign = inverse ? -1.f : 1.f;
  // heads a thread: all of them when the tokens fill the chip, else fewer
  const int nvec = cdiv(D, Row<T>::V), total = H + Hk;
  a.hpt = total;
  while (a.hpt > 1 && (long)B * Tn * nvec * cdiv(total, a.hpt) < 256L * 1024) a.hpt = (a.hpt + 1) / 2;
  a.hchunks = cdiv(total, a.hpt);
  const long nb = ((long)B * Tn * nvec * a.hchunks + 255) / 256;
  if (nb > 0x7fffffffL) return INDM_E_SHAPE;
#define ROT_LAUNCH(P)                                                                                             \
  do {                                                                                                            \
    if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, P, true>), dim3((unsigned)nb), dim3(256), 0, st, a);    \
    else hipLaunchKernelGGL((rotary_kernel<T, P, false>), dim3((unsigned)nb), dim3(256), 0, st, a);               \
  } while (0)
  if (pos_type == 0) ROT_LAUNCH(int);
  else if (pos_type == 1) ROT_LAUNCH(float);
  else ROT_LAUNCH(long);
#undef ROT_LAUNCH
  return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
}

}  // namespace

INDM_API int indm_layernorm_fwd_f32(const float* x, long ldx, const float* gamma, const float* beta, float* y, float* mean,
                                    float* rstd, long R, int C, float eps, void* stream) {
  return ln_fwd<float>(x, ldx, gamma, beta, y, mean, rstd, R, C, eps, (hipStream_t)stream);
}
INDM_API int indm_layernorm_fwd_bf16(const void* x, long ldx, const float* gamma, const float* beta, void* y, float* mean,
                                     float* rstd, long R, int C, float eps, void* stream) {
  return ln_fwd<unsigned short>((const unsigned short*)x, ldx, gamma, beta, (unsigned short*)y, mean, rstd, R, C, eps,
                                (hipStream_t)stream);
}

INDM_API long indm_layernorm_bwd_ws_floats(long R, int C, int elem_bytes) {
  if (R <= 0 || C <= 0 || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  return (long)ln_bwd_blocks(R, C, 16 / elem_bytes) * 2 * C;
}
INDM_API int indm_layernorm_bwd_f32(const float* dy, const float* x, long ldx, const float* gamma, const float* mean,
                                    const float* rstd, float* dx, float* dgamma, float* dbeta, float* ws, long R, int C,
                                    void* stream) {
  return ln_bwd<float>(dy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, ws, R, C, (hipStream_t)stream);
}
INDM_API int indm_layernorm_bwd_bf16(const void* dy, const void* x, long ldx, const float* gamma, const float* mean,
                                     const float* rstd, void* dx, float* dgamma, float* dbeta, float* ws, long R, int C,
                                     void* stream) {
  return ln_bwd<unsigned short>((const unsigned short*)dy, (const unsigned short*)x, ldx, gamma, mean, rstd, (unsigned short*)dx,
                                dgamma, dbeta, ws, R, C, (hipStream_t)stream);
}

INDM_API int indm_dropout_f32(const float* x, const float* res, float* y, long n, float p, unsigned long long seed,
                              const void* seed_dev, void* stream) {
  return dropout<float>(x, res, y, n, p, seed, (const uint64_t*)seed_dev, (hipStream_t)stream);
}
INDM_API int indm_dropout_bf16(const void* x, const void* res, void* y, long n, float p, unsigned long long seed,
                               const void* seed_dev, void* stream) {
  return dropout<unsigned short>((const unsigned short*)x, (const unsigned short*)res, (unsigned short*)y, n, p, seed,
                                 (const uint64_t*)seed_dev, (hipStream_t)stream);
}

INDM_API int indm_rotary_f32(const float* q, const float* k, float* yq, float* yk, const long* strides, int B, long T, int H, int Hk,
                             int D, const void* pos, int pos_type, long pos_sb, const double* freqs, const int* sections, int axes,
                             int interleaved, int inverse, void* stream) {
  return rotary<float>(q, k, yq, yk, strides, B, T, H, Hk, D, pos, pos_type, pos_sb, freqs, sections, axes, interleaved, inverse,
                       (hipStream_t)stream);
}
INDM_API int indm_rotary_bf16(const void* q, const void* k, void* yq, void* yk, const long* strides, int B, long T, int H, int Hk,
                              int D, const void* pos, int pos_type, long pos_sb, const double* freqs, const int* sections, int axes,
                              int interleaved, int inverse, void* stream) {
  return rotary<unsigned short>((const unsigned short*)q, (const unsigned short*)k, (unsigned short*)yq, (unsigned short*)yk, strides,
                                B, T, H, Hk, D, pos, pos_type, pos_sb, freqs, sections, axes, interleaved, inverse,
                                (hipStream_t)stream);
}
