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
typedef unsigned u32x2t __attribute__((ext_vector_type(2)));

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
__device__ __forceinline__ typename Row<T>::raw load_raw(const T* p, int n) {
  typename Row<T>::raw w = {0u, 0u, 0u, 0u};
  if (n >= Row<T>::V) {
    w = Row<T>::load(p);
  } else if (n > 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        if (i < n) w[i] = __float_as_uint(p[i]);
      } else {
        const unsigned lo = 2 * i < n ? p[2 * i] : 0u, hi = 2 * i + 1 < n ? p[2 * i + 1] : 0u;
        w[i] = lo | hi << 16;
      }
    }
  }
  return w;
}
template <typename T>
__device__ __forceinline__ void load_part(const T* p, int n, float (&v)[Row<T>::V]) {
  Row<T>::unpack(load_raw<T>(p, n), v);
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
// HBM-bound.  131072 rows of 256, bf16: forward 24 us (5.6 TB/s, a copy's rate), backward 39 us (5.1 TB/s) and 4 us for the parameters'
// sums; 4099 rows of 1153, fp32, out of wider rows: 10 us, 16.5 us and 4 us (384 and 512 slots for the 289 vectors of a row, and backward
// four barriers a row); 256 rows: 2.8 us, a launch.  Rows that start on odd bf16
// elements cost the backward pass half its rate (2.4 TB/s: the memory pipe splits those accesses).
// Sum over the team; every lane gets the same bits (each step adds a pair, whichever order).  Within a wavefront all steps are
// vector instructions: lanes 1, 2, then mirrored quads and halves of a row of 16, then rows and halves of the wavefront traded.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  const int i = __float_as_int(v);
  return v + __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xF, 0xF, false));
}
template <int L>
__device__ __forceinline__ float team_sum(float v, float* sh) {
  v = dpp_add<0xB1>(v);    // quad_perm [1, 0, 3, 2]
  v = dpp_add<0x4E>(v);    // quad_perm [2, 3, 0, 1]
  v = dpp_add<0x141>(v);   // row_half_mirror
  v = dpp_add<0x140>(v);   // row_mirror
  if constexpr (L >= 32) {
    const unsigned u = __float_as_uint(v);
    const u32x2t r = __builtin_bit_cast(u32x2t, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (L >= 64) {
    const unsigned u = __float_as_uint(v);
    const u32x2t r = __builtin_bit_cast(u32x2t, __builtin_amdgcn_permlane32_swap(u, u, false, false));
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (L > 64) {   // the team is the whole workgroup
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) v += sh[i];
  }
  return v;
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

// dx = rstd (h - mean(h) - xh mean(h xh)),  h = dy gamma,  xh = (x - mean) rstd  (dx may be NULL);  per-workgroup partial sums of
// dgamma = sum dy xh and dbeta = sum dy in registers over the workgroup's rows, folded over its teams in a fixed order and
// written to part[workgroup][2][C] (layernorm_param_kernel adds those up: no atomics, the same bits every time).
template <typename T, int L, int NV, int RPT>
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
  const long step = (long)gridDim.x * TEAMS * RPT;
  // (the loop's trip count is the same for every team of a workgroup: team_sum's barriers are reached by all)
  for (long rb = (long)blockIdx.x * TEAMS * RPT; rb < R; rb += step) {
    float d[RPT][NV][V], xh[RPT][NV][V], m[RPT], rs[RPT], s1[RPT], s2[RPT];
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const long r = rb + k * TEAMS + team;
      const bool live = r < R;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * L + lane) * V;
        load_part<T>(x + r * ldx + c, live ? C - c : 0, xh[k][j]);
        load_part<T>(dy + r * C + c, live ? C - c : 0, d[k][j]);
      }
      m[k] = live ? mean[r] : 0.f;
      rs[k] = live ? rstd[r] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      s1[k] = s2[k] = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) xh[k][j][i] = (xh[k][j][i] - m[k]) * rs[k];
        const int n = C - (j * L + lane) * V;
        if (n < V) {   // (places behind the row have d = 0, but -m rs may have overflowed there)
#pragma unroll
          for (int i = 0; i < V; ++i) xh[k][j][i] = i < n ? xh[k][j][i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float h = d[k][j][i] * g[j][i];
          dg[j][i] += d[k][j][i] * xh[k][j][i];
          db[j][i] += d[k][j][i];
          s1[k] += h;
          s2[k] += h * xh[k][j][i];
        }
      }
    }
    if (dx == nullptr) continue;   // (the same for all: the parameters' gradients alone are wanted)
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      s1[k] = team_sum<L>(s1[k], sh) * inv;
      s2[k] = team_sum<L>(s2[k], sh) * inv;
    }
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const long r = rb + k * TEAMS + team;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * L + lane) * V;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = rs[k] * (d[k][j][i] * g[j][i] - s1[k] - xh[k][j][i] * s2[k]);
        store_part<T>(dx + r * C + c, r < R ? C - c : 0, o);
      }
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

// The team that owns rows of n vectors.  Forward: the fewest lanes that hold one with 32 elements a lane, so that rows up to 2048
// elements need no barrier (fp32, 4099 rows of 1153: 64 lanes x 6 vectors 10 us, 256 lanes x 2 13 us).  Backward: a lane holds five
// values of each of its columns, so from 128 vectors on fewer of them on more lanes win (fp32, 16384 rows of 2048: 64 lanes x 8 97 us,
// 256 lanes x 2 83 us) -- and below, one wavefront does (fp32, 87381 rows of 384: 64 x 2 83 us, 256 x 1 122 us).
constexpr int LN_MAX_C = 16384;
#define LN_DISPATCH_FWD(CALL)                                    \
  const int n = cdiv(C, Row<T>::V);                              \
  if (n <= 16) return CALL(16, 1);                               \
  if (n <= 32) return CALL(32, 1);                               \
  if (n <= 64) return CALL(64, 1);                               \
  if (n <= 128) return CALL(64, 2);                              \
  if (n <= 192) return CALL(64, 3);                              \
  if (n <= 256) return CALL(64, 4);                              \
  if constexpr (Row<T>::V == 4) {                                \
    if (n <= 384) return CALL(64, 6);                            \
    if (n <= 512) return CALL(64, 8);                            \
    if (n <= 1024) return CALL(256, 4);                          \
    if (n <= 2048) return CALL(1024, 2);                         \
    return CALL(1024, 4);                                        \
  } else {                                                       \
    if (n <= 512) return CALL(256, 2);                           \
    if (n <= 1024) return CALL(256, 4);                          \
    return CALL(1024, 2);                                        \
  }
#define LN_DISPATCH_BWD(CALL)                                    \
  const int n = cdiv(C, Row<T>::V);                              \
  if (n <= 16) return CALL(16, 1);                               \
  if (n <= 32) return CALL(32, 1);                               \
  if (n <= 64) return CALL(64, 1);                               \
  if (n <= 128) return CALL(64, 2);                              \
  if (n <= 256) return CALL(256, 1);                             \
  if (n <= 512) return CALL(256, 2);                             \
  if (n <= 1024) return CALL(512, 2);                            \
  if constexpr (Row<T>::V == 4) {                                \
    if (n <= 2048) return CALL(512, 4);                          \
    return CALL(1024, 4);                                        \
  } else {                                                       \
    return CALL(1024, 2);                                        \
  }

// rows a team takes at once: up to 32 elements a lane in flight
constexpr int ln_rpt(int V, int NV, int L) { return L > 256 ? 1 : NV * V <= 8 ? 4 : NV * V <= 16 ? 2 : 1; }
constexpr int ln_bwd_rpt(int V, int NV, int L) { return L <= 64 && NV * V <= 8 ? 2 : 1; }

// workgroups of the backward pass: enough to fill the chip, but few enough that the partial sums (16 C bytes a workgroup, written and
// read) stay a sixth of the rows' 3 R C elem bytes, from 4096 rows of bf16 or 2048 of fp32 on.  Fewer rows still have up to 256 workgroups, whose
// partial sums may be more than the rows themselves (256 rows of 8192 bf16: 33 MB next to 12.6 MB).
inline int ln_bwd_blocks(long R, int teams, int elem) {
  const long rows = (R + teams - 1) / teams;
  long nb = R * elem / 32;
  if (nb > 1024) nb = 1024;
  if (nb < 256) nb = 256;
  return (int)(nb < rows ? nb : rows);
}
template <typename T, int L, int NV>
int launch_ln_fwd(const T* x, long ldx, const float* gamma, const float* beta, T* y, float* mean, float* rstd, long R, int C,
                  float eps, hipStream_t st) {
  constexpr int BLOCK = L > 256 ? L : 256, TEAMS = BLOCK / L, RPT = ln_rpt(Row<T>::V, NV, L);
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
  constexpr int BLOCK = L > 256 ? L : 256, TEAMS = BLOCK / L, RPT = ln_bwd_rpt(Row<T>::V, NV, L);
  const int nb = ln_bwd_blocks(R, TEAMS, sizeof(T));
  const bool params = dgamma != nullptr || dbeta != nullptr;
  const size_t lds = params && L < 256 ? 2 * (size_t)C * sizeof(float) : 0;   // (at most 2 x 1024 floats: four teams of 64 lanes with 16 elements each)
  if (R >= (long)nb * TEAMS * RPT)
    hipLaunchKernelGGL((layernorm_bwd_kernel<T, L, NV, RPT>), dim3(nb), dim3(BLOCK), lds, st, dy, x, ldx, gamma, mean, rstd, dx,
                       params ? part : nullptr, R, C);
  else
    hipLaunchKernelGGL((layernorm_bwd_kernel<T, L, NV, 1>), dim3(nb), dim3(BLOCK), lds, st, dy, x, ldx, gamma, mean, rstd, dx,
                       params ? part : nullptr, R, C);
  if (hipGetLastError() != hipSuccess) return INDM_E_LAUNCH;
  if (params) {
    hipLaunchKernelGGL(layernorm_param_kernel, dim3(cdiv(2L * C, 32)), dim3(1024), 0, st, part, dgamma, dbeta, nb, C);
    if (hipGetLastError() != hipSuccess) return INDM_E_LAUNCH;
  }
  return INDM_OK;
}

template <typename T>
int ln_fwd(const T* x, long ldx, const float* gamma, const float* beta, T* y, float* mean, float* rstd, long R, int C, float eps,
           hipStream_t st) {
  if (R < 0 || C <= 0 || C > LN_MAX_C || ldx < 0) return INDM_E_SHAPE;
  if ((mean == nullptr) != (rstd == nullptr)) return INDM_E_ARG;
  if (R == 0) return INDM_OK;
  if (x == nullptr || y == nullptr) return INDM_E_ARG;
#define LN_FWD(L, NV) launch_ln_fwd<T, L, NV>(x, ldx, gamma, beta, y, mean, rstd, R, C, eps, st)
  LN_DISPATCH_FWD(LN_FWD)
#undef LN_FWD
}

template <typename T>
int ln_bwd(const T* dy, const T* x, long ldx, const float* gamma, const float* mean, const float* rstd, T* dx, float* dgamma,
           float* dbeta, float* ws, long R, int C, hipStream_t st) {
  if (R < 0 || C <= 0 || C > LN_MAX_C || ldx < 0) return INDM_E_SHAPE;
  if (R == 0) {   // the gradients of no rows are zeros
    if (dgamma == nullptr && dbeta == nullptr) return INDM_OK;
    hipLaunchKernelGGL(layernorm_param_kernel, dim3(cdiv(2L * C, 32)), dim3(1024), 0, st, ws, dgamma, dbeta, 0, C);
    return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
  }
  if (dx == nullptr && dgamma == nullptr && dbeta == nullptr) return INDM_OK;
  if (dy == nullptr || x == nullptr || mean == nullptr || rstd == nullptr) return INDM_E_ARG;
  if ((dgamma != nullptr || dbeta != nullptr) && ws == nullptr) return INDM_E_ARG;
#define LN_BWD(L, NV) launch_ln_bwd<T, L, NV>(dy, x, ldx, gamma, mean, rstd, dx, dgamma, dbeta, ws, R, C, st)
  LN_DISPATCH_BWD(LN_BWD)
#undef LN_BWD
}

template <typename T>
long ln_ws(long R, int C) {
#define LN_WS(L, NV) (long)ln_bwd_blocks(R, L > 256 ? 1 : 256 / L, sizeof(T)) * 2 * C
  LN_DISPATCH_BWD(LN_WS)
#undef LN_WS
}

// ------------------------------------------------------------------------------------------------ dropout
// which of the 4 elements of flat quad idx4 stay: the mask of the fused GroupNorm + dropout (norm_act.hip: same seed, same mask).
// There an element stays when ((word >> 8) + 1) 2^-24 > p, whose left side is exact: that is word >> 8 >= floor(p 2^24) = drop.
// (Each round's products are written as 64-bit ones: one instruction instead of a high and a low half.)
__device__ __forceinline__ void keep4(uint64_t seed, uint64_t idx4, uint32_t drop, bool (&k)[4]) {
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
  uint32_t c0 = (uint32_t)idx4, c1 = (uint32_t)(idx4 >> 32), c2 = 0u, c3 = 0u;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  k[0] = (c0 >> 8) >= drop;
  k[1] = (c1 >> 8) >= drop;
  k[2] = (c2 >> 8) >= drop;
  k[3] = (c3 >> 8) >= drop;
}

// y = (res) + keep x / (1 - p).  A dropped element is 0 whatever x holds there (also an infinity or a NaN).  HBM-bound, with the
// generator's products close behind: 20 of them at a quarter of the rate for every 4 elements, 17 of the 25 us below.  One vector a
// lane, nothing carried over: 2^25 elements of bf16 take 25 us (5.4 TB/s; a loop of 8 vectors a lane 27), with a residual 39 us (5.2
// TB/s; 40), 2^22 + 3 of fp32 6.8 us.  Stores that bypass the caches measured 22 and 30 us on the same tensors again and again, but no
// gain on fresh ones, and the layer norm that reads 128 MB next lost 10 us to them.
template <typename T, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, T* y, long n,   // (y may be x or res)
                                                      uint32_t drop, float factor, uint64_t seed, const uint64_t* seed_dev) {
  constexpr int V = Row<T>::V;
  if (seed_dev) seed += *seed_dev;
  const long i = (long)blockIdx.x * 256 + threadIdx.x, at = i * V;
  const int left = n - at < V ? (int)(n - at) : V;
  float v[V], w[V], o[V];
  load_part<T>(x + at, left, v);
  if constexpr (RES) load_part<T>(res + at, left, w);
#pragma unroll
  for (int h = 0; h < V; h += 4) {
    bool k[4];
    keep4(seed, (uint64_t)i * (V / 4) + h / 4, drop, k);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[h + e] = k[e] ? v[h + e] * factor : 0.f;
      if constexpr (RES) o[h + e] += w[h + e];
    }
  }
  store_part<T>(y + at, left, o);
}

template <typename T>
int dropout(const T* x, const T* res, T* y, long n, float p, uint64_t seed, const uint64_t* seed_dev, hipStream_t st) {
  if (n < 0) return INDM_E_SHAPE;
  if (!(p >= 0.f && p <= 1.f)) return INDM_E_ARG;
  if (n == 0) return INDM_OK;
  if (x == nullptr || y == nullptr) return INDM_E_ARG;
  const float factor = p < 1.f ? 1.f / (1.f - p) : 0.f;   // p = 1 drops every element: word >> 8 < 2^24
  const uint32_t drop = (uint32_t)(p * 16777216.f);
  const long grid = (n + 256L * Row<T>::V - 1) / (256L * Row<T>::V);
  if (grid > 0x7fffffffL) return INDM_E_SHAPE;
  if (res != nullptr)
    hipLaunchKernelGGL((dropout_kernel<T, true>), dim3((unsigned)grid), dim3(256), 0, st, x, res, y, n, drop, factor, seed, seed_dev);
  else
    hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)grid), dim3(256), 0, st, x, res, y, n, drop, factor, seed, seed_dev);
  return hipGetLastError() == hipSuccess ? INDM_OK : INDM_E_LAUNCH;
}

// ------------------------------------------------------------------------------------------------ rotary positions
// A head's first sum(sections) entries are rotated in pairs (a, b) -> (a cos - b sin, b cos + a sin) by the angle
// pos[token][axis of the pair's section] * freqs[pair]; the rest passes through.  A pair of a section of n entries at offset o is
// (o + j, o + n/2 + j), or (o + 2 j, o + 2 j + 1) when interleaved.  The angle is formed and reduced to a quadrant in 64 bits
// (a far position times a frequency needs more than fp32's 24 bits), its sine and cosine on [-pi/4, pi/4] in fp32.
// A workgroup takes tp positions of ts samples that share them: their sines and cosines go to LDS once (one 64-bit angle a thread, not
// one per head and sample).  A head is cut
// into units of one vector (V entries): a unit of a section's first half takes its second half along, so that every entry is loaded
// once; an interleaved section's units hold whole pairs, the rest of the head passes through.  What no unit covers (halves, or a rest,
// that are no multiple of V) goes entry by entry.  Bound by HBM and, half as much, by the angles: 64 x 1024 tokens of 8 heads of 64
// entries (q and k out of a fused product, bf16, 134 MB) take 29 us (4.6 TB/s; a copy of as much 24 us); with every vector loading its
// mates a second time they took 34 us.
constexpr int ROT_AXES = 8, ROT_MAX_D = 4096;

struct RotArgs {
  const void* x[2];   // q, k: [B, T, heads, D] with these strides (elements), D contiguous
  void* y[2];         // the same, contiguous
  long sb[2], st[2], sh[2];
  int heads[2];
  const void* pos;    // [T, A] or [B, T, A]
  const double* freqs;
  long T, S, N;       // tokens of a sample; positions that differ, and the samples that share them: T and B, or B T and 1
  long tiles;         // of positions
  int D, axes, ts, tp, units, loose;   // ts samples at tp positions a workgroup
  int end[ROT_AXES];  // end offset of each section
  float sign;         // -1: the inverse rotation (the backward pass)
};

// the regions that are cut into units: a section's first half, or all that is interleaved; and the rest of the head.  Calls
// f(first entry, entries, first pair, distance of the mates -- 0: passes through) for each.
template <bool INTER, typename F>
__host__ __device__ __forceinline__ void rot_regions(const RotArgs& a, F f) {
  const int sum = a.end[a.axes - 1];
  if (INTER) {
    f(0, sum, 0, 1);
  } else {
    for (int k = 0, from = 0; k < a.axes; from = a.end[k++]) f(from, (a.end[k] - from) >> 1, from >> 1, (a.end[k] - from) >> 1);
  }
  f(sum, a.D - sum, 0, 0);
}

template <typename T, typename P, bool INTER>
__global__ __launch_bounds__(512) void rotary_kernel(RotArgs a) {
    constexpr int V = Row<T>::V, U = 4;   // tokens a lane has in flight
  typedef typename Row<T>::raw raw;
  // [tp][pairs] (cos, sin); a token's offsets in q and k, its index and the row of its sines; a unit's, and a loose entry's (first entry, first pair, mate)
  extern __shared__ __attribute__((aligned(16))) float2 turn[];
  const int hq = a.heads[0], heads = hq + a.heads[1], pairs = a.end[a.axes - 1] >> 1;
  long4* place = (long4*)(turn + (a.tp * pairs + 1) / 2 * 2);
  int4* unit = (int4*)(place + a.ts * a.tp);
  int4* loose = unit + a.units;
  const long s0 = blockIdx.x / a.tiles * a.ts, p0 = blockIdx.x % a.tiles * a.tp;
  const int np = a.S - p0 < a.tp ? (int)(a.S - p0) : a.tp, ns = a.N - s0 < a.ts ? (int)(a.N - s0) : a.ts, nt = np * ns;
  for (int t = threadIdx.x; t < nt; t += blockDim.x) {
    const int s = t / np;
    const long p = p0 + t - s * np, b = a.N > 1 ? s0 + s : p / a.T, at = a.N > 1 ? p : p - b * a.T;
    place[t] = make_long4(b * a.sb[0] + at * a.st[0], b * a.sb[1] + at * a.st[1], (s0 + s) * a.S + p, t - s * np);
  }
  for (int w = threadIdx.x; w < a.units + a.loose; w += blockDim.x) {
    int u = w, l = w - a.units;   // its place among the units, and among the loose entries
    rot_regions<INTER>(a, [&](int from, int n, int pair, int mate) {
      const int nu = n / V, nl = n - nu * V;
      const int d = w < a.units ? u * V : nu * V + l;
      if (w < a.units ? u >= 0 && u < nu : l >= 0 && l < nl)
        unit[w] = make_int4(from + d, mate == 0 ? 0 : pair + (INTER ? d >> 1 : d), INTER && mate != 0 && (d & 1) ? -1 : mate, 0);
      u -= nu;
      l -= nl;
    });
  }
  __syncthreads();

  const T *xq = (const T*)a.x[0], *xk = (const T*)a.x[1];
  T *yq = (T*)a.y[0], *yk = (T*)a.y[1];
  // a lane keeps its unit and head and takes every subs-th token: only the token's offset and its sines change
  const int per = heads * a.units, width = per < (int)blockDim.x ? per : (int)blockDim.x, subs = width > 0 ? blockDim.x / width : 0;
  const int sub = width > 0 ? threadIdx.x / width : 0;
  int i = threadIdx.x - sub * width;
  bool more = i < per && sub < subs;
  raw own[U], mate[U];
  const T* x = nullptr;
  T* y = nullptr;
  const long* at = nullptr;
  int4 un = make_int4(0, 0, 0, 0);
  int stride = 0, out = 0;
  auto take = [&]() {   // item i: its unit and head
    const int h = i / a.units;
    un = unit[i - h * a.units];
    const bool isq = h < hq;
    const int hw = isq ? h : h - hq;
    stride = (isq ? hq : heads - hq) * a.D;
    x = (isq ? xq : xk) + hw * (isq ? a.sh[0] : a.sh[1]) + un.x;
    y = (isq ? yq : yk) + hw * a.D + un.x;
    at = (const long*)place + (isq ? 0 : 1);
    out = isq ? 2 : 1;
  };
  auto load = [&](int t) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int tu = t + u * subs;
      if (tu < nt) {
        const T* src = x + at[4 * tu];
        own[u] = Row<T>::load(src);
        if (!INTER && un.z != 0) mate[u] = Row<T>::load(src + un.z);
      }
    }
  };
  if (more) {   // (the first tokens are on their way while the angles are worked out)
    take();
    load(sub);
  }
  // (a division for the first of a lane's angles only: the next ones are blockDim pairs further)
  const int dt = blockDim.x / pairs, dj = blockDim.x - dt * pairs;
  for (int t = threadIdx.x / pairs, j = threadIdx.x - t * pairs; t < np;) {
    int ax = 0;
    while (2 * j >= a.end[ax]) ++ax;    // (pairs never straddle sections; j < pairs, so ax < axes)
    const P pos = ((const P*)a.pos)[(p0 + t) * a.axes + ax];
    const double quarter = (double)pos * a.freqs[j] * 0.63661977236758134308;   // the angle in units of pi / 2
    const double q = __builtin_rint(quarter);
    float sn, cs;
    indm_sincos_quadrant((float)((quarter - q) * 1.57079632679489661923), (int)(q - 4.0 * __builtin_floor(q * 0.25)), sn, cs);
    turn[t * pairs + j] = make_float2(cs, sn * a.sign);
    t += dt;
    j += dj;
    if (j >= pairs) {
      j -= pairs;
      ++t;
    }
  }
  __syncthreads();
  for (bool first = true; more; first = false) {
    for (int t = sub; t < nt; t += subs * U) {
      if (!first || t != sub) load(t);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int tu = t + u * subs;
        if (tu < nt) {
          T* dst = y + at[4 * tu + out] * stride;
          if (un.z == 0) {
            *(raw*)dst = own[u];
          } else {
            const float2* tr = turn + (int)at[4 * tu + out + 1] * pairs + un.y;
            float p[V], o[V];
            Row<T>::unpack(own[u], p);
            if constexpr (INTER) {
#pragma unroll
              for (int e = 0; e < V; e += 2) {
                const float2 cs = tr[e >> 1];
                o[e] = __builtin_fmaf(p[e], cs.x, -p[e + 1] * cs.y);
                o[e + 1] = __builtin_fmaf(p[e + 1], cs.x, p[e] * cs.y);
              }
              Row<T>::store(dst, o);
            } else {
              float m[V], w[V];
              Row<T>::unpack(mate[u], m);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float2 cs = tr[e];
                o[e] = __builtin_fmaf(p[e], cs.x, -m[e] * cs.y);
                w[e] = __builtin_fmaf(m[e], cs.x, p[e] * cs.y);
              }
              Row<T>::store(dst, o);
              Row<T>::store(dst + un.z, w);
            }
          }
        }
      }
    }
    i += width;
    more = i < per;
    if (more) take();
  }
  // the loose entries of each head; a section's halves go together
  const int entries = nt * heads * a.loose;
  for (int w = threadIdx.x; w < entries; w += blockDim.x) {
    const int th = w / a.loose, h = th % heads, t = th / heads;
    const int4 un = loose[w - th * a.loose];
    const T* src = (h < hq ? xq + place[t].x + h * a.sh[0] : xk + place[t].y + (h - hq) * a.sh[1]) + un.x;
    T* dst = (h < hq ? yq + (place[t].z * hq + h) * a.D : yk + (place[t].z * (heads - hq) + h - hq) * a.D) + un.x;
    if (un.z == 0) {
      *dst = *src;
    } else {
      const float2 cs = turn[(int)place[t].w * pairs + un.y];
      const float p = Row<T>::get(src), m = Row<T>::get(src + un.z);
      Row<T>::put(dst, __builtin_fmaf(p, cs.x, un.z < 0 ? m * cs.y : -m * cs.y));
      if (!INTER) Row<T>::put(dst + un.z, __builtin_fmaf(m, cs.x, p * cs.y));
    }
  }
}

template <typename T>
int rotary(const T* q, const T* k, T* yq, T* yk, const long* strides, int B, long Tn, int H, int Hk, int D, const void* pos,
           int pos_type, long pos_sb, const double* freqs, const int* sections, int axes, int interleaved, int inverse,
           hipStream_t st) {
  if (B < 0 || Tn < 0 || H < 0 || Hk < 0 || D <= 0 || D > ROT_MAX_D || axes <= 0 || axes > ROT_AXES) return INDM_E_SHAPE;
  if (strides == nullptr || sections == nullptr || pos_type < 0 || pos_type > 2) return INDM_E_ARG;
  RotArgs a = {};
  int at = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] <= 0 || (sections[i] & 1) || sections[i] > D - at) return INDM_E_SHAPE;
    a.end[i] = at += sections[i];
  }
  if (pos_sb != 0 && pos_sb != Tn * axes) return INDM_E_ARG;
  if (B == 0 || Tn == 0 || H + Hk == 0) return INDM_OK;
  if ((H > 0 && (q == nullptr || yq == nullptr)) || (Hk > 0 && (k == nullptr || yk == nullptr)) || pos == nullptr || freqs == nullptr)
    return INDM_E_ARG;
  a.x[0] = q; a.x[1] = k; a.y[0] = yq; a.y[1] = yk;
  for (int w = 0; w < 2; ++w) {
    a.sb[w] = strides[3 * w]; a.st[w] = strides[3 * w + 1]; a.sh[w] = strides[3 * w + 2];
  }
  a.heads[0] = H; a.heads[1] = Hk;
  a.pos = pos; a.freqs = freqs; a.T = Tn; a.D = D; a.axes = axes;
  a.S = pos_sb == 0 ? Tn : B * Tn; a.N = pos_sb == 0 ? B : 1;
  a.sign = inverse ? -1.f : 1.f;
  // lanes: as many whole tokens as fill wavefronts best (up to 512 lanes; a token of more units is walked in several steps)
  const int pairs = at / 2;
  auto count = [&](int, int n, int, int) {
    a.units += n / Row<T>::V;
    a.loose += n % Row<T>::V;
  };
  if (interleaved) rot_regions<true>(a, count);
  else rot_regions<false>(a, count);
  const long heads = (long)H + Hk, per = heads * a.units, tokens = (long)B * Tn;
  int lanes = 256;
  if (per > 0 && per <= 512) {
    double best = 0.;
    for (int k = 1; k * per <= 512; ++k) {
      const int n = (int)(k * per + 63) / 64 * 64;
      const double full = (double)(k * per) / n * (n >= 256 ? 1. : n >= 128 ? 0.97 : 0.9);   // (few wavefronts share the sines badly)
      if (full > best + 1e-9) {
        best = full;
        lanes = n;
      }
    }
  }
  // tokens a workgroup: 8 a lane where that still makes 1024 workgroups, down to one; the sines fit 32 KB of LDS
  long tb = per > 0 && per <= lanes ? lanes / per * 8 : 8;
  if (tb > 64) tb = 64;
  while (tb > 1 && (tokens + tb - 1) / tb < 1024) tb = (tb + 1) / 2;
  while (tb > 1 && tb * pairs * (long)sizeof(float2) > 32768) tb = (tb + 1) / 2;
  // samples that share their positions: up to four of them at one position (64 x 1024 tokens, bf16: 2 heads of 256 entries 45 -> 31 us, 8
  // of 64 31 -> 29 us; eight or sixteen samples gain no more)
  a.ts = a.N < 4 ? (int)a.N : 4;
  if (a.ts > tb) a.ts = (int)tb;
  a.tp = (int)(tb / a.ts);
  a.tiles = (a.S + a.tp - 1) / a.tp;
  const size_t lds = ((size_t)a.tp * pairs + 1) / 2 * 2 * sizeof(float2) + a.ts * a.tp * sizeof(long4) + (a.units + a.loose) * sizeof(int4);
  const long nb = a.tiles * ((a.N + a.ts - 1) / a.ts);
  if (nb > 0x7fffffffL || heads * D * tb > 0x3fffffffL) return INDM_E_SHAPE;   // (a workgroup's own offsets are 32-bit)
#define ROT_LAUNCH(P)                                                                                             \
  do {                                                                                                            \
    if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, P, true>), dim3((unsigned)nb), dim3(lanes), lds, st, a);  \
    else hipLaunchKernelGGL((rotary_kernel<T, P, false>), dim3((unsigned)nb), dim3(lanes), lds, st, a);             \
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
  return elem_bytes == 4 ? ln_ws<float>(R, C) : ln_ws<unsigned short>(R, C);
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
