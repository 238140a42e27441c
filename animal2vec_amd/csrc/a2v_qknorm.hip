// Norm of queries and keys for each head with the position rotation in the same pass:
//     y = R(pos) (x r w),   r = (mean(x^2) + eps)^(-1/2) over the HD channels of a head,   w (HD) fp32, shared by the heads
// R turns the channel pairs (a_p, b_p), p < R/2, by the angle pos_axis(p) * inv_freq[p]; the HD - R channels behind them are only
// normalised.  A pair is (p, p + R/2), or (2p, 2p + 1) with `inter`.  The pairs are cut into up to three runs, one for each axis of
// the position (time, and what else a recording has: microphone, band).
// Backward:  g = R^T dy,   dw = sum g x r,   dx = r (g w - x r mean(g w x r)).
//
// Bound by HBM: q and k once in, once out (backward: q, k and both gradients in, two out).  A lane holds eight whole pairs of a head
// (two 16-byte loads in 16-bit types), so the rotation needs no exchange and the norm HD / 16 lanes; a workgroup takes a few rows and
// all their heads, so that the row's R/2 angles are formed once (one per thread, in LDS) for H + HK heads.
// Measured: 64 clips of 2000 rows, 16 + 16 heads of 64 channels in bf16, 202 us = 5.2 TB/s, what a large copy reaches; forward and backward of
// 192 x 140 rows 117 us = 4.7 TB/s; one row of five streams 4 us, most of a launch.
// Angles: pos * inv_freq in 64 bits, reduced to a fraction of a turn before it is rounded -- a position of 10^9 keeps 2e-7 of a radian.
#include "a2v_common.h"

#define QKN_ROWS 16            /* most rows of a workgroup */
struct QknOne {                // queries or keys
  const void* x; const void* dy; void* y;                        // y: the result (forward), dx (backward)
  long long xn, xs, xh, dn, ds, dh, yn, ys, yh;                  // strides in elements: sequence, row, head
  const float* w;
  int heads;
};
struct QknArgs {
  QknOne t[2];
  const float* inv_freq; const int* pos;                         // pos null: the row's index
  long long pn, ps;
  long long M;                                                   // rows in all
  int S, R, axes, e0, e1, rows;                                  // e0, e1: first pair of the second and the third axis; rows of a workgroup
  float eps;
  float* part;                                                   // backward: (grid.x, 2, HD) partial sums of dw
};

template <int HD, bool INTER> struct QknLane {                   // the eight pairs of lane j of a head
  int da, db;                                                    // first channel of each 8-element load
  bool turn;
  __device__ __forceinline__ QknLane(int j, int R) {
    if (INTER) { da = 16 * j; db = da + 8; turn = da < R; return; }
    turn = j < R / 16;
    da = turn ? 8 * j : 16 * j;                                  // (behind the pairs: R + 16 (j - R / 16))
    db = turn ? R / 2 + 8 * j : da + 8;
  }
};
// a[i], b[i]: the two channels of pair i of this lane, from / to the two loads
template <typename T, bool INTER> __device__ __forceinline__ void qkn_load(const T* p, int da, int db, float* a, float* b) {
  float u[16];
  Vec8<T>::load(p + da, u);
  Vec8<T>::load(p + db, u + 8);
#pragma unroll
  for (int i = 0; i < 8; ++i) { a[i] = INTER ? u[2 * i] : u[i]; b[i] = INTER ? u[2 * i + 1] : u[8 + i]; }
}
template <typename T, bool INTER> __device__ __forceinline__ void qkn_store(T* p, int da, int db, const float* a, const float* b) {
  float u[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) { u[INTER ? 2 * i : i] = a[i]; u[INTER ? 2 * i + 1 : 8 + i] = b[i]; }
  Vec8<T>::store(p + da, u);
  Vec8<T>::store(p + db, u + 8);
}
template <int LPH> __device__ __forceinline__ float qkn_sum(float v) {       // over the LPH (2, 4 or 8) lanes of a head
#define QKN_ADD(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true))
  QKN_ADD(0xB1);                                                 // quad_perm [1,0,3,2]
  if (LPH > 2) QKN_ADD(0x4E);                                    // quad_perm [2,3,0,1]
  if (LPH > 4) QKN_ADD(0x141);                                   // row_half_mirror
#undef QKN_ADD
  return v;
}

template <int HD> struct QknShared {
  float cs[QKN_ROWS][HD / 2], sn[QKN_ROWS][HD / 2];
  long long off[QKN_ROWS][2][3];                                 // element offset of a row in x, dy and y
};
// the rows' angles and offsets; `n` rows from row m0
template <int HD> __device__ __forceinline__ void qkn_table(const QknArgs& a, QknShared<HD>& sm, long long m0, int n) {
  const int half = a.R / 2;
  for (int i = threadIdx.x; i < n * half; i += 256) {
    const int t = i / half, p = i - t * half;
    const long long m = m0 + t, b = m / a.S, s = m - b * a.S;
    const int axis = (p >= a.e0) + (p >= a.e1);
    const double x = a.pos ? (double)a.pos[b * a.pn + s * a.ps + axis] : (double)s;
    double turns = x * ((double)a.inv_freq[p] * 0.15915494309189533577);
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.f * (float)turns, &sn, &cs);
    sm.cs[t][p] = cs;
    sm.sn[t][p] = sn;
  }
  for (int i = threadIdx.x; i < n * 2; i += 256) {
    const int t = i >> 1, w = i & 1;
    const long long m = m0 + t, b = m / a.S, s = m - b * a.S;
    const QknOne& o = a.t[w];
    sm.off[t][w][0] = b * o.xn + s * o.xs;
    sm.off[t][w][1] = b * o.dn + s * o.ds;
    sm.off[t][w][2] = b * o.yn + s * o.ys;
  }
}

template <typename T, int HD, bool INTER>
__global__ __launch_bounds__(256) void qkn_fwd_kernel(QknArgs a) {
  constexpr int LPH = HD / 16;
  __shared__ __attribute__((aligned(16))) QknShared<HD> sm;
  const long long m0 = (long long)blockIdx.x * a.rows;
  const int n = a.M - m0 < a.rows ? (int)(a.M - m0) : a.rows;
  qkn_table<HD>(a, sm, m0, n);
  __syncthreads();
  const int j = threadIdx.x % LPH;
  const QknLane<HD, INTER> at(j, a.R);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const QknOne& o = a.t[w];
    float wa[8], wb[8];
    qkn_load<float, INTER>(o.w, at.da, at.db, wa, wb);
    for (int it = threadIdx.x / LPH; it < n * o.heads; it += 256 / LPH) {
      const int t = it / o.heads, h = it - t * o.heads;
      float x[8], y[8];
      qkn_load<T, INTER>((const T*)o.x + sm.off[t][w][0] + h * o.xh, at.da, at.db, x, y);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
      const float r = rsqrtf(qkn_sum<LPH>(ss) * (1.f / HD) + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) { x[i] *= r * wa[i]; y[i] *= r * wb[i]; }
      if (at.turn) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = sm.cs[t][8 * j + i], s = sm.sn[t][8 * j + i], u = x[i];
          x[i] = u * c - y[i] * s;
          y[i] = y[i] * c + u * s;
        }
      }
      qkn_store<T, INTER>((T*)o.y + sm.off[t][w][2] + h * o.yh, at.da, at.db, x, y);
    }
  }
}

// grid (blocks, 2): queries and keys apart, each workgroup walks groups of rows and keeps its part of dw in registers
template <typename T, int HD, bool INTER>
__global__ __launch_bounds__(256) void qkn_bwd_kernel(QknArgs a) {
  constexpr int LPH = HD / 16;
  __shared__ __attribute__((aligned(16))) QknShared<HD> sm;
  __shared__ float red[4][HD];
  const int j = threadIdx.x % LPH, w = blockIdx.y;
  const QknLane<HD, INTER> at(j, a.R);
  const QknOne& o = a.t[w];
  float wa[8], wb[8], ga[8], gb[8];
  qkn_load<float, INTER>(o.w, at.da, at.db, wa, wb);
#pragma unroll
  for (int i = 0; i < 8; ++i) ga[i] = gb[i] = 0.f;
  for (long long m0 = (long long)blockIdx.x * a.rows; m0 < a.M; m0 += (long long)gridDim.x * a.rows) {
    const int n = a.M - m0 < a.rows ? (int)(a.M - m0) : a.rows;
    qkn_table<HD>(a, sm, m0, n);
    __syncthreads();
    for (int it = threadIdx.x / LPH; it < n * o.heads; it += 256 / LPH) {
      const int t = it / o.heads, h = it - t * o.heads;
      float x[8], y[8], p[8], q[8];
      qkn_load<T, INTER>((const T*)o.x + sm.off[t][w][0] + h * o.xh, at.da, at.db, x, y);
      qkn_load<T, INTER>((const T*)o.dy + sm.off[t][w][1] + h * o.dh, at.da, at.db, p, q);
      if (at.turn) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = sm.cs[t][8 * j + i], s = sm.sn[t][8 * j + i], u = p[i];
          p[i] = u * c + q[i] * s;
          q[i] = q[i] * c - u * s;
        }
      }
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
      const float r = rsqrtf(qkn_sum<LPH>(ss) * (1.f / HD) + a.eps);
      float gx = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= r; y[i] *= r;
        ga[i] += p[i] * x[i]; gb[i] += q[i] * y[i];
        p[i] *= wa[i]; q[i] *= wb[i];
        gx += p[i] * x[i] + q[i] * y[i];
      }
      gx = qkn_sum<LPH>(gx) * (1.f / HD);
#pragma unroll
      for (int i = 0; i < 8; ++i) { p[i] = r * (p[i] - x[i] * gx); q[i] = r * (q[i] - y[i] * gx); }
      qkn_store<T, INTER>((T*)o.y + sm.off[t][w][2] + h * o.yh, at.da, at.db, p, q);
    }
    __syncthreads();
  }
  // the lanes of one j in a fixed order: inside the wave, then over the four waves, then (qkn_dw_kernel) over the workgroups
#pragma unroll
  for (int x = LPH; x < 64; x <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) { ga[i] += __shfl_xor(ga[i], x, 64); gb[i] += __shfl_xor(gb[i], x, 64); }
  if ((threadIdx.x & 63) < LPH) qkn_store<float, INTER>(red[threadIdx.x >> 6], at.da, at.db, ga, gb);
  __syncthreads();
  if (threadIdx.x < HD) {
    const int d = threadIdx.x;
    a.part[((long long)blockIdx.x * 2 + w) * HD + d] = (red[0][d] + red[1][d]) + (red[2][d] + red[3][d]);
  }
}
// dw += the partial rows' sums, 16 channels to a workgroup, 64 strands of rows each with eight loads in flight (one strand per channel
// and workgroup took 18 us for 1024 rows)
__global__ __launch_bounds__(1024) void qkn_dw_kernel(const float* part, int blocks, int HD, float* dwq, float* dwk) {
  __shared__ float red[1024];
  const int w = blockIdx.y, c = threadIdx.x & 15, d = blockIdx.x * 16 + c, k = threadIdx.x >> 4;
  const float* const p = part + (long long)w * HD + d;
  float v = 0.f;
#pragma unroll 8
  for (int i = k; i < blocks; i += 64) v += p[(long long)i * 2 * HD];
  red[threadIdx.x] = v;
  __syncthreads();
  for (int n = 32; n >= 1; n >>= 1) {
    if (k < n) red[threadIdx.x] += red[threadIdx.x + 16 * n];
    __syncthreads();
  }
  if (k == 0) (w ? dwk : dwq)[d] += red[c];
}

// ------------------------------------------------------------------------------------------------------------------ host side
#define QKN_BLOCKS 512         /* workgroups of the backward pass (times two, what fits the card): each leaves HD partial sums */
static int qkn_rows(long long M, int heads, int HD) {
  // rows of a workgroup: four trips of 256 lanes over its heads; fewer where that would leave compute units without a workgroup
  long long rows = 4LL * 256 / ((long long)heads * (HD / 16));
  if (rows > M / 512) rows = M / 512;
  return rows < 1 ? 1 : (rows > QKN_ROWS ? QKN_ROWS : (int)rows);
}
static int qkn_blocks(long long M, int rows) {
  const long long b = (M + rows - 1) / rows;
  return b < QKN_BLOCKS ? (int)b : QKN_BLOCKS;
}
static bool qkn_tensor_ok(const void* p, const long long* st, int es) {
  return p && !((uintptr_t)p & 15) && !((st[0] * es) & 15) && !((st[1] * es) & 15) && !((st[2] * es) & 15);
}
static int qkn_fill(QknArgs& a, int dtype, const float* q_weight, const float* k_weight, const float* inv_freq, const int* pos, const long long* pos_strides,
                    int axes, const int* sections, float eps, int N, int S, int H, int HK, int HD) {
  if (dtype != A2V_F32 && dtype != A2V_BF16) return A2V_ERR_DTYPE;
  if (!q_weight || !k_weight || !inv_freq || !sections || (pos && !pos_strides) || (((uintptr_t)q_weight | (uintptr_t)k_weight) & 15) || axes < 1 || axes > 3 ||
      (!pos && axes != 1) || N < 0 || S < 0 || H <= 0 || HK <= 0 || (HD != 32 && HD != 64 && HD != 128))
    return A2V_ERR_ARG;
  long long half = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] > HD / 2) return A2V_ERR_ARG;
    half += sections[i];
  }
  if (half % 8 || half < 8 || half > HD / 2) return A2V_ERR_ARG;
  a.inv_freq = inv_freq; a.pos = pos;
  a.pn = pos ? pos_strides[0] : 0; a.ps = pos ? pos_strides[1] : 0;
  a.M = (long long)N * S; a.S = S; a.R = 2 * (int)half; a.axes = axes; a.eps = eps; a.part = nullptr;
  a.e0 = axes > 1 ? sections[0] : (int)half;
  a.e1 = axes > 2 ? sections[0] + sections[1] : (int)half;
  a.rows = 1;
  a.t[0].w = q_weight; a.t[0].heads = H;
  a.t[1].w = k_weight; a.t[1].heads = HK;
  return A2V_OK;
}
#define QKN_LAUNCH(kern_, grid_)                                                                        \
  do {                                                                                                  \
    const dim3 g_ = grid_;                                                                              \
    if (dtype == A2V_F32) { QKN_HD(kern_, float, g_); } else { QKN_HD(kern_, bf16, g_); }               \
  } while (0)
#define QKN_HD(kern_, T_, g_)                                                                           \
  if (HD == 32) QKN_INTER(kern_, T_, 32, g_); else if (HD == 64) QKN_INTER(kern_, T_, 64, g_); else QKN_INTER(kern_, T_, 128, g_)
#define QKN_INTER(kern_, T_, HD_, g_)                                                                   \
  do {                                                                                                  \
    if (interleaved) hipLaunchKernelGGL((kern_<T_, HD_, true>), g_, dim3(256), 0, stream, a);           \
    else hipLaunchKernelGGL((kern_<T_, HD_, false>), g_, dim3(256), 0, stream, a);                      \
  } while (0)

extern "C" int a2v_qk_norm_rope_fwd(int dtype, const void* q, const void* k, void* q_out, void* k_out, const long long* strides, const float* q_weight,
                                    const float* k_weight, const float* inv_freq, const int* pos, const long long* pos_strides, int axes,
                                    const int* sections, int interleaved, float eps, int N, int S, int H, int HK, int HD, hipStream_t stream) {
  QknArgs a;
  if (int e = qkn_fill(a, dtype, q_weight, k_weight, inv_freq, pos, pos_strides, axes, sections, eps, N, S, H, HK, HD)) return e;
  if (!strides) return A2V_ERR_ARG;
  if (a.M == 0) return A2V_OK;
  const int es = dtype == A2V_F32 ? 4 : 2;
  const long long* const s = strides;
  if (!qkn_tensor_ok(q, s, es) || !qkn_tensor_ok(k, s + 3, es) || !qkn_tensor_ok(q_out, s + 6, es) || !qkn_tensor_ok(k_out, s + 9, es)) return A2V_ERR_ARG;
  a.t[0] = QknOne{q, nullptr, q_out, s[0], s[1], s[2], 0, 0, 0, s[6], s[7], s[8], q_weight, H};
  a.t[1] = QknOne{k, nullptr, k_out, s[3], s[4], s[5], 0, 0, 0, s[9], s[10], s[11], k_weight, HK};
  a.rows = qkn_rows(a.M, H + HK, HD);
  const long long blocks = (a.M + a.rows - 1) / a.rows;
  if (blocks >= (1LL << 24)) return A2V_ERR_ARG;                  // (2^32 threads)
  QKN_LAUNCH(qkn_fwd_kernel, dim3((unsigned)blocks));
  A2V_CHECK_LAUNCH();
  return A2V_OK;
}

extern "C" size_t a2v_qk_norm_rope_workspace(int N, int S, int H, int HK, int HD) {
  if (N <= 0 || S <= 0 || H <= 0 || HK <= 0 || HD <= 0) return 0;
  const long long M = (long long)N * S;
  return (size_t)qkn_blocks(M, qkn_rows(M, H > HK ? H : HK, HD)) * 2 * HD * sizeof(float);
}

extern "C" int a2v_qk_norm_rope_bwd(int dtype, const void* dq_out, const void* dk_out, const void* q, const void* k, void* dq, void* dk,
                                    const long long* strides, const float* q_weight, const float* k_weight, float* dq_weight, float* dk_weight,
                                    const float* inv_freq, const int* pos, const long long* pos_strides, int axes, const int* sections, int interleaved,
                                    float eps, int N, int S, int H, int HK, int HD, void* ws, size_t ws_bytes, hipStream_t stream) {
  QknArgs a;
  if (int e = qkn_fill(a, dtype, q_weight, k_weight, inv_freq, pos, pos_strides, axes, sections, eps, N, S, H, HK, HD)) return e;
  if (!strides || !dq_weight || !dk_weight) return A2V_ERR_ARG;
  if (a.M == 0) return A2V_OK;
  const int es = dtype == A2V_F32 ? 4 : 2;
  const long long* const s = strides;
  const void* const t[6] = {dq_out, dk_out, q, k, dq, dk};
  for (int i = 0; i < 6; ++i)
    if (!qkn_tensor_ok(t[i], s + 3 * i, es)) return A2V_ERR_ARG;
  if (!ws || ((uintptr_t)ws & 15) || ws_bytes < a2v_qk_norm_rope_workspace(N, S, H, HK, HD)) return A2V_ERR_ARG;
  a.t[0] = QknOne{q, dq_out, dq, s[6], s[7], s[8], s[0], s[1], s[2], s[12], s[13], s[14], q_weight, H};
  a.t[1] = QknOne{k, dk_out, dk, s[9], s[10], s[11], s[3], s[4], s[5], s[15], s[16], s[17], k_weight, HK};
  a.rows = qkn_rows(a.M, H > HK ? H : HK, HD);
  a.part = (float*)ws;
  const int blocks = qkn_blocks(a.M, a.rows);
  QKN_LAUNCH(qkn_bwd_kernel, dim3(blocks, 2));
  hipLaunchKernelGGL(qkn_dw_kernel, dim3(HD / 16, 2), dim3(1024), 0, stream, a.part, blocks, HD, dq_weight, dk_weight);
  A2V_CHECK_LAUNCH();
  return A2V_OK;
}
