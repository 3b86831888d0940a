// Root-mean-square norm with the residual's addition:
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  y = s rstd w
// its backward pass, and the form whose output is 8 bits (OCP e4m3) with one scale per row.  No counterpart in the
// reference (its networks use LayerNorm, rowops.hip).
//
// Bound by memory: a row is read once into registers, reduced, and written; 16 or 32 lanes take a row of up to
// 16 or 32 vectors of 16 bytes (16: 262144 x 128 bf16 83 -> 42 us, 500000 x 33 both ways 360 -> 128 us against a wave per row), a
// wave one of up to 128 (no LDS, no barrier), a workgroup of 256 or 1024 threads a longer one.  The norm is of the sum as it is
// STORED (rounded to the residual's type): later layers and the backward pass see the values that were normed.
// 16384 x 4096 bf16: forward call after call 79 us (6.8 TB/s: part of it from the caches), both ways 93 + 82 + 5 us (5.2 TB/s), the 5 for
// the shares of the weight's gradient; to e4m3 74 us, 64 rows 4 us.
#include "seqtypes.h"

#define RMS_MAXN 32768
#define RMS_MAXR 0x7fff0000  // a row number and the step to the next one fit 31 bits
#define RMS_LAUNCH (1 << 21) // rows of one forward launch: at 1024 threads each it has less than 2^32
#define RMS_PARTS 512        // rows of partial weight gradients: at most this many workgroups in the backward pass,
#define RMS_MOSTPARTS 8192   // more for short rows

struct RmsArgs {
  const void *x, *res, *w, *ds;      // backward: x = dy, res = s
  long long ldx, ldres, ldds;
  void *y, *sum; long long ldy, ldsum;
  float *scale, *rstd_out, *part;
  const float* rstd_in;
  int R, N, w_f32; float eps;
};

// Where round i of thread t lies in a row of N columns, VEC apiece.  LOOSE: the row's length is no multiple of VEC, or its rows start
// at any element; the last vector then moves left to end with the row (N >= VEC), and its first `skip` columns are the left
// neighbour's, computed twice and counted once.  A column behind the row reads some of its last (or first) ones, not used.
// Against single elements: 5840 x 4295 fp16 with an fp32 residual 694 -> 57 us, 20000 x 1001
// bf16 both ways 98 -> 71 us.
template <int THREADS, int NV, int VEC, bool LOOSE> struct RmsAt {
  int n, skip;
  bool in;
  __device__ __forceinline__ RmsAt(int i, int t, int N) {
    const int c = (i * THREADS + t) * VEC;
    const bool whole = i < NV / 2;      // the row has more than NV / 2 rounds: see the choice of the shape
    in = whole || c < N;
    n = whole ? c : LOOSE ? min(c, N - VEC) : in ? c : 0;
    skip = LOOSE ? c - n : 0;
  }
  __device__ __forceinline__ bool counts(int v) const { return LOOSE ? v >= skip : in; }
};

// VEC weights from column n on, in the tensors' own 16-bit type or fp32
template <typename T, int VEC, bool LOOSE>
__device__ __forceinline__ void rms_weight(const RmsArgs& a, int n, float (&w)[VEC]) {
  if (T::code == SERL_F32 || a.w_f32) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) w[v] = ((const float*)a.w)[n + v];
  } else {
    Raw<T, VEC> r;
    r.template load<LOOSE>((const typename T::bits*)a.w + n);
    r.get(w);
  }
}

// over a row's lanes of a wave: all of them, or the THREADS of a short row
template <int THREADS> __device__ __forceinline__ float rms_sum(float v) { return sq_wave_sum<(THREADS < 64 ? THREADS : 64)>(v); }
template <int THREADS> __device__ __forceinline__ unsigned rms_max(unsigned v) {
  return sq_over_lanes<(THREADS < 64 ? THREADS : 64)>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// e4m3 codes of four values: rounded to nearest even, clipped to +-448 (an infinity as well), NaN stays NaN
__device__ __forceinline__ float rms_clip(float v) { return v != v ? v : fminf(fmaxf(v, -448.f), 448.f); }
__device__ __forceinline__ uint32_t rms_e4m3x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(rms_clip(a), rms_clip(b), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(rms_clip(c), rms_clip(d), r, true);
  return (uint32_t)r;
}

// y / scale, rounded once to fp32 in front of e4m3's own rounding: a product with 1 / scale rounds twice and moved some 5 codes in 10^5
// next to the middle of two.  With the scale brought to b in [1/2, 1) and inv = 1 / b correctly rounded, the product's remainder is exact and
// one correction gives the correctly rounded quotient (P. Markstein's method; 4 instructions per element, where
// the division's 11 made rows of 1001 8 % slower).  An infinite scale: finite values give 0, infinities NaN.
struct RmsOver {
  int e;
  float b, inv;
  __device__ __forceinline__ explicit RmsOver(float scale) {
    e = __builtin_amdgcn_frexp_expf(scale);
    b = __builtin_amdgcn_ldexpf(scale, -e);
    inv = 1.f / b;
    b = b == INFINITY ? 0.f : b;
  }
  __device__ __forceinline__ float operator()(float y) const {
    y = __builtin_amdgcn_ldexpf(y, -e);
    const float q = y * inv;
    return fmaf(fmaf(-q, b, y), inv, q);
  }
};

template <typename TX, typename TR, bool FP8, int THREADS, int NV, int VEC, bool LOOSE, bool STREAM>
__global__ __launch_bounds__(THREADS <= 64 ? 256 : THREADS) void rms_fwd_kernel(const RmsArgs a) {
  constexpr int WAVES = THREADS <= 64 ? 1 : THREADS / 64;
  __shared__ float red[WAVES];
  __shared__ unsigned redm[WAVES];
  const int t = threadIdx.x % THREADS, wave = t >> 6, lane = t & 63;
  const int row = THREADS <= 64 ? (int)(blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS) : (int)blockIdx.x;
  if (THREADS <= 64 && row >= a.R) return;
  const typename TX::bits* x = (const typename TX::bits*)a.x + row * a.ldx;
  Raw<TX, VEC> rx[NV];
  Raw<TR, VEC> rr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
    rx[i].template load<LOOSE, STREAM>(x + at.n);
  }
  if (a.res) {
    const typename TR::bits* res = (const typename TR::bits*)a.res + row * a.ldres;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
      rr[i].template load<LOOSE, STREAM>(res + at.n);
    }
  }
  float s[NV][VEC], ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
    rx[i].get(s[i]);
    if (a.res) {
      float r[VEC];
      rr[i].get(r);
#pragma unroll
      for (int v = 0; v < VEC; ++v) s[i][v] += r[v];
      rr[i].put(s[i]);
      rr[i].get(s[i]);
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) ss = at.counts(v) ? fmaf(s[i][v], s[i][v], ss) : ss;
  }
  const auto put_sum = [&]() {
    if (a.sum) {
      typename TR::bits* sum = (typename TR::bits*)a.sum + row * a.ldsum;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
        if (at.in) rr[i].template store<LOOSE>(sum + at.n);
      }
    }
  };
  if constexpr (!LOOSE) put_sum();
  ss = rms_sum<THREADS>(ss);
  if constexpr (WAVES > 1) {
    if (lane == 0) red[wave] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) ss += red[w];
  }
  if constexpr (LOOSE) put_sum();       // when all have read: sum may be the residual, and two threads read some columns
  const float rstd = rsqrtf(ss / (float)a.N + a.eps);
  if (a.rstd_out && t == 0) a.rstd_out[row] = rstd;
  unsigned top = 0;                     // |y| as bits: ordered like the values, NaN above infinity
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
    float w[VEC];
    rms_weight<TX, VEC, LOOSE>(a, at.n, w);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      s[i][v] = s[i][v] * rstd * w[v];
      if (FP8) {
        const unsigned m = __float_as_uint(s[i][v]) & 0x7fffffffu;
        top = at.in && m > top ? m : top;
      }
    }
    if (!FP8 && at.in) {
      rx[i].put(s[i]);
      rx[i].template store<LOOSE>((typename TX::bits*)a.y + row * a.ldy + at.n);
    }
  }
  if constexpr (FP8) {
    top = rms_max<THREADS>(top);
    if constexpr (WAVES > 1) {
      if (lane == 0) redm[wave] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) top = redm[w] > top ? redm[w] : top;
    }
    float scale = __uint_as_float(top) / 448.f;
    scale = scale < 1.17549435e-38f ? 1.17549435e-38f : scale;      // so that 1 / scale is finite
    scale = top == 0 ? 1.f : scale;
    if (t == 0) a.scale[row] = scale;
    const RmsOver over(scale);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
      unsigned char* q = (unsigned char*)a.y + row * a.ldy + at.n;
      if (at.in) {
        if constexpr (VEC == 8) {
          const sq_u32x2 c = {rms_e4m3x4(over(s[i][0]), over(s[i][1]), over(s[i][2]), over(s[i][3])),
                              rms_e4m3x4(over(s[i][4]), over(s[i][5]), over(s[i][6]), over(s[i][7]))};
          if constexpr (LOOSE) __builtin_memcpy(q, &c, 8);
          else *(sq_u32x2*)q = c;
        } else if constexpr (VEC == 4) {
          const uint32_t c = rms_e4m3x4(over(s[i][0]), over(s[i][1]), over(s[i][2]), over(s[i][3]));
          if constexpr (LOOSE) __builtin_memcpy(q, &c, 4);
          else *(uint32_t*)q = c;
        } else {
          *q = (unsigned char)(rms_e4m3x4(over(s[i][0]), 0.f, 0.f, 0.f) & 0xffu);
        }
      }
    }
  }
}

// dx = rstd (w dy - xh mean(w dy xh)) + ds with xh = s rstd; dw = sum over rows of dy xh.  A workgroup (THREADS = 64: a
// wave, less: that many lanes) takes every gridDim-th row and keeps its share of dw in registers; the shares are added in a fixed order by
// rms_dw_kernel, so the result does not depend on timing.
template <typename TY, typename TS, int THREADS, int NV, int VEC, bool LOOSE, bool STREAM>
__global__ __launch_bounds__(THREADS <= 64 ? 256 : THREADS) void rms_bwd_kernel(const RmsArgs a) {
  constexpr int WAVES = THREADS <= 64 ? 1 : THREADS / 64;
  __shared__ float red[2][WAVES];
  const int t = threadIdx.x % THREADS, wave = t >> 6, lane = t & 63;
  const int first = THREADS <= 64 ? (int)(blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS) : (int)blockIdx.x;
  const int step = THREADS <= 64 ? (int)gridDim.x * (256 / THREADS) : (int)gridDim.x;
  // The weights stay in registers, and ds is fetched with the rest; with 32 columns per thread they would not fit the 128
  // registers, so both are read where they are used, the weights twice a row (from the L2).  2048 x 32768 bf16 383 -> 356 us.
  constexpr bool HOLD = THREADS < 1024 || NV * VEC <= 16;
  float w[HOLD ? NV : 1][VEC], dw[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
    if (HOLD) rms_weight<TY, VEC, LOOSE>(a, at.n, w[HOLD ? i : 0]);
#pragma unroll
    for (int v = 0; v < VEC; ++v) dw[i][v] = 0.f;
  }
  int buf = 0;
  for (int row = first; row < a.R; row += step, buf ^= 1) {
    const typename TY::bits* dy = (const typename TY::bits*)a.x + row * a.ldx;
    const typename TS::bits* s = (const typename TS::bits*)a.res + row * a.ldres;
    const typename TS::bits* ds = (const typename TS::bits*)a.ds + row * a.ldds;
    const float rstd = a.rstd_in[row];
    Raw<TY, VEC> ry[NV];
    Raw<TS, VEC> rs[NV], rd[HOLD ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
      ry[i].template load<LOOSE, STREAM>(dy + at.n);
      rs[i].template load<LOOSE, STREAM>(s + at.n);
    }
    if (HOLD && a.ds) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
        rd[HOLD ? i : 0].template load<LOOSE, STREAM>(ds + at.n);
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
      float y[VEC], x[VEC];
      if (!HOLD) rms_weight<TY, VEC, LOOSE>(a, at.n, w[0]);
      ry[i].get(y);
      rs[i].get(x);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float d = y[v] * (x[v] * rstd);
        dw[i][v] += d;
        dot = at.counts(v) ? fmaf(w[HOLD ? i : 0][v], d, dot) : dot;
      }
    }
    dot = rms_sum<THREADS>(dot);
    if constexpr (WAVES > 1) {
      if (lane == 0) red[buf][wave] = dot;
      __syncthreads();
      dot = 0.f;
#pragma unroll
      for (int q = 0; q < WAVES; ++q) dot += red[buf][q];
    }
    dot /= (float)a.N;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
      float y[VEC], x[VEC], d[VEC];
      if (!HOLD) rms_weight<TY, VEC, LOOSE>(a, at.n, w[0]);
      if (!HOLD && a.ds) rd[0].template load<LOOSE, STREAM>(ds + at.n);
      sq_again(ry[i]);
      sq_again(rs[i]);
      ry[i].get(y);
      rs[i].get(x);
#pragma unroll
      for (int v = 0; v < VEC; ++v) d[v] = 0.f;
      if (a.ds) rd[HOLD ? i : 0].get(d);
#pragma unroll
      for (int v = 0; v < VEC; ++v) d[v] = fmaf(rstd, fmaf(-(x[v] * rstd), dot, y[v] * w[HOLD ? i : 0][v]), d[v]);
      typename TS::bits* dx = (typename TS::bits*)a.y + row * a.ldy + at.n;
      rs[i].put(d);
      if (LOOSE && WAVES > 1 && at.skip > 0) {       // its own columns alone: dx may be ds, of which the left neighbour, of another wave, may have
#pragma unroll
        for (int v = 1; v < VEC; ++v)   // stored the first ones over what was read here
          if (v >= at.skip && at.in) dx[v] = sq_bits(TS(), d[v]);
      } else if (at.in) {
        rs[i].template store<LOOSE>(dx);
      }
    }
  }
  if constexpr (THREADS < 64) {          // the wave's rows side by side
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int v = 0; v < VEC; ++v)
#pragma unroll
        for (int o = THREADS; o < 64; o <<= 1) dw[i][v] += __shfl_xor(dw[i][v], o);
    if (lane >= THREADS) return;
  }
  float* part = a.part + (long long)(THREADS < 64 ? blockIdx.x * 4 + (threadIdx.x >> 6) : first) * a.N;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const RmsAt<THREADS, NV, VEC, LOOSE> at(i, t, a.N);
    if (at.in)
#pragma unroll
      for (int v = 0; v < VEC; ++v) part[at.n + v] = dw[i][v];
  }
}

// dw[n] = sum over the parts, 32 columns x 32 part lanes per workgroup, the lanes' sums added in order
__global__ __launch_bounds__(1024) void rms_dw_kernel(const float* part, int parts, int N, float* dw) {
  __shared__ float sum[32][33];
  const int c = threadIdx.x & 31, p0 = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int p = p0; p < parts; p += 32) s += part[(long long)p * N + n];
  }
  sum[p0][c] = s;
  __syncthreads();
  if (p0 == 0 && n < N) {
    s = 0.f;
#pragma unroll
    for (int p = 0; p < 32; ++p) s += sum[p][c];
    dw[n] = s;
  }
}

// ---------------------------------------------------------------------------------------------------------- host side
template <typename TX, typename TR, bool FP8, int THREADS, int NV, int VEC, bool LOOSE, bool STREAM>
static void rms_go_fwd(const RmsArgs& a, hipStream_t st) {
  const unsigned grid = THREADS <= 64 ? (unsigned)cdiv(a.R, 256 / THREADS) : (unsigned)a.R;
  hipLaunchKernelGGL((rms_fwd_kernel<TX, TR, FP8, THREADS, NV, VEC, LOOSE, STREAM>), dim3(grid), dim3(THREADS <= 64 ? 256 : THREADS), 0, st, a);
}
template <typename TX, typename TR, bool FP8, bool LOOSE, bool STREAM>
static void rms_shape_fwd(const RmsArgs& a, hipStream_t st) {
  constexpr int V = TX::code == SERL_F32 ? 4 : 8;
  const int n = cdiv(a.N, V);          // vectors of a row; more than half of those of a shape with several rounds (RmsAt)
  if (n <= 16) rms_go_fwd<TX, TR, FP8, 16, 1, V, LOOSE, STREAM>(a, st);
  else if (n <= 32) rms_go_fwd<TX, TR, FP8, 32, 1, V, LOOSE, STREAM>(a, st);
  else if (n <= 64) rms_go_fwd<TX, TR, FP8, 64, 1, V, LOOSE, STREAM>(a, st);
  else if (n <= 128) rms_go_fwd<TX, TR, FP8, 64, 2, V, LOOSE, STREAM>(a, st);
  else if (n <= 256) rms_go_fwd<TX, TR, FP8, 256, 1, V, LOOSE, STREAM>(a, st);
  else if (n <= 512) rms_go_fwd<TX, TR, FP8, 256, 2, V, LOOSE, STREAM>(a, st);
  else if (n <= 1024) rms_go_fwd<TX, TR, FP8, 256, 4, V, LOOSE, STREAM>(a, st);
  else if constexpr (STREAM) return;                    // not chosen
  else if (n <= 2048) rms_go_fwd<TX, TR, FP8, 1024, 2, V, LOOSE, STREAM>(a, st);
  else if (n <= 4096) rms_go_fwd<TX, TR, FP8, 1024, 4, V, LOOSE, STREAM>(a, st);
  else if constexpr (TX::code == SERL_F32) rms_go_fwd<TX, TR, FP8, 1024, 8, V, LOOSE, STREAM>(a, st);      // RMS_MAXN elements
}
// Inputs are streamed past the caches where a call moves more than they hold and rows are whole cache lines: 16384 x 4096 bf16
// forward 91 -> 78 us, both ways 197 -> 175; just above the caches' size 16384 x 2048 forward loses, 42.6 -> 44.3.  Not with rows of
// 1024 threads (2048 x 16384 both ways 111 -> 119 us) or a residual of another type (16384 x 4096 with fp32 317 -> 331 us).
static bool rms_stream(const RmsArgs& a, int type, int tensors) {
  const int e = sq_size(type);
  return a.N * e % 128 == 0 && a.ldx * e % 128 == 0 && a.ldres * e % 128 == 0 && a.N * e <= 1024 * 16 &&
         sq_aligned(a.x, 128) && sq_aligned(a.res, 128) &&
         (long long)a.R * a.N * e * tensors > SQ_STREAM;
}

template <typename TX, typename TR, bool FP8>
static void rms_pick_fwd(const RmsArgs& a, bool wide, hipStream_t st) {
  if (wide && TX::code == TR::code && rms_stream(a, TX::code, a.res ? 4 : 2)) rms_shape_fwd<TX, TR, FP8, false, true>(a, st);
  else if (wide) rms_shape_fwd<TX, TR, FP8, false, false>(a, st);
  else if (a.N >= (TX::code == SERL_F32 ? 4 : 8)) rms_shape_fwd<TX, TR, FP8, true, false>(a, st);
  else rms_go_fwd<TX, TR, FP8, 16, 1, 1, false, false>(a, st);      // a row of less than a vector
}

// Rows of the partial weight gradients: one per row of the input (rounded up to 4), at most RMS_PARTS, one per workgroup or, for
// short rows, per wave.  Short rows get more, as many as keep the partial sums at 8 MB and 8 rows to each: 131072 x 512 bf16
// 355 -> 207 us both ways, 20000 x 1536 99 -> 84 us; but without the 8 rows 5000 x 1001 fp32 36 -> 39 us, and longer rows lose by
// it (32768 x 2048 with 2048 parts 193 -> 210 us).  A workgroup of 1024 threads has a CU to itself, so 256 parts: 2048 x 32768
// bf16 356 -> 324 us.  vec: elements per access.
static int rms_parts(int R, int N, int vec) {
  const int n = cdiv(N, vec);
  int most = n <= 128 ? (1 << 21) / N : n <= 256 ? (3 << 19) / N : n <= 1024 ? RMS_PARTS : RMS_PARTS / 2;
  if (n <= 256) {
    most = most > RMS_MOSTPARTS ? RMS_MOSTPARTS : most;
    most = most > R / 8 ? R / 8 : most;
    most = most < RMS_PARTS ? RMS_PARTS : most / 4 * 4;
  }
  return R < most ? (R + 3) / 4 * 4 : most;
}

template <typename TY, typename TS, int THREADS, int NV, int VEC, bool LOOSE, bool STREAM>
static void rms_go_bwd(const RmsArgs& a, hipStream_t st) {
  const int parts = rms_parts(a.R, a.N, TY::code == SERL_F32 ? 4 : 8);
  hipLaunchKernelGGL((rms_bwd_kernel<TY, TS, THREADS, NV, VEC, LOOSE, STREAM>), dim3(THREADS <= 64 ? parts / 4 : parts),
                     dim3(THREADS <= 64 ? 256 : THREADS), 0, st, a);
}
template <typename TY, typename TS, bool LOOSE, bool STREAM>
static void rms_shape_bwd(const RmsArgs& a, hipStream_t st) {
  constexpr int V = TY::code == SERL_F32 ? 4 : 8;
  const int n = cdiv(a.N, V);          // as in rms_shape_fwd
  if (n <= 16) rms_go_bwd<TY, TS, 16, 1, V, LOOSE, STREAM>(a, st);
  else if (n <= 32) rms_go_bwd<TY, TS, 32, 1, V, LOOSE, STREAM>(a, st);
  else if (n <= 64) rms_go_bwd<TY, TS, 64, 1, V, LOOSE, STREAM>(a, st);
  else if (n <= 128) rms_go_bwd<TY, TS, 64, 2, V, LOOSE, STREAM>(a, st);
  else if (n <= 256) rms_go_bwd<TY, TS, 256, 1, V, LOOSE, STREAM>(a, st);
  else if (n <= 512) rms_go_bwd<TY, TS, 256, 2, V, LOOSE, STREAM>(a, st);
  else if (n <= 1024) rms_go_bwd<TY, TS, 256, 4, V, LOOSE, STREAM>(a, st);
  else if constexpr (STREAM) return;                    // not chosen
  else if (n <= 2048) rms_go_bwd<TY, TS, 1024, 2, V, LOOSE, STREAM>(a, st);
  else if (n <= 4096) rms_go_bwd<TY, TS, 1024, 4, V, LOOSE, STREAM>(a, st);
  else if constexpr (TY::code == SERL_F32) rms_go_bwd<TY, TS, 1024, 8, V, LOOSE, STREAM>(a, st);
}
template <typename TY, typename TS>
static void rms_pick_bwd(const RmsArgs& a, bool wide, hipStream_t st) {
  if (wide && TY::code == TS::code && rms_stream(a, TY::code, a.ds ? 4 : 3)) rms_shape_bwd<TY, TS, false, true>(a, st);
  else if (wide) rms_shape_bwd<TY, TS, false, false>(a, st);
  else if (a.N >= (TY::code == SERL_F32 ? 4 : 8)) rms_shape_bwd<TY, TS, true, false>(a, st);
  else rms_go_bwd<TY, TS, 16, 1, 1, false, false>(a, st);
}

static bool rms_wide(int type, int elems, const void* p, long long ld) {
  const int e = type == SERL_F32 ? 4 : 2;
  return !p || (sq_aligned(p, 16) && ld % elems == 0 && (ld * e) % 16 == 0);
}

// x and y of type `type`, residual and sum of type `stream_type` (the same, or fp32), weight of type `type` or fp32.
static int rms_check(const char* what, int type, int stream_type, int weight_type, int R, int N) {
  SERL_CHECK_ARG(type >= 0 && type <= 2, "%s: type must be 0 (fp32), 1 (bf16) or 2 (fp16)", what);
  SERL_CHECK_ARG(stream_type == type || stream_type == SERL_F32, "%s: the residual's type must be x's or fp32", what);
  SERL_CHECK_ARG(weight_type == type || weight_type == SERL_F32, "%s: the weight's type must be x's or fp32", what);
  SERL_CHECK_ARG(R >= 0 && R <= RMS_MAXR && N >= 1 && N <= RMS_MAXN, "%s: N must be in [1, %d], R in [0, %d]", what, RMS_MAXN, RMS_MAXR);
  return SERL_OK;
}

extern "C" int serl_rms_norm_fwd(int type, int stream_type, int weight_type, int R, int N, const void* x, long long ldx,
                                 const void* residual, long long ldres, const void* weight, float eps, void* y,
                                 long long ldy, int y_fp8, float* scale, void* sum, long long ldsum, float* rstd,
                                 void* stream) {
  const int bad = rms_check("rms_norm_fwd", type, stream_type, weight_type, R, N);
  if (bad) return bad;
  if (R == 0) return SERL_OK;
  SERL_CHECK_ARG(x && weight && y, "rms_norm_fwd: null pointer");
  SERL_CHECK_ARG((residual != nullptr) == (sum != nullptr), "rms_norm_fwd: residual and sum go together");
  SERL_CHECK_ARG(residual || stream_type == type, "rms_norm_fwd: without a residual its type is x's");
  SERL_CHECK_ARG(!y_fp8 || scale, "rms_norm_fwd: 8-bit output needs the scales' buffer");
  SERL_CHECK_ARG(ldx >= 0 && ldres >= 0 && (R <= 1 || (ldy >= N && (!sum || ldsum >= N))),
                 "rms_norm_fwd: negative row stride, or output rows overlap");
  SERL_CHECK_ARG(R <= 1 || ((y != x || ldy * (y_fp8 ? 1 : sq_size(type)) == ldx * sq_size(type)) && (!sum || sum != residual || ldsum == ldres)),
                 "rms_norm_fwd: in place needs the same row stride");
  const int V = type == SERL_F32 ? 4 : 8;
  const bool wide = N % V == 0 && rms_wide(type, V, x, ldx) && rms_wide(stream_type, V, residual, ldres) &&
                    rms_wide(stream_type, V, sum, ldsum) && sq_aligned(weight, 16) &&
                    (y_fp8 ? sq_aligned(y, V) && ldy % V == 0 : rms_wide(type, V, y, ldy));
  RmsArgs a{};
  a.ldx = ldx; a.ldres = ldres; a.w = weight; a.w_f32 = weight_type == SERL_F32; a.ldy = ldy; a.ldsum = ldsum; a.N = N;
  a.eps = eps;
  hipStream_t st = (hipStream_t)stream;
#define RMS_GO(TX, TR) (y_fp8 ? rms_pick_fwd<TX, TR, true>(a, wide, st) : rms_pick_fwd<TX, TR, false>(a, wide, st))
  for (int first = 0; first < R; first += RMS_LAUNCH) {
    const long long e = sq_size(type), es = sq_size(stream_type);
    a.R = R - first < RMS_LAUNCH ? R - first : RMS_LAUNCH;
    a.x = (const char*)x + first * ldx * e;
    a.res = residual ? (const char*)residual + first * ldres * es : nullptr;
    a.y = (char*)y + first * ldy * (y_fp8 ? 1 : e);
    a.sum = sum ? (char*)sum + first * ldsum * es : nullptr;
    a.scale = scale ? scale + first : nullptr;
    a.rstd_out = rstd ? rstd + first : nullptr;
    if (type == SERL_F32) RMS_GO(F32, F32);
    else if (type == SERL_BF16) { if (stream_type == SERL_F32) RMS_GO(BF16, F32); else RMS_GO(BF16, BF16); }
    else { if (stream_type == SERL_F32) RMS_GO(F16, F32); else RMS_GO(F16, F16); }
  }
#undef RMS_GO
  SERL_CHECK_LAUNCH("rms_norm_fwd");
  return SERL_OK;
}

extern "C" long long serl_rms_norm_bwd_workspace_bytes(int R, int N) {
  if (R < 0 || R > RMS_MAXR || N < 1 || N > RMS_MAXN) {
    serl_set_error("rms_norm_bwd: N must be in [1, %d], R in [0, %d]", RMS_MAXN, RMS_MAXR);
    return -1;
  }
  const int most = rms_parts(R, N, 8);
  return (long long)(most > rms_parts(R, N, 4) ? most : rms_parts(R, N, 4)) * N * 4;
}

extern "C" int serl_rms_norm_bwd(int type, int stream_type, int weight_type, int R, int N, const void* dy, long long lddy,
                                 const void* sum, long long ldsum, const float* rstd, const void* weight, const void* ds,
                                 long long ldds, void* dx, long long lddx, float* dweight, float* workspace,
                                 long long workspace_bytes, void* stream) {
  const int bad = rms_check("rms_norm_bwd", type, stream_type, weight_type, R, N);
  if (bad) return bad;
  SERL_CHECK_ARG(dweight && (R == 0 || (dy && sum && rstd && weight && dx)), "rms_norm_bwd: null pointer");
  SERL_CHECK_ARG(lddy >= 0 && ldsum >= 0 && ldds >= 0 && (R <= 1 || lddx >= N),
                 "rms_norm_bwd: negative row stride, or output rows overlap");
  SERL_CHECK_ARG(R <= 1 || ((dx != ds || lddx == ldds) && (dx != sum || lddx == ldsum)), "rms_norm_bwd: in place needs the same row stride");
  const int V = type == SERL_F32 ? 4 : 8;
  const bool wide = N % V == 0 && rms_wide(type, V, dy, lddy) && rms_wide(stream_type, V, sum, ldsum) &&
                    rms_wide(stream_type, V, ds, ldds) && rms_wide(stream_type, V, dx, lddx) && sq_aligned(weight, 16);
  const int parts = rms_parts(R, N, V);
  const long long need = (long long)parts * N * 4;
  SERL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                 "rms_norm_bwd: workspace of %lld bytes needed, %lld available", need, workspace ? workspace_bytes : 0);
  RmsArgs a{};
  a.x = dy; a.ldx = lddy; a.res = sum; a.ldres = ldsum; a.rstd_in = rstd; a.w = weight; a.w_f32 = weight_type == SERL_F32;
  a.ds = ds; a.ldds = ldds; a.y = dx; a.ldy = lddx; a.part = workspace; a.R = R; a.N = N;
  hipStream_t st = (hipStream_t)stream;
  if (R > 0) {
    if (type == SERL_F32) rms_pick_bwd<F32, F32>(a, wide, st);
    else if (type == SERL_BF16) { if (stream_type == SERL_F32) rms_pick_bwd<BF16, F32>(a, wide, st); else rms_pick_bwd<BF16, BF16>(a, wide, st); }
    else { if (stream_type == SERL_F32) rms_pick_bwd<F16, F32>(a, wide, st); else rms_pick_bwd<F16, F16>(a, wide, st); }
  }
  hipLaunchKernelGGL(rms_dw_kernel, dim3(cdiv(N, 32)), dim3(1024), 0, st, (const float*)workspace, parts, N, dweight);
  SERL_CHECK_LAUNCH("rms_norm_bwd");
  return SERL_OK;
}
