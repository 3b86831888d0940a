// Gated linear recurrence over time, the memory of a sequence policy: per channel
//   f = sigmoid(gate),  h_t = f_t * (start_t ? 0 : h_{t-1}) + (1 - f_t) * x_t,   y_t = h_t
// and its backward pass, and the single step an acting policy takes.  No counterpart in the reference (its policies see
// history through frame stacks only).
//
// The recurrence is an affine map h -> k h + b per step (k = f, or 0 at the start of an episode, or the identity behind
// a sequence's length), and maps compose: (k2, b2) o (k1, b1) = (k1 k2, k2 b1 + b2).  A workgroup of 256 threads takes
// one sequence and 128 bytes of channels (a full line per row) and walks through time in tiles of TC * L steps: a
// thread reads L consecutive rows of 16 bytes, composes them, the maps of the TC threads of a channel are joined by
// wave shuffles and, over the four waves, through LDS (one barrier per tile), and each thread then runs its L steps from
// the state that reaches it.  Every input is read once and every output written once; the next tile's loads are issued
// before the current tile is computed.
#include "seqtypes.h"

#define SCAN_CKPT 128       // steps between the states that the forward pass keeps for the backward pass
#define SCAN_THREADS 256
#define SCAN_MAXSEG 32      // most pieces the time axis is split into

struct ScanArgs {
  const void *gate, *x, *dy;
  long long gate_bs, gate_ts, x_bs, x_ts, dy_bs, dy_ts;      // strides in elements of a sequence and of a step
  void *y, *dgate, *dx;
  long long y_bs, y_ts, dgate_bs, dgate_ts, dx_bs, dx_ts;
  const float *h0, *dh_last;                                 // (B, D) or null
  float *h_last, *dh0;                                       // (B, D)
  const unsigned char* starts; long long starts_bs;          // (B, T) bytes or null
  const int* lengths;                                        // (B) or null
  float *ckpt;                                               // (B, ceil(T / 128), D) or null
  float *seg;                                                // (B, nseg, 2, D): the maps of the pieces, nseg > 1 only
  int B, T, D, ndb, nseg, seg_len;                           // channel blocks; pieces of the time axis and their length
};

// f and 1 - f, both to within 2 ulp: the smaller one is computed, the larger is one minus it (a memory of n steps needs
// 1 - f = 1/n to its full relative precision, and f's rounding unbiased).
__device__ __forceinline__ void scan_gate(float z, float& f, float& rest) {
  const float u = __expf(-fabsf(z));
  const float r = __builtin_amdgcn_rcpf(1.f + u);
  const float small = u * r, big = fmaf(-u, r, 1.f);
  f = z >= 0.f ? big : small;
  rest = z >= 0.f ? small : big;
  if (z != z) f = rest = z;
}

// k c + b where k = 0 cuts whatever c is: an infinity or NaN of one episode ends with it
__device__ __forceinline__ float scan_apply(float k, float c, float b) { return k == 0.f ? b : fmaf(k, c, b); }
__device__ __forceinline__ float scan_times(float k, float kp) { return k == 0.f || kp == 0.f ? 0.f : k * kp; }

__device__ __forceinline__ int scan_len(const ScanArgs& a, int b) {
  if (!a.lengths) return a.T;
  const int n = a.lengths[b];
  return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// state in front of piece `seg`: the maps of the pieces before it applied to h0
template <int VEC>
__device__ __forceinline__ void scan_join_fwd(const ScanArgs& a, int b, int seg, int d0, float (&c)[VEC]) {
  const float* p = a.seg + ((long long)b * a.nseg * 2) * a.D + d0;
#pragma unroll 4
  for (int s = 0; s < seg; ++s, p += 2 * (long long)a.D) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) c[v] = scan_apply(p[v], c[v], p[a.D + v]);
  }
}
// the same from the end: the gradient that leaves piece seg + 1 towards piece `seg`
template <int VEC>
__device__ __forceinline__ void scan_join_bwd(const ScanArgs& a, int b, int seg, int d0, float (&c)[VEC]) {
  const float* p = a.seg + ((long long)b * a.nseg + a.nseg - 1) * 2 * a.D + d0;
#pragma unroll 4
  for (int s = a.nseg - 1; s > seg; --s, p -= 2 * (long long)a.D) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) c[v] = scan_apply(p[v], c[v], p[a.D + v]);
  }
}

// Joins the maps (k, b) of the threads of one channel in the order of time (REV: against it).  In: the thread's own map.
// Out: `in` = the state that reaches the thread's steps when `carry` enters the tile; carry = the state that leaves it.
// Lanes of a wave are (64 / CG) time chunks of CG channel groups; waves follow each other in time.
template <int VEC, int CG, bool REV>
__device__ __forceinline__ void scan_join_tile(float (&k)[VEC], float (&b)[VEC], float (&carry)[VEC], float (&in)[VEC],
                                               float* lds, int wave, int lane) {
#pragma unroll
  for (int o = CG; o < 64; o <<= 1) {
    const bool has = REV ? lane + o < 64 : lane >= o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float kp = REV ? __shfl_down(k[v], o) : __shfl_up(k[v], o);
      const float bp = REV ? __shfl_down(b[v], o) : __shfl_up(b[v], o);
      b[v] = has ? scan_apply(k[v], bp, b[v]) : b[v];
      k[v] = has ? scan_times(k[v], kp) : k[v];
    }
  }
  const int cg = lane & (CG - 1);
  if (REV ? lane < CG : lane >= 64 - CG) {        // the whole wave's map
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      lds[((wave * 2) * VEC + v) * CG + cg] = k[v];
      lds[((wave * 2 + 1) * VEC + v) * CG + cg] = b[v];
    }
  }
  __syncthreads();
  const bool first = REV ? lane + CG >= 64 : lane < CG;
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float ke = REV ? __shfl_down(k[v], CG & 63) : __shfl_up(k[v], CG & 63);
    float be = REV ? __shfl_down(b[v], CG & 63) : __shfl_up(b[v], CG & 63);
    if (first) { ke = 1.f; be = 0.f; }
    float c = carry[v], mine = c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int w = REV ? 3 - i : i;
      mine = w == wave ? c : mine;
      c = scan_apply(lds[((w * 2) * VEC + v) * CG + cg], c, lds[((w * 2 + 1) * VEC + v) * CG + cg]);
    }
    carry[v] = c;
    in[v] = scan_apply(ke, mine, be);
  }
}

// ------------------------------------------------------------------------------------------------------------ forward
// SUMMARY: write the piece's map instead of the outputs (first of two launches when the time axis is split).
template <typename T, int VEC, int CG, int L, bool SUMMARY>
__global__ __launch_bounds__(SCAN_THREADS, 2) void scan_fwd_kernel(const ScanArgs a) {
  constexpr int TC = SCAN_THREADS / CG, TILE = TC * L;
  static_assert(SCAN_CKPT % L == 0, "kept states lie between the chunks of two threads");
  __shared__ float lds[2][4 * 2 * VEC * CG];
  typedef typename T::bits bits;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, cg = tid % CG, tc = tid / CG;
  const int db = blockIdx.x % a.ndb, q = blockIdx.x / a.ndb, seg = q % a.nseg, b = q / a.nseg;
  const int dwant = (db * CG + cg) * VEC;
  const bool dok = dwant < a.D;
  const int d0 = dok ? dwant : 0;
  const int tb = seg * a.seg_len, te = min(a.T, tb + a.seg_len), len = min(te, scan_len(a, b));
  const bits* gate = (const bits*)a.gate + b * a.gate_bs + d0;
  const bits* x = (const bits*)a.x + b * a.x_bs + d0;
  const unsigned char* starts = a.starts ? a.starts + b * a.starts_bs : nullptr;

  float carry[VEC], all[VEC];        // all: product of the piece's k (SUMMARY)
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    carry[v] = !SUMMARY && a.h0 ? a.h0[(long long)b * a.D + d0 + v] : 0.f;
    all[v] = 1.f;
  }
  if (!SUMMARY && a.nseg > 1) scan_join_fwd<VEC>(a, b, seg, d0, carry);

  Raw<T, VEC> rg[L], rx[L];
  unsigned char rs[L];
  const auto fetch = [&](int t0) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      const int t = min(t0 + tc * L + l, te - 1);       // rows behind the piece: its last one again, not used
      rg[l].load(gate + t * a.gate_ts);
      rx[l].load(x + t * a.x_ts);
      rs[l] = starts ? starts[t] : 0;
    }
  };
  fetch(tb);
  int buf = 0;
  for (int t0 = tb; t0 < te; t0 += TILE, buf ^= 1) {
    float k[L][VEC], add[L][VEC];
    const int tt = t0 + tc * L;
    unsigned cut = 0;                    // bit l: an episode starts at the step
#pragma unroll
    for (int l = 0; l < L; ++l) {
      float g[VEC], xv[VEC];
      rg[l].get(g);
      rx[l].get(xv);
      const bool live = tt + l < len;
      cut |= live && rs[l] ? 1u << l : 0u;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float f, rest;
        scan_gate(g[v], f, rest);
        k[l][v] = live ? f : 1.f;
        add[l][v] = live ? rest * xv[v] : 0.f;
      }
    }
    if (t0 + TILE < te) fetch(t0 + TILE);
    float kk[VEC], bb[VEC], c[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { kk[v] = 1.f; bb[v] = 0.f; }
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        bb[v] = cut >> l & 1 ? add[l][v] : fmaf(k[l][v], bb[v], add[l][v]);
        kk[v] *= k[l][v];
      }
#pragma unroll
    for (int v = 0; v < VEC; ++v) kk[v] = cut ? 0.f : kk[v];
    scan_join_tile<VEC, CG, false>(kk, bb, carry, c, lds[buf], wave, lane);
    if constexpr (SUMMARY) {
#pragma unroll
      for (int v = 0; v < VEC; ++v)
#pragma unroll
        for (int w = 0; w < 4; ++w) all[v] = scan_times(lds[buf][((w * 2) * VEC + v) * CG + cg], all[v]);
    } else {
      if (a.ckpt && dok && tt < te && tt % SCAN_CKPT == 0) {
        float* p = a.ckpt + ((long long)b * ((a.T + SCAN_CKPT - 1) / SCAN_CKPT) + tt / SCAN_CKPT) * a.D + d0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) p[v] = c[v];
      }
      bits* y = (bits*)a.y + b * a.y_bs + d0;
#pragma unroll
      for (int l = 0; l < L; ++l) {
        float o[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          c[v] = cut >> l & 1 ? add[l][v] : fmaf(k[l][v], c[v], add[l][v]);
          o[v] = tt + l < len ? c[v] : 0.f;
        }
        Raw<T, VEC> r;
        r.put(o);
        if (dok && tt + l < te) r.store(y + (tt + l) * a.y_ts);
      }
    }
  }
  if (tc == 0 && dok) {
    if constexpr (SUMMARY) {
      float* p = a.seg + ((long long)b * a.nseg + seg) * 2 * a.D + d0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) { p[v] = all[v]; p[a.D + v] = carry[v]; }
    } else if (te == a.T) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) a.h_last[(long long)b * a.D + d0 + v] = carry[v];
    }
  }
}

// ----------------------------------------------------------------------------------------------------------- backward
// With C_t = k_t G_t the gradient that leaves step t backwards in time: G_t = dy_t + C_{t+1}, C_t = k_t (dy_t + C_{t+1}),
// C_T = dh_last, dh0 = C_0; dx = G (1 - f), dgate = G (k_t/f_t h_{t-1} - x) f (1 - f).  h is recomputed from the state that
// the forward pass kept at the tile's first step (in 32 bits, where y was rounded), so y is not read.
template <typename T, int VEC, int CG, int L>
__global__ __launch_bounds__(SCAN_THREADS, 2) void scan_bwd_kernel(const ScanArgs a) {
  constexpr int TC = SCAN_THREADS / CG, TILE = TC * L;
  static_assert(TILE == SCAN_CKPT, "one kept state per tile");
  __shared__ float lds[2][2][4 * 2 * VEC * CG];
  typedef typename T::bits bits;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, cg = tid % CG, tc = tid / CG;
  const int db = blockIdx.x % a.ndb, q = blockIdx.x / a.ndb, seg = q % a.nseg, b = q / a.nseg;
  const int dwant = (db * CG + cg) * VEC;
  const bool dok = dwant < a.D;
  const int d0 = dok ? dwant : 0;
  const int tb = seg * a.seg_len, te = min(a.T, tb + a.seg_len), len = min(te, scan_len(a, b));
  const bits* gate = (const bits*)a.gate + b * a.gate_bs + d0;
  const bits* x = (const bits*)a.x + b * a.x_bs + d0;
  const bits* dy = (const bits*)a.dy + b * a.dy_bs + d0;
  const unsigned char* starts = a.starts ? a.starts + b * a.starts_bs : nullptr;
  const float* ckpt = a.ckpt + (long long)b * ((a.T + SCAN_CKPT - 1) / SCAN_CKPT) * a.D + d0;

  float carry[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) carry[v] = a.dh_last ? a.dh_last[(long long)b * a.D + d0 + v] : 0.f;
  if (a.nseg > 1) scan_join_bwd<VEC>(a, b, seg, d0, carry);

  Raw<T, VEC> rg[L], rx[L], rd[L];
  unsigned char rs[L];
  float kept[VEC];
  const auto fetch = [&](int t0) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      const int t = min(t0 + tc * L + l, te - 1);
      rg[l].load(gate + t * a.gate_ts);
      rx[l].load(x + t * a.x_ts);
      rd[l].load(dy + t * a.dy_ts);
      rs[l] = starts ? starts[t] : 0;
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) kept[v] = ckpt[(long long)(t0 / SCAN_CKPT) * a.D + v];
  };
  const int last = tb + (te - 1 - tb) / TILE * TILE;
  fetch(last);
  int buf = 0;
  for (int t0 = last; t0 >= tb; t0 -= TILE, buf ^= 1) {
    float k[L][VEC], rest[L][VEC], w[L][VEC], d[L][VEC];
    const int tt = t0 + tc * L;
    float kk[VEC], hh[VEC], cc[VEC], h[VEC];
#pragma unroll
    for (int l = 0; l < L; ++l) {        // w: x for now
      float g[VEC];
      rg[l].get(g);
      rx[l].get(w[l]);
      rd[l].get(d[l]);
      const bool live = tt + l < len;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float f, r;
        scan_gate(g[v], f, r);
        k[l][v] = live ? f : 1.f;
        rest[l][v] = live ? r : 0.f;
        w[l][v] = live ? w[l][v] : 0.f;
        d[l][v] = live ? d[l][v] : 0.f;
      }
    }
    unsigned cut = 0;                    // bit l: an episode starts at the step (and the step is live)
#pragma unroll
    for (int l = 0; l < L; ++l) cut |= (rs[l] && tt + l < len) ? 1u << l : 0u;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      kk[v] = 1.f; hh[v] = 0.f; cc[v] = 0.f; h[v] = kept[v];
    }
    if (t0 - TILE >= tb) fetch(t0 - TILE);
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float add = rest[l][v] * w[l][v];
        hh[v] = cut >> l & 1 ? add : fmaf(k[l][v], hh[v], add);
        kk[v] *= k[l][v];
      }
#pragma unroll
    for (int v = 0; v < VEC; ++v) kk[v] = cut ? 0.f : kk[v];
#pragma unroll
    for (int l = L - 1; l >= 0; --l)
#pragma unroll
      for (int v = 0; v < VEC; ++v) cc[v] = cut >> l & 1 ? 0.f : k[l][v] * (d[l][v] + cc[v]);
    float hin[VEC], cin[VEC], k2[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) k2[v] = kk[v];
    scan_join_tile<VEC, CG, false>(kk, hh, h, hin, lds[buf][0], wave, lane);
    scan_join_tile<VEC, CG, true>(k2, cc, carry, cin, lds[buf][1], wave, lane);
    // forwards: h_{t-1} of every step, folded at once into w = (h_{t-1} - x) f (1 - f)
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float hp = cut >> l & 1 ? 0.f : hin[v], xv = w[l][v], r = rest[l][v], f = k[l][v];
        w[l][v] = (hp - xv) * (f * r);
        hin[v] = fmaf(f, hp, r * xv);
      }
    // backwards
    bits* dgate = (bits*)a.dgate + b * a.dgate_bs + d0;
    bits* dx = (bits*)a.dx + b * a.dx_bs + d0;
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      float og[VEC], ox[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float G = d[l][v] + cin[v];
        og[v] = tt + l < len ? G * w[l][v] : 0.f;
        ox[v] = tt + l < len ? G * rest[l][v] : 0.f;
        cin[v] = cut >> l & 1 ? 0.f : k[l][v] * G;
      }
      Raw<T, VEC> r;
      if (dok && tt + l < te) {
        r.put(og);
        r.store(dgate + (tt + l) * a.dgate_ts);
        r.put(ox);
        r.store(dx + (tt + l) * a.dx_ts);
      }
    }
  }
  if (seg == 0 && tc == 0 && dok) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) a.dh0[(long long)b * a.D + d0 + v] = carry[v];
  }
}

// The map of a piece for the backward direction: C entering from the right -> C leaving to the left (reads gate and dy).
template <typename T, int VEC, int CG, int L>
__global__ __launch_bounds__(SCAN_THREADS, 2) void scan_bwd_summary_kernel(const ScanArgs a) {
  constexpr int TC = SCAN_THREADS / CG, TILE = TC * L;
  __shared__ float lds[2][4 * 2 * VEC * CG];
  typedef typename T::bits bits;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, cg = tid % CG, tc = tid / CG;
  const int db = blockIdx.x % a.ndb, q = blockIdx.x / a.ndb, seg = q % a.nseg, b = q / a.nseg;
  const int dwant = (db * CG + cg) * VEC;
  const bool dok = dwant < a.D;
  const int d0 = dok ? dwant : 0;
  const int tb = seg * a.seg_len, te = min(a.T, tb + a.seg_len), len = min(te, scan_len(a, b));
  const bits* gate = (const bits*)a.gate + b * a.gate_bs + d0;
  const bits* dy = (const bits*)a.dy + b * a.dy_bs + d0;
  const unsigned char* starts = a.starts ? a.starts + b * a.starts_bs : nullptr;
  float carry[VEC], all[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) { carry[v] = 0.f; all[v] = 1.f; }
  Raw<T, VEC> rg[L], rd[L];
  unsigned char rs[L];
  const auto fetch = [&](int t0) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      const int t = min(t0 + tc * L + l, te - 1);
      rg[l].load(gate + t * a.gate_ts);
      rd[l].load(dy + t * a.dy_ts);
      rs[l] = starts ? starts[t] : 0;
    }
  };
  const int last = tb + (te - 1 - tb) / TILE * TILE;
  fetch(last);
  int buf = 0;
  for (int t0 = last; t0 >= tb; t0 -= TILE, buf ^= 1) {
    const int tt = t0 + tc * L;
    float kk[VEC], cc[VEC], in[VEC];
    bool cuts = false;
#pragma unroll
    for (int v = 0; v < VEC; ++v) { kk[v] = 1.f; cc[v] = 0.f; }
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      float g[VEC], d[VEC];
      rg[l].get(g);
      rd[l].get(d);
      const bool live = tt + l < len, cut = live && rs[l];
      cuts |= cut;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float f, r;
        scan_gate(g[v], f, r);
        f = live ? f : 1.f;
        cc[v] = cut ? 0.f : f * ((live ? d[v] : 0.f) + cc[v]);
        kk[v] *= f;
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) kk[v] = cuts ? 0.f : kk[v];
    if (t0 - TILE >= tb) fetch(t0 - TILE);
    scan_join_tile<VEC, CG, true>(kk, cc, carry, in, lds[buf], wave, lane);
#pragma unroll
    for (int v = 0; v < VEC; ++v)
#pragma unroll
      for (int w = 0; w < 4; ++w) all[v] = scan_times(lds[buf][((w * 2) * VEC + v) * CG + cg], all[v]);
  }
  if (tc == 0 && dok) {
    float* p = a.seg + ((long long)b * a.nseg + seg) * 2 * a.D + d0;
#pragma unroll
    for (int v = 0; v < VEC; ++v) { p[v] = all[v]; p[a.D + v] = carry[v]; }
  }
}

// ---------------------------------------------------------------------------------------------------- a few steps
// One thread per VEC channels of a sequence runs the steps in order: acting (T = 1), or windows too short for a tile.
template <typename T, int VEC>
__global__ __launch_bounds__(SCAN_THREADS) void scan_short_kernel(const ScanArgs a) {
  typedef typename T::bits bits;
  const long long i = (long long)blockIdx.x * SCAN_THREADS + threadIdx.x;
  const int b = (int)(i / a.ndb), d0 = (int)(i % a.ndb) * VEC;
  if (b >= a.B) return;
  float h[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) h[v] = a.h0 ? a.h0[(long long)b * a.D + d0 + v] : 0.f;
  const int len = scan_len(a, b);
  for (int t = 0; t < a.T; ++t) {
    if (a.ckpt && t % SCAN_CKPT == 0) {
      float* p = a.ckpt + ((long long)b * ((a.T + SCAN_CKPT - 1) / SCAN_CKPT) + t / SCAN_CKPT) * a.D + d0;
#pragma unroll
      for (int v = 0; v < VEC; ++v) p[v] = h[v];
    }
    Raw<T, VEC> rg, rx;
    rg.load((const bits*)a.gate + b * a.gate_bs + t * a.gate_ts + d0);
    rx.load((const bits*)a.x + b * a.x_bs + t * a.x_ts + d0);
    const bool cut = a.starts && a.starts[b * a.starts_bs + t];
    float g[VEC], xv[VEC], o[VEC];
    rg.get(g);
    rx.get(xv);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float f, rest;
      scan_gate(g[v], f, rest);
      const float n = fmaf(f, cut ? 0.f : h[v], rest * xv[v]);
      h[v] = t < len ? n : h[v];
      o[v] = t < len ? n : 0.f;
    }
    rx.put(o);
    rx.store((bits*)a.y + b * a.y_bs + t * a.y_ts + d0);
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) a.h_last[(long long)b * a.D + d0 + v] = h[v];
}

// ---------------------------------------------------------------------------------------------------------- host side
struct ScanPlan { int vec, cg, ndb, nseg, seg_len; };
// wide: rows of whole 16-byte pieces.  The time axis is split (two launches, gate and x read twice) only when sequences
// and channels alone give fewer workgroups than there are CUs.
static ScanPlan scan_plan(int type, int B, int T, int D, bool wide) {
  ScanPlan p;
  p.vec = !wide ? 1 : type == SERL_F32 ? 4 : 8;
  p.cg = wide ? 8 : 64;
  p.ndb = cdiv(D, p.vec * p.cg);
  p.nseg = 1;
  p.seg_len = T;
  const long long blocks = (long long)B * p.ndb;
  if (blocks < 256 && T > 1024) {
    const int want = (int)cdivll(512, blocks);
    p.seg_len = cdiv(cdiv(T, want < SCAN_MAXSEG ? want : SCAN_MAXSEG), 512) * 512;
    p.nseg = cdiv(T, p.seg_len);
  }
  return p;
}

static long long scan_ws(const ScanPlan& p, int B, int D) { return p.nseg > 1 ? (long long)B * p.nseg * 2 * D * 4 : 0; }

extern "C" long long serl_gated_scan_workspace_bytes(int type, int B, int T, int D) {
  if (type < 0 || type > 2 || B < 0 || T < 0 || D < 0) {
    serl_set_error("gated_scan: bad type or sizes");
    return -1;
  }
  if (B == 0 || D == 0) return 0;
  const long long w = scan_ws(scan_plan(type, B, T, D, true), B, D), n = scan_ws(scan_plan(type, B, T, D, false), B, D);
  return w > n ? w : n;
}

extern "C" long long serl_gated_scan_states_floats(int B, int T, int D) {
  if (B < 0 || T < 0 || D < 0) {
    serl_set_error("gated_scan: bad sizes");
    return -1;
  }
  return (long long)B * cdivll(T, SCAN_CKPT) * D;
}

static bool scan_wide(int type, int D, const void* p, long long bs, long long ts) {
  const int vec = type == SERL_F32 ? 4 : 8;
  return D % vec == 0 && bs % vec == 0 && ts % vec == 0 && sq_aligned(p, 16);
}

template <typename T>
static void scan_launch_fwd(const ScanArgs& a, const ScanPlan& p, hipStream_t st) {
  constexpr int W = T::code == SERL_F32 ? 4 : 8;
  const dim3 grid((unsigned)((long long)a.B * a.nseg * a.ndb)), blk(SCAN_THREADS);
  if (p.vec == 1) {
    if (a.nseg > 1) hipLaunchKernelGGL((scan_fwd_kernel<T, 1, 64, 32, true>), grid, blk, 0, st, a);
    hipLaunchKernelGGL((scan_fwd_kernel<T, 1, 64, 32, false>), grid, blk, 0, st, a);
  } else {
    if (a.nseg > 1) hipLaunchKernelGGL((scan_fwd_kernel<T, W, 8, 4, true>), grid, blk, 0, st, a);
    hipLaunchKernelGGL((scan_fwd_kernel<T, W, 8, 4, false>), grid, blk, 0, st, a);
  }
}
template <typename T>
static void scan_launch_bwd(const ScanArgs& a, const ScanPlan& p, hipStream_t st) {
  constexpr int W = T::code == SERL_F32 ? 4 : 8;
  const dim3 grid((unsigned)((long long)a.B * a.nseg * a.ndb)), blk(SCAN_THREADS);
  if (p.vec == 1) {
    if (a.nseg > 1) hipLaunchKernelGGL((scan_bwd_summary_kernel<T, 1, 64, 32>), grid, blk, 0, st, a);
    hipLaunchKernelGGL((scan_bwd_kernel<T, 1, 64, 32>), grid, blk, 0, st, a);
  } else {
    if (a.nseg > 1) hipLaunchKernelGGL((scan_bwd_summary_kernel<T, W, 8, 4>), grid, blk, 0, st, a);
    hipLaunchKernelGGL((scan_bwd_kernel<T, W, 8, 4>), grid, blk, 0, st, a);
  }
}
template <typename T>
static void scan_launch_short(ScanArgs a, bool wide, hipStream_t st) {
  constexpr int W = T::code == SERL_F32 ? 4 : 8;
  a.ndb = wide ? a.D / W : a.D;
  const dim3 grid((unsigned)cdivll((long long)a.B * a.ndb, SCAN_THREADS)), blk(SCAN_THREADS);
  if (wide) hipLaunchKernelGGL((scan_short_kernel<T, W>), grid, blk, 0, st, a);
  else hipLaunchKernelGGL((scan_short_kernel<T, 1>), grid, blk, 0, st, a);
}

#define SCAN_SHORT 8        // up to this many steps one thread runs them in order: a tile of 128 would be mostly empty

extern "C" int serl_gated_scan_fwd(int type, int B, int T, int D, const void* gate, long long gate_bs, long long gate_ts,
                                   const void* x, long long x_bs, long long x_ts, const float* h0,
                                   const unsigned char* starts, long long starts_bs, const int* lengths, void* y,
                                   long long y_bs, long long y_ts, float* h_last, float* states, float* workspace,
                                   long long workspace_bytes, void* stream) {
  SERL_CHECK_ARG(type >= 0 && type <= 2, "gated_scan_fwd: type must be 0 (fp32), 1 (bf16) or 2 (fp16)");
  SERL_CHECK_ARG(B >= 0 && T >= 0 && D >= 0, "gated_scan_fwd: negative size");
  if (B == 0 || D == 0) return SERL_OK;
  SERL_CHECK_ARG(h_last && (T == 0 || (gate && x && y)), "gated_scan_fwd: null pointer");
  SERL_CHECK_ARG(gate_bs >= 0 && gate_ts >= 0 && x_bs >= 0 && x_ts >= 0 && (!starts || starts_bs >= 0),
                 "gated_scan_fwd: negative stride");
  SERL_CHECK_ARG((T <= 1 || y_ts >= D) && (T == 0 || B <= 1 || y_bs >= D), "gated_scan_fwd: rows of y overlap");
  SERL_CHECK_ARG(T < 0x7fff0000, "gated_scan_fwd: T too large");
  const bool wide = scan_wide(type, D, gate, gate_bs, gate_ts) && scan_wide(type, D, x, x_bs, x_ts) &&
                    scan_wide(type, D, y, y_bs, y_ts);
  const ScanPlan p = scan_plan(type, B, T, D, wide);
  SERL_CHECK_ARG((long long)B * p.nseg * p.ndb <= 0x7fffffffll && (long long)B * D <= 0x7fffffffll * SCAN_THREADS,
                 "gated_scan_fwd: B * D too large");
  ScanArgs a{};
  a.gate = gate; a.gate_bs = gate_bs; a.gate_ts = gate_ts; a.x = x; a.x_bs = x_bs; a.x_ts = x_ts;
  a.y = y; a.y_bs = y_bs; a.y_ts = y_ts; a.h0 = h0; a.h_last = h_last; a.starts = starts; a.starts_bs = starts_bs;
  a.lengths = lengths; a.ckpt = states; a.B = B; a.T = T; a.D = D;
  a.ndb = p.ndb; a.nseg = p.nseg; a.seg_len = p.seg_len; a.seg = workspace;
  hipStream_t st = (hipStream_t)stream;
  if (T <= SCAN_SHORT) {
    if (type == SERL_F32) scan_launch_short<F32>(a, wide, st);
    else if (type == SERL_BF16) scan_launch_short<BF16>(a, wide, st);
    else scan_launch_short<F16>(a, wide, st);
  } else {
    const long long need = scan_ws(p, B, D);
    SERL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                   "gated_scan_fwd: workspace of %lld bytes needed, %lld available", need, workspace ? workspace_bytes : 0);
    if (type == SERL_F32) scan_launch_fwd<F32>(a, p, st);
    else if (type == SERL_BF16) scan_launch_fwd<BF16>(a, p, st);
    else scan_launch_fwd<F16>(a, p, st);
  }
  SERL_CHECK_LAUNCH("gated_scan_fwd");
  return SERL_OK;
}

extern "C" int serl_gated_scan_bwd(int type, int B, int T, int D, const void* gate, long long gate_bs, long long gate_ts,
                                   const void* x, long long x_bs, long long x_ts, const unsigned char* starts,
                                   long long starts_bs, const int* lengths, const float* states, const void* dy,
                                   long long dy_bs, long long dy_ts, const float* dh_last, void* dgate,
                                   long long dgate_bs, long long dgate_ts, void* dx, long long dx_bs, long long dx_ts,
                                   float* dh0, float* workspace, long long workspace_bytes, void* stream) {
  SERL_CHECK_ARG(type >= 0 && type <= 2, "gated_scan_bwd: type must be 0 (fp32), 1 (bf16) or 2 (fp16)");
  SERL_CHECK_ARG(B >= 0 && T >= 1 && D >= 0, "gated_scan_bwd: bad size (T must be >= 1)");
  if (B == 0 || D == 0) return SERL_OK;
  SERL_CHECK_ARG(gate && x && states && dy && dgate && dx && dh0, "gated_scan_bwd: null pointer");
  SERL_CHECK_ARG(gate_bs >= 0 && gate_ts >= 0 && x_bs >= 0 && x_ts >= 0 && dy_bs >= 0 && dy_ts >= 0 &&
                 (!starts || starts_bs >= 0), "gated_scan_bwd: negative stride");
  SERL_CHECK_ARG((T <= 1 || (dgate_ts >= D && dx_ts >= D)) && (B <= 1 || (dgate_bs >= D && dx_bs >= D)),
                 "gated_scan_bwd: rows of dgate or dx overlap");
  SERL_CHECK_ARG(T < 0x7fff0000, "gated_scan_bwd: T too large");
  const bool wide = scan_wide(type, D, gate, gate_bs, gate_ts) && scan_wide(type, D, x, x_bs, x_ts) &&
                    scan_wide(type, D, dy, dy_bs, dy_ts) && scan_wide(type, D, dgate, dgate_bs, dgate_ts) &&
                    scan_wide(type, D, dx, dx_bs, dx_ts);
  const ScanPlan p = scan_plan(type, B, T, D, wide);
  SERL_CHECK_ARG((long long)B * p.nseg * p.ndb <= 0x7fffffffll, "gated_scan_bwd: B * D too large");
  const long long need = scan_ws(p, B, D);
  SERL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                 "gated_scan_bwd: workspace of %lld bytes needed, %lld available", need, workspace ? workspace_bytes : 0);
  ScanArgs a{};
  a.gate = gate; a.gate_bs = gate_bs; a.gate_ts = gate_ts; a.x = x; a.x_bs = x_bs; a.x_ts = x_ts;
  a.dy = dy; a.dy_bs = dy_bs; a.dy_ts = dy_ts; a.dh_last = dh_last; a.starts = starts; a.starts_bs = starts_bs;
  a.lengths = lengths; a.ckpt = const_cast<float*>(states); a.dgate = dgate; a.dgate_bs = dgate_bs; a.dgate_ts = dgate_ts;
  a.dx = dx; a.dx_bs = dx_bs; a.dx_ts = dx_ts; a.dh0 = dh0; a.B = B; a.T = T; a.D = D;
  a.ndb = p.ndb; a.nseg = p.nseg; a.seg_len = p.seg_len; a.seg = workspace;
  hipStream_t st = (hipStream_t)stream;
  if (type == SERL_F32) scan_launch_bwd<F32>(a, p, st);
  else if (type == SERL_BF16) scan_launch_bwd<BF16>(a, p, st);
  else scan_launch_bwd<F16>(a, p, st);
  SERL_CHECK_LAUNCH("gated_scan_bwd");
  return SERL_OK;
}
