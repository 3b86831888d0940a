// Gated linear recurrence over time, the memory of a sequence policy: per channel
//   f = sigmoid(gate),  h_t = f_t * (start_t ? 0 : h_{t-1}) + (1 - f_t) * x_t,   y_t = h_t
// and its backward pass, and the single step an acting policy takes.  No counterpart in the reference (its policies see
// history through frame stacks only).
//
// The recurrence is an affine map h -> k h + b per step (k = f, or 0 at the start of an episode, or the identity behind
// a sequence's length), and maps compose: (k2, b2) o (k1, b1) = (k1 k2, k2 b1 + b2).  A workgroup takes one sequence and 128
// bytes of channels (a cache line per row; 64 bytes were 10 % slower) and walks through time in tiles of up to 128 steps: a thread
// reads 4 channels of 4 consecutive steps, composes them, the maps of the threads of a channel are joined by wave shuffles and,
// between the waves, through LDS (one barrier per direction and tile), and each thread then runs its steps from the state that
// reaches it.  Every input is read once and every output written once; the next tile's loads are issued before the current tile
// is joined.  16 elements per thread: with 32 the kernels were 10 to 20 % slower (registers, too few waves).
//
// Bound by memory and, to half, by the vector ALU (26 instructions per element forward, 46 backward).  8 x 4096 x 2048 bf16:
// forward 95 us (4.2 TB/s where a large copy reaches 5.2), backward 164 us (4.1 TB/s).
#include "seqtypes.h"

#define SCAN_CKPT 64        // steps between the states that the forward pass keeps for the backward pass
#define SCAN_TILE 128       // steps of a tile where the time axis may be split
#define SCAN_THREADS 256    // of the kernel for a few steps
#define SCAN_MAXD (1 << 26)  // channels
#define SCAN_MAXT 0x7fff0000 // steps: a step and the tile behind it fit 31 bits
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
  float *ckpt;                                               // (B, ceil(T / 64), D) or null
  float *seg;                                                // (B, nseg, 2, D): the maps of the pieces, nseg > 1 only
  int B, T, D, ndb, nseg, seg_len;                           // channel blocks; pieces of the time axis and their length
  int share;                                                 // rows start inside cache lines
};

// f and 1 - f, each to a few roundings of its own size plus that of the exponent, |z| 2^-24: a memory of n steps needs 1 - f = 1/n
// to its relative precision, and f's rounding unbiased, so f above a half is one minus the other.  z = +inf: f = 1, 1 - f = 0.
__device__ __forceinline__ void scan_gate(float z, float& f, float& rest) {
  const float e = __expf(z);
  rest = __builtin_amdgcn_rcpf(1.f + e);
  f = z > 0.f ? 1.f - rest : e * rest;
}

// The k of a map of several steps is 0 where an episode starts in them and only there: k c + b then cuts whatever c is (0 * NaN = 0 in the
// legacy product), so an infinity or NaN of one episode ends with it.  Products of gates alone stay at SCAN_LEAST, fp32's smallest
// number, or above it, however many (0.9^1000 is below it), so that elsewhere an infinity or NaN reaches every later step; of a finite
// state c it leaves 1.4e-45 c, less than 5e-7 of the largest.
#define SCAN_LEAST 0x1p-149f
__device__ __forceinline__ float scan_apply(float k, float c, float b) {
  float r;
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(k), "v"(c));
  return r + b;
}
// k2 k1: 0 if one of them is, else at least SCAN_LEAST
__device__ __forceinline__ float scan_times(float k2, float k1) {
  float r, p = k2 * k1;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(k2), "v"(k1), "s"(SCAN_LEAST));
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(p), "v"(r));
  return r;
}

__device__ __forceinline__ int scan_len(const ScanArgs& a, int b) {
  if (!a.lengths) return a.T;
  const int n = a.lengths[b];
  return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// state in front of piece `seg` for channel ch: the maps of the pieces before it applied to h0
__device__ __forceinline__ float scan_join_fwd(const ScanArgs& a, int b, int seg, int ch, float c) {
  const float* p = a.seg + ((long long)b * a.nseg * 2) * a.D + ch;
#pragma unroll 4
  for (int s = 0; s < seg; ++s, p += 2 * (long long)a.D) c = scan_apply(p[0], c, p[a.D]);
  return c;
}
// the same from the end: the gradient that leaves piece seg + 1 towards piece `seg`
__device__ __forceinline__ float scan_join_bwd(const ScanArgs& a, int b, int seg, int ch, float c) {
  const float* p = a.seg + ((long long)b * a.nseg + a.nseg - 1) * 2 * a.D + ch;
#pragma unroll 4
  for (int s = a.nseg - 1; s > seg; --s, p -= 2 * (long long)a.D) c = scan_apply(p[0], c, p[a.D]);
  return c;
}

// a thread's own product of gates, before its starts are looked at
template <int VEC> __device__ __forceinline__ void scan_floor(float (&k)[VEC]) {
#pragma unroll
  for (int v = 0; v < VEC; ++v) k[v] = fmaxf(k[v], SCAN_LEAST);
}

// Joins the maps (k, b) of the threads of one channel in the order of time (REV: against it).  In: the thread's own map.
// Out: `in` = the state that reaches the thread's steps when the tile is entered with `carry`; carry = the state that leaves
// it, all = the product of k so far.  Lanes of a wave are (64 / CG) time chunks of CG channel groups; waves follow each other
// in time.  Between waves every wave walks the maps of all of them, one channel per lane (`carry` and `all` are kept so).
template <int VEC, int CG, int WAVES, bool REV>
__device__ __forceinline__ void scan_join_tile(float (&k)[VEC], float (&b)[VEC], float& carry, float& all, float (&in)[VEC],
                                               float* lds, int wave, int lane) {
  constexpr int CH = VEC * CG;
  static_assert(CH <= 64, "a lane per channel");
#pragma unroll
  for (int o = CG; o < 64; o <<= 1) {
    const bool has = REV ? lane + o < 64 : lane >= o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      const float kp = REV ? __shfl_down(k[v], o) : __shfl_up(k[v], o);
      const float bp = REV ? __shfl_down(b[v], o) : __shfl_up(b[v], o);
      const float bj = scan_apply(k[v], bp, b[v]), kj = scan_times(k[v], kp);      // unconditional: no branch per lane
      b[v] = has ? bj : b[v];
      k[v] = has ? kj : k[v];
    }
  }
  const int c0 = (lane & (CG - 1)) * VEC;
  if (REV ? lane < CG : lane >= 64 - CG) {        // the whole wave's map
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      lds[wave * 2 * CH + c0 + v] = k[v];
      lds[(wave * 2 + 1) * CH + c0 + v] = b[v];
    }
  }
  __syncthreads();
  float own = carry;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const int w = REV ? WAVES - 1 - i : i;
    const float kw = lds[w * 2 * CH + (lane & (CH - 1))], bw = lds[(w * 2 + 1) * CH + (lane & (CH - 1))];
    own = w == wave ? carry : own;
    carry = scan_apply(kw, carry, bw);
    all = scan_times(kw, all);
  }
  const bool first = REV ? lane + CG >= 64 : lane < CG;
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    in[v] = VEC == 1 && CG == 64 ? own : __shfl(own, c0 + v);
    if (CG < 64) {
      const float ke = REV ? __shfl_down(k[v], CG & 63) : __shfl_up(k[v], CG & 63);
      const float be = REV ? __shfl_down(b[v], CG & 63) : __shfl_up(b[v], CG & 63);
      const float j = scan_apply(ke, in[v], be);
      in[v] = first ? in[v] : j;
    }
  }
}

// What a thread of the tile kernels is: VEC channels from d0 on, L steps of every tile; a wave's steps are 64 / CG * L rows.
// Where D is no multiple of VEC the last thread's channels are the row's last VEC: some it has in common with the thread
// before, and both compute and store the same bits for those.
template <int VEC, int CG, int L>
struct ScanSpot {
  static constexpr int ROWS = 64 / CG * L;
  int wave, lane, first, d0, seg, b, tb, te, len;      // first: the thread's first step within its wave's
  int ch;                                              // the one channel of the lane (states, maps of pieces), in range
  bool dok, chok;                                      // chok: wave 0 writes channel ch
  __device__ __forceinline__ explicit ScanSpot(const ScanArgs& a) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    first = lane / CG * L;
    // Workgroups go to the 8 XCDs in turn.  Where rows start inside a cache line, neighbours in channels share lines and are
    // kept on one XCD, in its cache (64 x 512 x 1001 fp32 both ways 336 -> 266 us); else in turn is better (16 x 1024 x 2048
    // fp32 267 -> 236 us).
    const int n = gridDim.x, xcd = blockIdx.x % 8;
    const int id = a.share ? xcd * (n / 8) + min(xcd, n % 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
    const int db = id % a.ndb, q = id / a.ndb, want = (db * CG + lane % CG) * VEC;
    seg = q % a.nseg;
    b = q / a.nseg;
    dok = want < a.D;
    d0 = dok ? min(want, a.D - VEC) : 0;
    const int slot = lane % (CG * VEC), group = (db * CG + slot / VEC) * VEC;
    ch = min(group, a.D - VEC) + slot % VEC;
    chok = wave == 0 && lane < CG * VEC && group < a.D;
    tb = seg * a.seg_len;
    te = tb + min(a.seg_len, a.T - tb);
    len = min(te, scan_len(a, b));
  }
};

// One (B, T, D) tensor as a wave sees it: `base` is its sequence (uniform), `off` the thread's byte offset from its wave's
// first row, or behind everything for channels that do not exist.  FAR (VEC = 1, where a wave's rows are one thread's):
// steps may lie any distance apart; beyond 2^27 bytes each row is addressed by itself (done always, narrow rows took 1.3 to 1.7 times as long).
template <typename T, int VEC, int L, typename Spot, bool FAR = false>
struct ScanRows {
  const char* base;
  long long ts;          // bytes from step to step
  uint32_t off;
  __device__ __forceinline__ bool far() const { return FAR && VEC == 1 && ts > 1 << 27; }
  __device__ __forceinline__ ScanRows(const Spot& me, const void* p, long long bs, long long step) {
    constexpr int E = sizeof(typename T::bits);
    base = (const char*)p + me.b * bs * E;
    ts = step * E;
    static_assert(VEC > 1 || (Spot::ROWS == L && L <= 8), "a wave's rows are each thread's; seven steps and a row are below 2^31 bytes");
    off = me.dok ? (uint32_t)(me.first * ts) + (uint32_t)(me.d0 * E) : SQ_NOWHERE;
  }
  // the wave's rows from step t on, as far as they are before `te` (a row is D wide)
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(int t, int te, int D) const {
    const int rows = min(te - t, Spot::ROWS);
    return sq_buffer(base + t * ts, rows > 0 ? (int)((uint32_t)(rows - 1) * (uint32_t)ts + (uint32_t)(D * (int)sizeof(typename T::bits))) : 0);
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t one(int t, int te, int D) const {
    return sq_buffer(base + t * ts, t < te ? D * (int)sizeof(typename T::bits) : 0);
  }
  template <bool STREAM = false> __device__ __forceinline__ void fetch(Raw<T, VEC> (&r)[L], int t, int te, int D) const {
    if (far()) {
#pragma unroll
      for (int l = 0; l < L; ++l) sq_load<STREAM>(r[l], one(t + l, te, D), off);
    } else {
      const __amdgpu_buffer_rsrc_t b = at(t, te, D);
#pragma unroll
      for (int l = 0; l < L; ++l) sq_load<STREAM>(r[l], b, off + l * (uint32_t)ts);
    }
  }
  // row l of those from step t on, `b` = at(t, te, D)
  template <bool STREAM> __device__ __forceinline__ void put(const Raw<T, VEC>& r, __amdgpu_buffer_rsrc_t b, int l, int t, int te, int D) const {
    if (far()) sq_store<STREAM>(r, one(t + l, te, D), off);
    else sq_store<STREAM>(r, b, off + l * (uint32_t)ts);
  }
};

// The starts of a thread's steps, one byte per lane: every thread of a time chunk loads one, scan_cuts collects them.
template <int CG, int L>
__device__ __forceinline__ unsigned char scan_start(const unsigned char* starts, int t, int te, int lane) {
  static_assert(L <= CG, "a chunk's starts fit its lanes");
  return starts ? starts[min(t + (lane & (CG - 1) & (L - 1)), te - 1)] : 0;
}
template <int CG, int L>
__device__ __forceinline__ unsigned scan_cuts(unsigned char start, int t, int len, int lane) {
  const unsigned long long all = __ballot(start != 0);
  const unsigned bits = (unsigned)(all >> (lane & ~(CG - 1))) & (L == 32 ? ~0u : (1u << (L & 31)) - 1u);
  const int live = len - t;            // steps at and behind the length start nothing
  return live >= L ? bits : live <= 0 ? 0u : bits & ((1u << live) - 1u);
}
// v = value where a step starts an episode (its k is 0, but k v + b would carry on a NaN of v)
// (the empty asm keeps the compiler from running these rare blocks always, as selects)
template <int VEC> __device__ __forceinline__ void scan_cut(float (&v)[VEC], bool cut, float value) {
  asm volatile("");
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = cut ? value : v[i];
}
template <int VEC> __device__ __forceinline__ void scan_cut(float (&v)[VEC], bool cut, const float (&value)[VEC]) {
  asm volatile("");
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = cut ? value[i] : v[i];
}
// value `keep ? r : fill` of every element (fill: the bits of a pair of 16-bit or of one 32-bit element)
template <typename T, int VEC>
__device__ __forceinline__ void scan_mask(Raw<T, VEC>& r, bool keep, uint32_t fill) {
  asm volatile("");
  if constexpr (VEC == 1) {
    r.w = keep ? r.w : (typename T::bits)fill;
  } else {
#pragma unroll
    for (int i = 0; i < Raw<T, VEC>::W; ++i) r.w[i] = keep ? r.w[i] : fill;
  }
}
template <typename T> __device__ __forceinline__ uint32_t scan_inf() {       // a gate of +inf: f = 1, the state is held
  return T::code == SERL_F32 ? 0x7f800000u : T::code == SERL_BF16 ? 0x7f807f80u : 0x7c007c00u;
}

// ------------------------------------------------------------------------------------------------------------ forward
// SUMMARY: write the piece's map instead of the outputs (first of two launches when the time axis is split).  STREAM: 1 the inputs, 2
// the outputs pass by the caches.
template <typename T, int VEC, int CG, int L, int THREADS, bool SUMMARY, int STREAM>
__global__ __launch_bounds__(THREADS) void scan_fwd_kernel(const ScanArgs a) {
  constexpr int TC = THREADS / CG, TILE = TC * L, WAVES = THREADS / 64;
  static_assert(SCAN_CKPT % L == 0, "kept states lie between the chunks of two threads");
  __shared__ __attribute__((aligned(16))) float lds[2][WAVES * 2 * VEC * CG];
  typedef ScanSpot<VEC, CG, L> Spot;
  const Spot me(a);
  typedef ScanRows<T, VEC, L, Spot> Rows;
  const Rows gate(me, a.gate, a.gate_bs, a.gate_ts), x(me, a.x, a.x_bs, a.x_ts), y(me, a.y, a.y_bs, a.y_ts);
  const unsigned char* starts = a.starts ? a.starts + me.b * a.starts_bs : nullptr;

  const long long state = (long long)me.b * a.D + me.ch;
  float all = 1.f, carry = !SUMMARY && a.h0 ? a.h0[state] : 0.f;      // all: product of the piece's k (SUMMARY)
  if (!SUMMARY && a.nseg > 1) carry = scan_join_fwd(a, me.b, me.seg, me.ch, carry);

  Raw<T, VEC> rg[L], rx[L];
  int tw = me.tb + me.wave * me.ROWS, buf = 0;          // the wave's first step of the tile
  gate.template fetch<STREAM == 1>(rg, tw, me.te, a.D);
  x.template fetch<STREAM == 1>(rx, tw, me.te, a.D);
  unsigned char rs = scan_start<CG, L>(starts, tw + me.first, me.te, me.lane);
  for (int t0 = me.tb; t0 < me.te; t0 += TILE, tw += TILE, buf ^= 1) {
    const int t = tw + me.first;
    const bool whole = t0 + TILE <= me.len;               // every step is before the sequence's length
    const unsigned cut = scan_cuts<CG, L>(rs, t, me.len, me.lane);
    const bool cuts = __any(cut != 0);                    // rare: an episode starts in the wave's steps
    float k[L][VEC], add[L][VEC], kk[VEC], bb[VEC], c[VEC];
#pragma unroll
    for (int l = 0; l < L; ++l) {
      if (!whole) {
        scan_mask(rg[l], t + l < me.len, scan_inf<T>());
        scan_mask(rx[l], t + l < me.len, 0);
      }
      float g[VEC], xv[VEC];
      rg[l].get(g);
      rx[l].get(xv);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float rest;
        scan_gate(g[v], k[l][v], rest);
        add[l][v] = rest * xv[v];
      }
      if (cuts) scan_cut<VEC>(k[l], cut >> l & 1, 0.f);
    }
    gate.template fetch<STREAM == 1>(rg, tw + TILE, me.te, a.D);
    x.template fetch<STREAM == 1>(rx, tw + TILE, me.te, a.D);
    rs = scan_start<CG, L>(starts, t + TILE, me.te, me.lane);
#pragma unroll
    for (int v = 0; v < VEC; ++v) { kk[v] = k[0][v]; bb[v] = add[0][v]; }
#pragma unroll
    for (int l = 1; l < L; ++l) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        bb[v] = fmaf(k[l][v], bb[v], add[l][v]);
        kk[v] *= k[l][v];
      }
      if (cuts) scan_cut<VEC>(bb, cut >> l & 1, add[l]);
    }
    scan_floor<VEC>(kk);
    if (cuts) scan_cut<VEC>(kk, cut != 0, 0.f);
    scan_join_tile<VEC, CG, WAVES, false>(kk, bb, carry, all, c, lds[buf], me.wave, me.lane);
    if constexpr (!SUMMARY) {
      if (a.ckpt && me.dok && t < me.te && t % SCAN_CKPT == 0) {
        float* p = a.ckpt + ((long long)me.b * ((a.T + SCAN_CKPT - 1) / SCAN_CKPT) + t / SCAN_CKPT) * a.D + me.d0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) p[v] = c[v];
      }
      const __amdgpu_buffer_rsrc_t out = y.at(tw, me.te, a.D);
#pragma unroll
      for (int l = 0; l < L; ++l) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) c[v] = fmaf(k[l][v], c[v], add[l][v]);
        if (cuts) scan_cut<VEC>(c, cut >> l & 1, add[l]);
        Raw<T, VEC> r;
        r.put(c);
        if (!whole) scan_mask(r, t + l < me.len, 0);
        y.template put<STREAM == 2>(r, out, l, tw, me.te, a.D);
      }
    }
  }
  if (me.chok) {
    if constexpr (SUMMARY) {
      float* p = a.seg + ((long long)me.b * a.nseg + me.seg) * 2 * a.D + me.ch;
      p[0] = all;
      p[a.D] = carry;
    } else if (me.te == a.T) {
      a.h_last[state] = carry;
    }
  }
}

// ----------------------------------------------------------------------------------------------------------- backward
// With C_t = k_t G_t the gradient that leaves step t backwards in time: G_t = dy_t + C_{t+1}, C_t = k_t (dy_t + C_{t+1}),
// C_T = dh_last, dh0 = C_0; dx = G (1 - f), dgate = G (k_t/f_t h_{t-1} - x) f (1 - f).  h is recomputed from the state that
// the forward pass kept at the tile's first step (in 32 bits, where y was rounded), so y is not read.
template <typename T, int VEC, int CG, int L, int THREADS, bool STREAM>
__global__ __launch_bounds__(THREADS) void scan_bwd_kernel(const ScanArgs a) {
  constexpr int TC = THREADS / CG, TILE = TC * L, WAVES = THREADS / 64;
  __shared__ __attribute__((aligned(16))) float lds[2][2][WAVES * 2 * VEC * CG];
  typedef ScanSpot<VEC, CG, L> Spot;
  const Spot me(a);
  typedef ScanRows<T, VEC, L, Spot, true> Rows;
  const Rows gate(me, a.gate, a.gate_bs, a.gate_ts), x(me, a.x, a.x_bs, a.x_ts), dy(me, a.dy, a.dy_bs, a.dy_ts);
  const Rows dgate(me, a.dgate, a.dgate_bs, a.dgate_ts), dx(me, a.dx, a.dx_bs, a.dx_ts);
  const unsigned char* starts = a.starts ? a.starts + me.b * a.starts_bs : nullptr;
  const float* ckpt = a.ckpt + (long long)me.b * ((a.T + SCAN_CKPT - 1) / SCAN_CKPT) * a.D + me.ch;
  const long long state = (long long)me.b * a.D + me.ch;
  const int last = me.tb + (me.te - 1 - me.tb) / TILE * TILE;
  float carry = a.dh_last ? a.dh_last[state] : 0.f, kept = ckpt[(long long)(last / SCAN_CKPT) * a.D], all = 1.f;
  if (a.nseg > 1) carry = scan_join_bwd(a, me.b, me.seg, me.ch, carry);

  Raw<T, VEC> rg[L], rx[L], rd[L];
  int tw = last + me.wave * me.ROWS, buf = 0;
  gate.fetch(rg, tw, me.te, a.D);
  x.fetch(rx, tw, me.te, a.D);
  dy.fetch(rd, tw, me.te, a.D);
  unsigned char rs = scan_start<CG, L>(starts, tw + me.first, me.te, me.lane);
  for (int t0 = last; t0 >= me.tb; t0 -= TILE, tw -= TILE, buf ^= 1) {
    const int t = tw + me.first;
    const bool whole = t0 + TILE <= me.len;
    const unsigned cut = scan_cuts<CG, L>(rs, t, me.len, me.lane);
    const bool cuts = __any(cut != 0);
    float k[L][VEC], rest[L][VEC], w[L][VEC];
    Raw<T, VEC> rc[L];                   // dy as it lies in memory: half the registers
#pragma unroll
    for (int l = 0; l < L; ++l) {        // w: x for now
      if (!whole) {
        scan_mask(rg[l], t + l < me.len, scan_inf<T>());
        scan_mask(rx[l], t + l < me.len, 0);
        scan_mask(rd[l], t + l < me.len, 0);
      }
      float g[VEC];
      rg[l].get(g);
      rx[l].get(w[l]);
      rc[l] = rd[l];
#pragma unroll
      for (int v = 0; v < VEC; ++v) scan_gate(g[v], k[l][v], rest[l][v]);      // k stays f at a start: what it leads to is cut, below
    }
    float h = kept;
    {                                    // the tile before (none: nothing is read)
      const int before = t0 - TILE >= me.tb ? me.te : 0, tp = max(tw - TILE, 0);
      gate.fetch(rg, tp, before, a.D);
      x.fetch(rx, tp, before, a.D);
      dy.fetch(rd, tp, before, a.D);
      rs = scan_start<CG, L>(starts, max(t - TILE, 0), me.te, me.lane);
      kept = ckpt[(long long)(max(t0 - TILE, 0) / SCAN_CKPT) * a.D];
    }
    // the chunk's maps in both directions
    float kk[VEC], k2[VEC], hh[VEC], cc[VEC], hin[VEC], cin[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { kk[v] = k[0][v]; hh[v] = rest[0][v] * w[0][v]; cc[v] = 0.f; }
#pragma unroll
    for (int l = 1; l < L; ++l) {
      float add[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        add[v] = rest[l][v] * w[l][v];
        hh[v] = fmaf(k[l][v], hh[v], add[v]);
        kk[v] *= k[l][v];
      }
      if (cuts) scan_cut<VEC>(hh, cut >> l & 1, add);
    }
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      float d[VEC];
      rc[l].get(d);
#pragma unroll
      for (int v = 0; v < VEC; ++v) cc[v] = k[l][v] * (d[v] + cc[v]);
      if (cuts) scan_cut<VEC>(cc, cut >> l & 1, 0.f);
    }
    scan_floor<VEC>(kk);
    if (cuts) scan_cut<VEC>(kk, cut != 0, 0.f);
#pragma unroll
    for (int v = 0; v < VEC; ++v) k2[v] = kk[v];
    scan_join_tile<VEC, CG, WAVES, false>(kk, hh, h, all, hin, lds[buf][0], me.wave, me.lane);
    scan_join_tile<VEC, CG, WAVES, true>(k2, cc, carry, all, cin, lds[buf][1], me.wave, me.lane);
    // forwards: h_{t-1} of every step, folded at once into w = (h_{t-1} - x) f (1 - f); where an episode starts h_{t-1} is 0
#pragma unroll
    for (int l = 0; l < L; ++l) {
      float add[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float xv = w[l][v];
        add[v] = rest[l][v] * xv;
        w[l][v] = (hin[v] - xv) * (k[l][v] * rest[l][v]);
        hin[v] = fmaf(k[l][v], hin[v], add[v]);
      }
      if (cuts) {
        asm volatile("");
        float old[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) old[v] = -add[v] * k[l][v];
        scan_cut<VEC>(w[l], cut >> l & 1, old);
        scan_cut<VEC>(hin, cut >> l & 1, add);
      }
    }
    // backwards
    const __amdgpu_buffer_rsrc_t og = dgate.at(tw, me.te, a.D), ox = dx.at(tw, me.te, a.D);
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      float d[VEC], g[VEC];
      sq_again(rc[l]);
      rc[l].get(d);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float G = d[v] + cin[v];
        g[v] = G * w[l][v];
        d[v] = G * rest[l][v];
        cin[v] = k[l][v] * G;
      }
      if (cuts) scan_cut<VEC>(cin, cut >> l & 1, 0.f);
      Raw<T, VEC> r1, r2;
      r1.put(g);
      r2.put(d);
      if (!whole) {
        scan_mask(r1, t + l < me.len, 0);
        scan_mask(r2, t + l < me.len, 0);
      }
      dgate.template put<STREAM>(r1, og, l, tw, me.te, a.D);
      dx.template put<STREAM>(r2, ox, l, tw, me.te, a.D);
    }
  }
  if (me.seg == 0 && me.chok) a.dh0[state] = carry;
}

// The map of a piece for the backward direction: C entering from the right -> C leaving to the left (reads gate and dy).
template <typename T, int VEC, int CG, int L, int THREADS>
__global__ __launch_bounds__(THREADS) void scan_bwd_summary_kernel(const ScanArgs a) {
  constexpr int TC = THREADS / CG, TILE = TC * L, WAVES = THREADS / 64;
  __shared__ __attribute__((aligned(16))) float lds[2][WAVES * 2 * VEC * CG];
  typedef ScanSpot<VEC, CG, L> Spot;
  const Spot me(a);
  typedef ScanRows<T, VEC, L, Spot> Rows;
  const Rows gate(me, a.gate, a.gate_bs, a.gate_ts), dy(me, a.dy, a.dy_bs, a.dy_ts);
  const unsigned char* starts = a.starts ? a.starts + me.b * a.starts_bs : nullptr;
  float carry = 0.f, all = 1.f;
  Raw<T, VEC> rg[L], rd[L];
  const int last = me.tb + (me.te - 1 - me.tb) / TILE * TILE;
  int tw = last + me.wave * me.ROWS, buf = 0;
  gate.fetch(rg, tw, me.te, a.D);
  dy.fetch(rd, tw, me.te, a.D);
  unsigned char rs = scan_start<CG, L>(starts, tw + me.first, me.te, me.lane);
  for (int t0 = last; t0 >= me.tb; t0 -= TILE, tw -= TILE, buf ^= 1) {
    const int t = tw + me.first;
    float kk[VEC], cc[VEC], in[VEC];
    const unsigned cut = scan_cuts<CG, L>(rs, t, me.len, me.lane);
    const bool cuts = __any(cut != 0);
#pragma unroll
    for (int v = 0; v < VEC; ++v) { kk[v] = 1.f; cc[v] = 0.f; }
#pragma unroll
    for (int l = L - 1; l >= 0; --l) {
      scan_mask(rg[l], t + l < me.len, scan_inf<T>());
      scan_mask(rd[l], t + l < me.len, 0);
      float g[VEC], d[VEC];
      rg[l].get(g);
      rd[l].get(d);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float f, r;
        scan_gate(g[v], f, r);
        cc[v] = f * (d[v] + cc[v]);
        kk[v] *= f;
      }
      if (cuts) scan_cut<VEC>(cc, cut >> l & 1, 0.f);
    }
    scan_floor<VEC>(kk);
    if (cuts) scan_cut<VEC>(kk, cut != 0, 0.f);
    const int before = t0 - TILE >= me.tb ? me.te : 0;
    gate.fetch(rg, max(tw - TILE, 0), before, a.D);
    dy.fetch(rd, max(tw - TILE, 0), before, a.D);
    rs = scan_start<CG, L>(starts, max(t - TILE, 0), me.te, me.lane);
    scan_join_tile<VEC, CG, WAVES, true>(kk, cc, carry, all, in, lds[buf], me.wave, me.lane);
  }
  if (me.chok) {
    float* p = a.seg + ((long long)me.b * a.nseg + me.seg) * 2 * a.D + me.ch;
    p[0] = all;
    p[a.D] = carry;
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
// wide: 4 elements per access.  The time axis is split (two launches, gate and x read twice) only where sequences and
// channels alone leave half of the CUs idle and there are more than 5 tiles.  bf16 forward: 8 x 4000 x 1024 (128 workgroups) 85 ->
// 68 us; but 12 x 4000 x 1024 (192) 89 -> 132 us, 4 x 512 x 1024 (4 tiles) 11.9 -> 16 us; both ways: 9 x 2000 x 1024 (144) 117 ->
// 128 us, 12 x 777 x 333 fp32 (132) 52 -> 44 us.
// 16-bit rows of up to 32 channels, or 65 to 96, are contiguous enough for groups of 32 channels, with fewer idle lanes: both ways
// 140 x 3000 x 32 bf16 157 -> 88 us, 45 x 14336 x 24 195 -> 123, 140 x 3000 x 80 292 -> 200; with half cache lines of wider rows
// 8 x 4096 x 2048 252 -> 357 us.
// How many pieces: a CU holds two workgroups of the forward kernels, one of the backward, so what counts is the rounds of 512 and
// 256 workgroups, times the tiles of a piece and three quarters of one for its start and end.  Against 512 workgroups or more
// whatever the rounds, both ways bf16: 1 x 24576 x 2424 468 -> 357 us, 6 x 4000 x 1024 179 -> 150, 6 x 10127 x 83 76 -> 61.
// fp32 has workgroups of 256 threads too, but its 128 bytes are 32 channels: counted as two to a CU it gained in one case (5 x 3000 x
// 1024 both ways 177 -> 158 us) and lost in most (8 x 3000 x 1024 186 -> 235, 12 x 700 x 500 49 -> 56, 2 x 4000 x 333 44 -> 55).
static ScanPlan scan_plan(int type, int B, int T, int D, bool wide) {
  ScanPlan p;
  p.vec = wide ? 4 : 1;
  p.cg = !wide ? 64 : type == SERL_F32 || (T > 64 && (D <= 32 || (D > 64 && D <= 96))) ? 8 : 16;
  p.ndb = cdiv(D, p.vec * p.cg);
  p.nseg = 1;
  p.seg_len = T;
  const long long blocks = (long long)B * p.ndb;
  const int fit = wide && type != SERL_F32 && p.cg == 8 ? 2 : 1;      // half the threads and registers: twice as many workgroups on a CU
  if (blocks <= 136 * fit && T > 5 * SCAN_TILE) {
    const int tiles = cdiv(T, SCAN_TILE);
    long long best = 0;
    for (int want = SCAN_MAXSEG; want > 1; --want) {
      const int n = cdiv(tiles, want);      // tiles of a piece
      const long long w = blocks * cdiv(tiles, n), cost = (4ll * n + 3) * (2 * cdivll(w, 512 * fit) + cdivll(w, 256 * fit));
      if (!best || cost <= best) {
        best = cost;
        p.seg_len = n * SCAN_TILE;
      }
    }
    p.nseg = cdiv(T, p.seg_len);
  }
  return p;
}

static long long scan_ws(const ScanPlan& p, int B, int D) { return p.nseg > 1 ? (long long)B * p.nseg * 2 * D * 4 : 0; }

extern "C" long long serl_gated_scan_workspace_bytes(int type, int B, int T, int D) {
  if (type < 0 || type > 2 || B < 0 || T < 0 || T >= SCAN_MAXT || D < 0 || D > SCAN_MAXD) {
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

// A wave addresses its rows of a tile (wide: at most 32, narrow: 8) with 31-bit byte offsets from the first.  Up to SCAN_SHORT steps there
// is no limit: the forward pass runs them in order, the backward pass addresses far rows one by one (ScanRows).
static bool scan_reach(int type, bool wide, int D, long long ts) {
  return ts < (1ll << 40) && ((wide ? 31 : 15) * ts + D) * sq_size(type) < (1ll << 31);
}
// whether every row of (B, T, D) starts at a multiple of `bytes`
static bool scan_rows(int type, int bytes, const void* p, long long bs, long long ts) {
  const int e = sq_size(type);
  return bs * e % bytes == 0 && ts * e % bytes == 0 && sq_aligned(p, bytes);
}
// Accesses of 4 elements: the hardware takes them at any element's address (24 x 3498 x 715 bf16 both ways 461 -> 414 us against single
// elements), so it only takes 4 channels.
static bool scan_wide(int type, int D, long long ts) { return D >= 4 && scan_reach(type, true, D, ts); }

// Tiles of 128 steps, of 16, 32 or 64 where no sequence is longer: 16 (fp32: up to 64 steps 8) elements per thread.  Wide: 128
// bytes of channels and 4 elements per thread and step (64 bytes of channels were 10 % slower, 32 elements per thread 10 to 20 %:
// registers).  Both ways bf16, tile of 64 -> smaller: 256 x 16 x 1024 57 -> 28 us, 181 x 24 x 1536 61 -> 36, 1024 x 10 x 512
// 106 -> 31.  16-bit types with two workgroups per CU to spare stay with 64 steps, half of which wait while the others work: both
// ways 256 x 130 x 1024 229 -> 164 us, 64 x 400 x 1024 124 -> 110; with fewer the larger tile is needed to keep enough loads in
// flight (8 x 4096 x 2048 264 against 344 us), and for many steps where rows start inside cache lines, whose parts are then still in
// the cache when the neighbours come (64 x 3498 x 511 471 against 591 us; 64 x 700 x 511 105 against 97).
#define SCAN_GO(KERNEL, V, C, L, N, ...) hipLaunchKernelGGL((KERNEL<T, V, C, L, N, ##__VA_ARGS__>), grid, dim3(N), 0, st, a)
#define SCAN_LONG(KERNEL, ...)                                                          \
  do {                                                                                  \
    if constexpr (T::code == SERL_F32) SCAN_GO(KERNEL, 4, 8, 4, 256, ##__VA_ARGS__);    \
    else if (p.cg == 8) SCAN_GO(KERNEL, 4, 8, 4, 256, ##__VA_ARGS__);                   \
    else SCAN_GO(KERNEL, 4, 16, 4, 512, ##__VA_ARGS__);                                 \
  } while (0)
#define SCAN_PICK(KERNEL, ...)                                                          \
  do {                                                                                  \
    const bool half = T::code != SERL_F32 && (long long)a.B * a.ndb >= 512 && (!a.share || a.T <= 768); \
    constexpr int C = T::code == SERL_F32 ? 8 : 16, L = T::code == SERL_F32 ? 2 : 4;    \
    if (a.T > 64 && (!half || p.cg == 8)) SCAN_LONG(KERNEL, ##__VA_ARGS__);             \
    else if (a.T > 32) SCAN_GO(KERNEL, 4, C, L, 256, ##__VA_ARGS__);                    \
    else if (a.T > 16) SCAN_GO(KERNEL, 4, C, L, 128, ##__VA_ARGS__);                    \
    else SCAN_GO(KERNEL, 4, C, L, 64, ##__VA_ARGS__);                                   \
  } while (0)
// Streaming where a call moves more than the caches hold and rows are whole cache lines (others lose: 20 x 3000 x 1000 bf16 both ways
// 347 -> 386 us).  Forward alone the inputs: 64 x 1024 x 1024 bf16 90 -> 80 us, 32 x 2048 x 1024 fp32 185 -> 156; where they are read
// again, by the second launch of a split axis or the backward pass, the outputs, and so backward: 4 x 8192 x 2048 forward 152 ->
// 128, both ways 16 x 4096 x 2048 490 -> 470 (with the inputs 501), 64 x 1024 x 1024 254 -> 240.
template <typename T>
static bool scan_stream(const ScanArgs& a, int tensors) {
  return !a.share && (long long)a.B * a.T * a.D * tensors * (long long)sizeof(typename T::bits) > SQ_STREAM;
}
template <typename T>
static void scan_launch_fwd(const ScanArgs& a, const ScanPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)((long long)a.B * a.nseg * a.ndb));
  const bool stream = scan_stream<T>(a, 3);
  if (p.vec == 1) {
    if (a.nseg > 1) SCAN_GO(scan_fwd_kernel, 1, 64, 8, 1024, true, 0);
    SCAN_GO(scan_fwd_kernel, 1, 64, 8, 1024, false, 0);
  } else if (a.nseg > 1) {
    SCAN_LONG(scan_fwd_kernel, true, 0);
    if (stream) SCAN_LONG(scan_fwd_kernel, false, 2);
    else SCAN_LONG(scan_fwd_kernel, false, 0);
  } else if (stream && a.ckpt) {
    SCAN_PICK(scan_fwd_kernel, false, 2);
  } else if (stream) {
    SCAN_PICK(scan_fwd_kernel, false, 1);
  } else {
    SCAN_PICK(scan_fwd_kernel, false, 0);
  }
}
template <typename T>
static void scan_launch_bwd(const ScanArgs& a, const ScanPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)((long long)a.B * a.nseg * a.ndb));
  if (p.vec == 1) {
    if (a.nseg > 1) SCAN_GO(scan_bwd_summary_kernel, 1, 64, 8, 1024);
    SCAN_GO(scan_bwd_kernel, 1, 64, 8, 1024, false);
    return;
  }
  if (a.nseg > 1) SCAN_LONG(scan_bwd_summary_kernel);
  if (scan_stream<T>(a, 5)) SCAN_PICK(scan_bwd_kernel, true);
  else SCAN_PICK(scan_bwd_kernel, false);
}
template <typename T>
static void scan_launch_short(ScanArgs a, bool wide, hipStream_t st) {
  constexpr int W = T::code == SERL_F32 ? 4 : 8;
  a.ndb = wide ? a.D / W : a.D;
  const dim3 grid((unsigned)cdivll((long long)a.B * a.ndb, SCAN_THREADS)), blk(SCAN_THREADS);
  if (wide) hipLaunchKernelGGL((scan_short_kernel<T, W>), grid, blk, 0, st, a);
  else hipLaunchKernelGGL((scan_short_kernel<T, 1>), grid, blk, 0, st, a);
}

// a launch has less than 2^32 threads (SCAN_PICK's workgroups)
static bool scan_fits(const ScanPlan& p, int type, int B, int T) {
  const int threads = p.vec == 1 ? 1024 : T <= 16 ? 64 : T <= 32 ? 128 : T <= 64 || type == SERL_F32 ? 256 : 512;
  return (long long)B * p.nseg * p.ndb < (1ll << 32) / threads;
}

// Rows of D elements of one output that share no memory with each other: sequences of steps, or steps of sequences.
static bool scan_apart(long long B, long long T, long long D, long long bs, long long ts) {
  if (B <= 1 || T <= 1) return (B <= 1 || bs >= D) && (T <= 1 || ts >= D);
  return bs >= D && ts >= D && (bs >= (T - 1) * (__int128)ts + D || ts >= (B - 1) * (__int128)bs + D);
}
// Whether two outputs whose rows lie alike, `delta` elements from each other, share memory: some |delta + b bs + t ts| < D with |b| < B,
// |t| < T.  One of the two strides spans all of the other (scan_apart), so of each the multiples next to what is left come in question.
static bool scan_meet(long long delta, long long B, long long T, long long D, long long bs, long long ts) {
  const __int128 span = (B > 1 ? (B - 1) * (__int128)bs : 0) + (T > 1 ? (T - 1) * (__int128)ts : 0) + D;
  if (delta >= span || -delta >= span) return false;      // two buffers
  const bool time = B <= 1 || (T > 1 && ts > bs);      // the wider stride is that of time
  const __int128 n1 = time ? T : B, n2 = time ? B : T, s1 = time ? ts : bs, s2 = time ? bs : ts;
  for (int i = -1; i <= 1; ++i) {
    const __int128 k1 = n1 > 1 ? -delta / s1 + i : i, left = delta + k1 * s1;
    if (k1 <= -n1 || k1 >= n1) continue;
    for (int j = -1; j <= 1; ++j) {
      const __int128 k2 = n2 > 1 ? -left / s2 + j : j, d = left + k2 * s2;
      if (k2 > -n2 && k2 < n2 && -D < d && d < D) return true;
    }
  }
  return false;
}

#define SCAN_SHORT 8        // up to this many steps one thread runs them in order: a tile would be mostly empty

extern "C" int serl_gated_scan_fwd(int type, int B, int T, int D, const void* gate, long long gate_bs, long long gate_ts,
                                   const void* x, long long x_bs, long long x_ts, const float* h0,
                                   const unsigned char* starts, long long starts_bs, const int* lengths, void* y,
                                   long long y_bs, long long y_ts, float* h_last, float* states, float* workspace,
                                   long long workspace_bytes, void* stream) {
  SERL_CHECK_ARG(type >= 0 && type <= 2, "gated_scan_fwd: type must be 0 (fp32), 1 (bf16) or 2 (fp16)");
  SERL_CHECK_ARG(B >= 0 && T >= 0 && D >= 0, "gated_scan_fwd: negative size");
  SERL_CHECK_ARG(D <= SCAN_MAXD, "gated_scan_fwd: D must be at most %d", SCAN_MAXD);
  if (B == 0 || D == 0) return SERL_OK;
  SERL_CHECK_ARG(h_last && (T == 0 || (gate && x && y)), "gated_scan_fwd: null pointer");
  SERL_CHECK_ARG(gate_bs >= 0 && gate_ts >= 0 && x_bs >= 0 && x_ts >= 0 && (!starts || starts_bs >= 0),
                 "gated_scan_fwd: negative stride");
  SERL_CHECK_ARG((T <= 1 || y_ts >= D) && (T == 0 || B <= 1 || y_bs >= D), "gated_scan_fwd: rows of y overlap");
  SERL_CHECK_ARG(T <= SCAN_SHORT || h_last != h0, "gated_scan_fwd: h_last may be h0 for up to %d steps", SCAN_SHORT);
  SERL_CHECK_ARG(T < SCAN_MAXT, "gated_scan_fwd: T too large");
  const bool few = T <= SCAN_SHORT;
  const bool wide = few ? D * sq_size(type) % 16 == 0 && scan_rows(type, 16, gate, gate_bs, gate_ts) &&
                              scan_rows(type, 16, x, x_bs, x_ts) && scan_rows(type, 16, y, y_bs, y_ts)
                        : scan_wide(type, D, gate_ts) && scan_wide(type, D, x_ts) && scan_wide(type, D, y_ts);
  const ScanPlan p = scan_plan(type, B, T, D, wide);
  SERL_CHECK_ARG(few ? (long long)B * (wide ? D * sq_size(type) / 16 : D) < (1ll << 32) - SCAN_THREADS : scan_fits(p, type, B, T),
                 "gated_scan_fwd: B * D too large");
  SERL_CHECK_ARG(few || (scan_reach(type, false, D, gate_ts) && scan_reach(type, false, D, x_ts) && scan_reach(type, false, D, y_ts)),
                 "gated_scan_fwd: 15 steps of a tensor must span less than 2^31 bytes");
  SERL_CHECK_ARG(T == 0 || scan_apart(B, T, D, y_bs, y_ts), "gated_scan_fwd: rows of y overlap");
  ScanArgs a{};
  a.gate = gate; a.gate_bs = gate_bs; a.gate_ts = gate_ts; a.x = x; a.x_bs = x_bs; a.x_ts = x_ts;
  a.y = y; a.y_bs = y_bs; a.y_ts = y_ts; a.h0 = h0; a.h_last = h_last; a.starts = starts; a.starts_bs = starts_bs;
  a.lengths = lengths; a.ckpt = states; a.B = B; a.T = T; a.D = D;
  a.ndb = p.ndb; a.nseg = p.nseg; a.seg_len = p.seg_len; a.seg = workspace;
  a.share = !(scan_rows(type, 128, gate, gate_bs, gate_ts) && scan_rows(type, 128, x, x_bs, x_ts) && scan_rows(type, 128, y, y_bs, y_ts));
  hipStream_t st = (hipStream_t)stream;
  if (few) {
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
  SERL_CHECK_ARG(D <= SCAN_MAXD, "gated_scan_bwd: D must be at most %d", SCAN_MAXD);
  if (B == 0 || D == 0) return SERL_OK;
  SERL_CHECK_ARG(gate && x && states && dy && dgate && dx && dh0, "gated_scan_bwd: null pointer");
  SERL_CHECK_ARG(gate_bs >= 0 && gate_ts >= 0 && x_bs >= 0 && x_ts >= 0 && dy_bs >= 0 && dy_ts >= 0 &&
                 (!starts || starts_bs >= 0), "gated_scan_bwd: negative stride");
  SERL_CHECK_ARG((T <= 1 || (dgate_ts >= D && dx_ts >= D)) && (B <= 1 || (dgate_bs >= D && dx_bs >= D)),
                 "gated_scan_bwd: rows of dgate or dx overlap");
  SERL_CHECK_ARG(T < SCAN_MAXT, "gated_scan_bwd: T too large");
  if (T == 1) gate_ts = x_ts = dy_ts = dgate_ts = dx_ts = D;      // one step: its strides mean nothing, but rows must not overlap
  const bool wide = scan_wide(type, D, gate_ts) && scan_wide(type, D, x_ts) && scan_wide(type, D, dy_ts) &&
                    scan_wide(type, D, dgate_ts) && scan_wide(type, D, dx_ts);
  const ScanPlan p = scan_plan(type, B, T, D, wide);
  SERL_CHECK_ARG(scan_fits(p, type, B, T), "gated_scan_bwd: B * D too large");
  SERL_CHECK_ARG(T <= SCAN_SHORT || (scan_reach(type, false, D, gate_ts) && scan_reach(type, false, D, x_ts) && scan_reach(type, false, D, dy_ts) &&
                                     scan_reach(type, false, D, dgate_ts) && scan_reach(type, false, D, dx_ts)),
                 "gated_scan_bwd: 15 steps of a tensor must span less than 2^31 bytes");
  SERL_CHECK_ARG(scan_apart(B, T, D, dgate_bs, dgate_ts) && scan_apart(B, T, D, dx_bs, dx_ts) && dgate != dx &&
                     ((B > 1 && dgate_bs != dx_bs) || (T > 1 && dgate_ts != dx_ts) ||
                      !scan_meet(((const char*)dx - (const char*)dgate) / sq_size(type), B, T, D, dgate_bs, dgate_ts)),
                 "gated_scan_bwd: rows of dgate or dx overlap");
  const long long need = scan_ws(p, B, D);
  SERL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                 "gated_scan_bwd: workspace of %lld bytes needed, %lld available", need, workspace ? workspace_bytes : 0);
  ScanArgs a{};
  a.gate = gate; a.gate_bs = gate_bs; a.gate_ts = gate_ts; a.x = x; a.x_bs = x_bs; a.x_ts = x_ts;
  a.dy = dy; a.dy_bs = dy_bs; a.dy_ts = dy_ts; a.dh_last = dh_last; a.starts = starts; a.starts_bs = starts_bs;
  a.lengths = lengths; a.ckpt = const_cast<float*>(states); a.dgate = dgate; a.dgate_bs = dgate_bs; a.dgate_ts = dgate_ts;
  a.dx = dx; a.dx_bs = dx_bs; a.dx_ts = dx_ts; a.dh0 = dh0; a.B = B; a.T = T; a.D = D;
  a.ndb = p.ndb; a.nseg = p.nseg; a.seg_len = p.seg_len; a.seg = workspace;
  a.share = !(scan_rows(type, 128, gate, gate_bs, gate_ts) && scan_rows(type, 128, x, x_bs, x_ts) &&
              scan_rows(type, 128, dy, dy_bs, dy_ts) && scan_rows(type, 128, dgate, dgate_bs, dgate_ts) &&
              scan_rows(type, 128, dx, dx_bs, dx_ts));
  hipStream_t st = (hipStream_t)stream;
  if (type == SERL_F32) scan_launch_bwd<F32>(a, p, st);
  else if (type == SERL_BF16) scan_launch_bwd<BF16>(a, p, st);
  else scan_launch_bwd<F16>(a, p, st);
  SERL_CHECK_LAUNCH("gated_scan_bwd");
  return SERL_OK;
}
