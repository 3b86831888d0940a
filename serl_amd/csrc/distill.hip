// Distillation from a teacher's top logits: with q = softmax(teacher / tau) over a row's K slots and
// p = softmax(logits / tau) over all V columns,
//   loss_r = c_r tau^2 sum_k q_k (log q_k - log p[i_k]),   dlogits = c_r tau (p - sum_k q_k [column = i_k])
// value and gradient in one pass, like the other losses (rowops.hip).  No counterpart in the reference (its only discrete
// head has two outcomes).
//
// Bound by memory: one read and one write of (R, V).  A row stays in the registers of one workgroup between the softmax's
// statistics and the gradient (up to 1024 threads x 20 pieces of 16 bytes: 160 Ki 16-bit columns); the workgroup walks
// through rows, and each piece's registers are refilled with the next row's as soon as its gradient is stored, so loads and
// stores overlap.  Few long rows, and rows too long for registers, are cut into pieces of their own workgroups: one launch
// for the statistics, one that joins them and writes the gradient (it reads the row again, from the caches where they hold it).
//
// 2048 x 131072 bf16, 128 slots: 217 us (5.0 TB/s where a large copy reaches 5.2; the first load and the last store of a
// workgroup's eight rows overlap nothing, and the vector ALU is half busy with two exponentials per column); the value alone 108 us,
// 2048 x 65536 fp32 226.
//
// Rows start at any alignment: the columns before the first 16-byte boundary and behind the last whole piece are taken by
// single threads (`head` and `tail`); the gradient is stored in the logits' pieces, which may lie at any element of its rows
// (against single elements where the two differ, 1500 x 50021 165 -> 75 us).  The teacher's columns are
// stored a second time, behind a barrier that all dense stores of the row have passed.
#include "seqtypes.h"

#define DIST_MAXK 512
#define DIST_MAXR 0x7fff0000  // a row number and the step to the next one fit 31 bits
#define DIST_LOG2E 1.44269504088896340736f
#define DIST_LN2 0.69314718055994530942f

struct DistArgs {
  const void *logits, *teacher, *index;
  void* dlogits;
  long long ldl, ldt, ldi, ldd;
  const float* coef;
  float *loss, *part, *taken;         // part: (R, pieces, 2) m and s; taken: (R, K) the student's logits at the slots
  int R, V, K, teacher_f32, index64, pieces, piece_vecs;
  float tau;
};

// all V columns of a row: [0, nh) head, nvec whole pieces of VEC, then the tail
struct DistRow { int nh, nvec, nt; };
template <typename T, int VEC>
__device__ __forceinline__ DistRow dist_row(const void* p, int V) {
  DistRow r;
  const int mis = (int)(((uintptr_t)p / sizeof(typename T::bits)) % VEC);
  r.nh = mis ? VEC - mis : 0;
  r.nvec = (V - r.nh) / VEC;
  r.nt = V - r.nh - r.nvec * VEC;
  return r;
}
// the single column that thread t takes besides its pieces, or -1: threads [0, nh) the head, [VEC, VEC + nt) the tail
template <int VEC>
__device__ __forceinline__ int dist_extra(const DistRow& r, int t) {
  if (VEC == 1) return -1;
  if (t < r.nh) return t;
  return t >= VEC && t < VEC + r.nt ? r.nh + r.nvec * VEC + t - VEC : -1;
}

// larger of three, without the canonicalising moves that fmaxf takes for values that come from memory; a NaN may or may not be
// passed over (it is in the sum then)
__device__ __forceinline__ float dist_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <int VEC> __device__ __forceinline__ float dist_max(float m, const float (&x)[VEC]) {
  if constexpr (VEC == 1) return dist_max3(m, x[0], x[0]);
#pragma unroll
  for (int v = 0; v + 1 < VEC; v += 2) m = dist_max3(m, x[v], x[v + 1]);
  return m;
}

// piece j of a row's whole pieces (`base`: the first one): a uniform address and a 32-bit offset per thread
template <bool STREAM = false, typename T, int VEC>
__device__ __forceinline__ void dist_load(Raw<T, VEC>& r, const typename T::bits* base, int j) {
  r.template load<false, STREAM>((const typename T::bits*)((const char*)base + (uint32_t)j * (uint32_t)(VEC * sizeof(typename T::bits))));
}
// (the gradient's rows may lie otherwise than the logits': at any element)
template <bool STREAM = false, typename T, int VEC>
__device__ __forceinline__ void dist_store(const Raw<T, VEC>& r, typename T::bits* base, int j) {
  r.template store<!STREAM, STREAM>((typename T::bits*)((char*)base + (uint32_t)j * (uint32_t)(VEC * sizeof(typename T::bits))));
}

template <typename T> __device__ __forceinline__ uint32_t dist_minus_inf() {
  return T::code == SERL_F32 ? 0xff800000u : T::code == SERL_BF16 ? 0xff80ff80u : 0xfc00fc00u;
}
template <typename T, int VEC> __device__ __forceinline__ void dist_mask(Raw<T, VEC>& r, bool keep) {
  if constexpr (VEC == 1) {
    r.w = keep ? r.w : (typename T::bits)dist_minus_inf<T>();
  } else {
#pragma unroll
    for (int i = 0; i < Raw<T, VEC>::W; ++i) r.w[i] = keep ? r.w[i] : dist_minus_inf<T>();
  }
}

// A partial softmax sum is kept as (m, s): m the part's largest x as it is, s = sum of 2^((x - m) k2), k2 = log2(e) / tau.
// Differences are taken before the scaling, so columns masked with the type's lowest value count as such (a row of nothing
// else is uniform).  An empty or all -inf part is (-inf, 0); NaN live in s alone.
__device__ __forceinline__ float dist_ref(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ float dist_exp(float x, float ref, float k2) { return __builtin_amdgcn_exp2f((x - ref) * k2); }
__device__ __forceinline__ void dist_join(float& m, float& s, float m2, float s2, float k2) {
  const float n = fmaxf(m, m2), ref = dist_ref(n);
  s = s * dist_exp(m, ref, k2) + s2 * dist_exp(m2, ref, k2);
  m = n;
}

__device__ __forceinline__ float dist_uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// a row's teacher in LDS: slot columns (-1: absent), weights q and the student's logits there
struct DistTeacher { int* idx; float *q, *lg; };
__device__ __forceinline__ DistTeacher dist_tables(float* lds, int K, int buf) {
  DistTeacher d;
  d.idx = (int*)lds + (buf * 3) * K;
  d.q = lds + (buf * 3 + 1) * K;
  d.lg = lds + (buf * 3 + 2) * K;
  return d;
}
__device__ __forceinline__ long long dist_column(const DistArgs& a, int row, int k) {
  return a.index64 ? ((const long long*)a.index)[row * a.ldi + k] : (long long)((const int*)a.index)[row * a.ldi + k];
}
// By one wave.  A slot is absent if its column is outside [0, V) or its logit is -inf; NaN and +inf are carried on.  As with the
// student, differences are taken before the temperature: slots that all hold the type's lowest value weigh the same.
// TAKEN: the student's logits are those that dist_stats_kernel took (the row may be half overwritten by now).
// Returns whether any slot is there.
template <typename T, bool TAKEN>
__device__ __forceinline__ bool dist_stage(const DistArgs& a, int row, const DistTeacher& d, int lane) {
  const typename T::bits* logits = (const typename T::bits*)a.logits + row * a.ldl;
  const float inv = 1.f / a.tau;
  float top = -INFINITY;
  bool any = false;
#pragma unroll TAKEN ? 4 : 1       // the kernel that holds rows has no registers to spare
  for (int k = lane; k < a.K; k += 64) {
    const long long id = dist_column(a, row, k);
    const float tv = a.teacher_f32 ? ((const float*)a.teacher)[row * a.ldt + k]
                                   : sq_val(T(), ((const typename T::bits*)a.teacher)[row * a.ldt + k]);
    const bool ok = id >= 0 && id < a.V && !(tv == -INFINITY);
    const float lg = TAKEN ? a.taken[(long long)row * a.K + k] : sq_val(T(), logits[ok ? id : 0]);
    d.idx[k] = ok ? (int)id : -1;
    d.q[k] = tv;
    d.lg[k] = lg;
    top = ok ? fmaxf(top, tv) : top;
    any |= ok;
  }
  top = sq_wave_max(top);
  float sum = 0.f;
#pragma unroll 1
  for (int k = lane; k < a.K; k += 64) {
    const float e = d.idx[k] >= 0 ? expf((d.q[k] - top) * inv) : 0.f;
    d.q[k] = e;
    sum += e;
  }
  sum = sq_wave_sum(sum);
  const float r = 1.f / sum;
  for (int k = lane; k < a.K; k += 64) d.q[k] = d.idx[k] >= 0 ? d.q[k] * r : 0.f;
  return __any(any);
}
// The same in two steps for one slot per lane (K <= 64), so that neither the slots nor the logits they name are waited for: the
// registers hold them as they lie in memory until dist_finish, a row later.  Same bits as dist_stage.
struct DistSlot { uint32_t lo, hi, tv; };
__device__ __forceinline__ long long dist_id(const DistArgs& a, const DistSlot& c) {
  return a.index64 ? (long long)((unsigned long long)c.hi << 32 | c.lo) : (long long)(int)c.lo;
}
template <typename T> __device__ __forceinline__ void dist_fetch(const DistArgs& a, int row, int lane, DistSlot& c) {
  const int k = lane < a.K ? lane : 0;
  if (a.index64) {
    const uint32_t* p = (const uint32_t*)((const long long*)a.index + row * a.ldi + k);
    c.lo = p[0]; c.hi = p[1];
  } else {
    c.lo = ((const uint32_t*)a.index)[row * a.ldi + k]; c.hi = 0;
  }
  c.tv = a.teacher_f32 ? ((const uint32_t*)a.teacher)[row * a.ldt + k] : (uint32_t)((const typename T::bits*)a.teacher)[row * a.ldt + k];
}
template <typename T> __device__ __forceinline__ bool dist_there(const DistArgs& a, const DistSlot& c, int lane, float& tv) {
  const long long id = dist_id(a, c);
  tv = a.teacher_f32 ? __uint_as_float(c.tv) : sq_val(T(), (typename T::bits)c.tv);
  return lane < a.K && id >= 0 && id < a.V && !(tv == -INFINITY);
}
template <typename T> __device__ __forceinline__ typename T::bits dist_gather(const DistArgs& a, int row, const DistSlot& c, int lane) {
  float tv;
  const bool ok = dist_there<T>(a, c, lane, tv);
  return ((const typename T::bits*)a.logits + row * a.ldl)[ok ? dist_id(a, c) : 0];
}
template <typename T>
__device__ __forceinline__ bool dist_finish(const DistArgs& a, const DistSlot& c, typename T::bits lg, const DistTeacher& d, int lane) {
  float tv;
  const bool ok = dist_there<T>(a, c, lane, tv);
  float top = ok ? fmaxf(-INFINITY, tv) : -INFINITY;
  top = sq_wave_max(top);
  const float e = ok ? expf((tv - top) * (1.f / a.tau)) : 0.f, sum = sq_wave_sum(e);
  if (lane < a.K) {
    d.idx[lane] = ok ? (int)dist_id(a, c) : -1;
    d.q[lane] = ok ? e * (1.f / sum) : 0.f;
    d.lg[lane] = sq_val(T(), lg);
  }
  return __any(ok);
}
// The loss over c tau, by the wave that staged the teacher: sum of q (tau (log q + log sum) - (logit - m)).  A column's logit is not scaled
// by 1 / tau and log2(e) on the way, which the type's lowest value (a masked column) would not bear.
__device__ __forceinline__ float dist_loss(const DistArgs& a, const DistTeacher& d, float m, float sum, int lane) {
  const float lsum = log2f(sum) * DIST_LN2;
  float s = 0.f;
#pragma unroll 1
  for (int k = lane; k < a.K; k += 64) {
    const float q = d.q[k];
    s += q == 0.f ? 0.f : q * (a.tau * (logf(q) + lsum) - (d.lg[k] - m));
  }
  return sq_wave_sum(s);
}
// All the wave's stores have been taken: behind the barrier that follows, another wave's store to the same place comes later.
__device__ __forceinline__ void dist_drain() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// the teacher's columns [lo, hi): scale (p - q summed over the slots of the column), slots in order
template <typename T>
__device__ __forceinline__ void dist_fix(const DistArgs& a, int row, const DistTeacher& d, float m, float inv_sum, float scale,
                                         int lo, int hi, int t, int threads) {
  typename T::bits* out = (typename T::bits*)a.dlogits + row * a.ldd;
  const float k2 = DIST_LOG2E / a.tau;
#pragma unroll 1
  for (int k = t; k < a.K; k += threads) {
    const int id = d.idx[k];
    if (id < lo || id >= hi) continue;
    float q = 0.f;
    int j = 0;
    for (; j + 8 <= a.K; j += 8) {       // both read whatever they are: the reads of eight slots are under way together
      int ij[8];
      float qj[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { ij[i] = d.idx[j + i]; qj[i] = d.q[j + i]; }
#pragma unroll
      for (int i = 0; i < 8; ++i) q += ij[i] == id ? qj[i] : 0.f;
    }
    for (; j < a.K; ++j) q += d.idx[j] == id ? d.q[j] : 0.f;
    out[id] = sq_bits(T(), scale * (dist_exp(d.lg[k], m, k2) * inv_sum - q));
  }
}

// -------------------------------------------------------------------------------------------- rows held in registers
// EARLY (one wave, K <= 64): the teacher's slots are fetched two rows ahead, the logits they name one row: 65536 x 1000 bf16 with 32
// slots 107 -> 79 us, 100000 x 256 123 -> 104 (with reductions of the vector ALU 84).
template <typename T, int VEC, int THREADS, int NV, bool STREAM, bool EARLY>
__global__ __launch_bounds__(THREADS) void dist_row_kernel(const DistArgs a) {
  constexpr int WAVES = THREADS / 64;
  static_assert(!EARLY || WAVES == 1, "one wave");
  extern __shared__ float tables[];           // 3 x K x {column, q, logit}: of the last, this and the next row
  __shared__ float red[2][WAVES][2];
  __shared__ int alive[3];
  typedef typename T::bits bits;
  const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
  const float k2 = DIST_LOG2E / a.tau;
  Raw<T, VEC> raw[NV];
  Raw<T, 1> extra;
  int row = blockIdx.x;
  const bits* p = (const bits*)a.logits + row * a.ldl;
  DistRow w = dist_row<T, VEC>(p, a.V);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = i * THREADS + t;
    dist_load<STREAM>(raw[i], p + w.nh, j < w.nvec ? j : 0);
  }
  extra.load(p + max(0, dist_extra<VEC>(w, t)));
  DistSlot slot, ahead;
  bits named = 0;
  if constexpr (EARLY) {
    dist_fetch<T>(a, row, lane, slot);
    dist_fetch<T>(a, min(row + (int)gridDim.x, a.R - 1), lane, ahead);
    named = dist_gather<T>(a, row, slot, lane);
  } else if (wave == 0) {
    const bool any = dist_stage<T, false>(a, row, dist_tables(tables, a.K, 0), lane);
    if (lane == 0) alive[0] = any;
  }
  int buf = 0, tab = 0, last = -1;
  float last_m = 0.f, last_inv = 0.f, last_scale = 0.f;
  for (; row < a.R; row += gridDim.x, buf ^= 1) {
    const int ex = dist_extra<VEC>(w, t);
    float m = -INFINITY, s = 0.f;
    int tm = t;          // the pieces' numbers are computed where they are used, not kept over the loop in registers
    asm volatile("" : "+v"(tm));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      dist_mask<T, VEC>(raw[i], i * THREADS + tm < w.nvec);
      float x[VEC];
      raw[i].get(x);
      m = dist_max<VEC>(m, x);
    }
    dist_mask<T, 1>(extra, ex >= 0);
    float xe[1];
    extra.get(xe);
    m = fmaxf(m, xe[0]);
    m = sq_wave_max(m);
    const float wref = dist_ref(m);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[VEC];
      sq_again(raw[i]);
      raw[i].get(x);
#pragma unroll
      for (int v = 0; v < VEC; ++v) s += dist_exp(x[v], wref, k2);
    }
    s += dist_exp(xe[0], wref, k2);
    s = sq_wave_sum(s);
    if (lane == 0) { red[buf][wave][0] = m; red[buf][wave][1] = s; }
    dist_drain();          // the last row's gradient; its loads are behind those of this row, which have arrived
    __syncthreads();
    if (last >= 0) dist_fix<T>(a, last, dist_tables(tables, a.K, tab == 0 ? 2 : tab - 1), last_m, last_inv, last_scale, 0, a.V, t, THREADS);
    if constexpr (WAVES > 1) {              // lane 0's join for everybody: the order of the parts, and so the bits, are its own
      m = red[buf][lane & (WAVES - 1)][0]; s = red[buf][lane & (WAVES - 1)][1];
#pragma unroll
      for (int o = 1; o < WAVES; o <<= 1) {
        const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
        dist_join(m, s, m2, s2, k2);
      }
    }
    m = dist_uniform(m);
    s = dist_uniform(s);
    bool any_slot;
    if constexpr (EARLY) {
      any_slot = dist_finish<T>(a, slot, named, dist_tables(tables, a.K, tab), lane);
      slot = ahead;
      named = dist_gather<T>(a, min(row + (int)gridDim.x, a.R - 1), slot, lane);
      dist_fetch<T>(a, min(row + 2 * (int)gridDim.x, a.R - 1), lane, ahead);
    } else {
      any_slot = alive[tab];
    }
    const float c = a.coef ? a.coef[row] : 1.f;
    const bool dead = !any_slot || c == 0.f;
    if (wave == 0) {
      const float l = dist_loss(a, dist_tables(tables, a.K, tab), m, s, lane);
      if (lane == 0) a.loss[row] = dead ? 0.f : c * a.tau * l;
    }
    const int next = row + (int)gridDim.x;
    const bool more = next < a.R;
    const bits* pn = (const bits*)a.logits + (more ? next : row) * a.ldl;
    const DistRow wn = dist_row<T, VEC>(pn, a.V);
    const int nn = more ? wn.nvec : 0;
    const float inv = 1.f / s, scale = c * a.tau, mul = scale * inv;
    bits* out = a.dlogits ? (bits*)a.dlogits + row * a.ldd : nullptr;
    asm volatile("" : "+v"(tm));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * THREADS + tm;
      if (out) {
        float x[VEC];
        sq_again(raw[i]);
        raw[i].get(x);
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[v] = dead ? 0.f : dist_exp(x[v], m, k2) * mul;
        Raw<T, VEC> g;
        g.put(x);
        if (j < w.nvec) dist_store<STREAM>(g, out + w.nh, j);
      }
      dist_load<STREAM>(raw[i], pn + wn.nh, j < nn ? j : 0);      // no next row (nn = 0): one cached line
    }
    if (out && ex >= 0) {
      Raw<T, 1> g;
      xe[0] = dead ? 0.f : dist_exp(xe[0], m, k2) * mul;
      g.put(xe);
      g.store(out + ex);
    }
    extra.load(pn + (more ? max(0, dist_extra<VEC>(wn, t)) : 0));
    last = out && !dead ? row : -1;
    last_m = m; last_inv = inv; last_scale = scale;
    tab = tab == 2 ? 0 : tab + 1;
    if (!EARLY && wave == 0 && more) {
      const bool any = dist_stage<T, false>(a, next, dist_tables(tables, a.K, tab), lane);
      if (lane == 0) alive[tab] = any;
    }
    w = wn;
  }
  dist_drain();
  __syncthreads();
  if (last >= 0) dist_fix<T>(a, last, dist_tables(tables, a.K, tab == 0 ? 2 : tab - 1), last_m, last_inv, last_scale, 0, a.V, t, THREADS);
}

// ------------------------------------------------------------------------------------------------- rows cut in pieces
#define DIST_CUT 256
template <typename T, int VEC>
__global__ __launch_bounds__(DIST_CUT) void dist_stats_kernel(const DistArgs a) {
  __shared__ float red[4][2];
  typedef typename T::bits bits;
  const int t = threadIdx.x, row = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  const bits* p = (const bits*)a.logits + row * a.ldl;
  const DistRow w = dist_row<T, VEC>(p, a.V);
  const int j0 = piece * a.piece_vecs, j1 = min(w.nvec, j0 + a.piece_vecs);
  const float k2 = DIST_LOG2E / a.tau;
  const int ex = piece == 0 ? dist_extra<VEC>(w, t) : -1;
  Raw<T, 1> extra;
  extra.load(p + max(0, ex));
  dist_mask<T, 1>(extra, ex >= 0);
  float xe[1];
  extra.get(xe);
  float m = fmaxf(xe[0], -INFINITY), s = dist_exp(xe[0], dist_ref(m), k2);
  constexpr int U = 4;
  for (int jb = j0; jb < j1; jb += DIST_CUT * U) {
    Raw<T, VEC> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = jb + u * DIST_CUT + t;
      dist_load(raw[u], p + w.nh, j < j1 ? j : j1 - 1);
    }
    float x[U][VEC], n = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      dist_mask<T, VEC>(raw[u], jb + u * DIST_CUT + t < j1);
      raw[u].get(x[u]);
      n = dist_max<VEC>(n, x[u]);
    }
    n = fmaxf(m, n);
    const float ref = dist_ref(n);
    s *= dist_exp(m, ref, k2);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < VEC; ++v) s += dist_exp(x[u][v], ref, k2);
    m = n;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
    dist_join(m, s, m2, s2, k2);
  }
  if ((t & 63) == 0) { red[t >> 6][0] = m; red[t >> 6][1] = s; }
  __syncthreads();
  if (t == 0) {
    for (int q = 1; q < 4; ++q) dist_join(m, s, red[q][0], red[q][1], k2);
    float* o = a.part + ((long long)row * a.pieces + piece) * 2;
    o[0] = m; o[1] = s;
  }
  if (piece == 0) {         // before any workgroup of the next launch overwrites the row, if it is in place
    for (int k = t; k < a.K; k += DIST_CUT) {
      const long long id = dist_column(a, row, k);
      a.taken[(long long)row * a.K + k] = sq_val(T(), p[id >= 0 && id < a.V ? id : 0]);
    }
  }
}

// Four waves write the gradient of a piece, a fifth takes the teacher meanwhile; only then the teacher's columns are put right.
template <typename T, int VEC>
__global__ __launch_bounds__(DIST_CUT + 64) void dist_grad_kernel(const DistArgs a) {
  extern __shared__ float tables[];
  __shared__ int alive;
  typedef typename T::bits bits;
  const int t = threadIdx.x, lane = t & 63, row = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  const bits* p = (const bits*)a.logits + row * a.ldl;
  const DistRow w = dist_row<T, VEC>(p, a.V);
  const int j0 = piece * a.piece_vecs, j1 = min(w.nvec, j0 + a.piece_vecs);
  const float k2 = DIST_LOG2E / a.tau;
  const DistTeacher d = dist_tables(tables, a.K, 0);
  const bool dense = t < DIST_CUT;
  constexpr int U = 4;
  Raw<T, VEC> raw[U];
  const auto fetch = [&](int jb) {
    if (jb < j1) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * DIST_CUT + t;
        dist_load(raw[u], p + w.nh, j < j1 ? j : j1 - 1);
      }
    }
  };
  if (dense && a.dlogits) fetch(j0);    // under way while the statistics are read
  bool any = false;
  if (!dense) any = dist_stage<T, true>(a, row, d, lane);
  float m = -INFINITY, s = 0.f;         // every wave joins the row's statistics
  for (int q = lane; q < a.pieces; q += 64) {
    const float* o = a.part + ((long long)row * a.pieces + q) * 2;
    dist_join(m, s, o[0], o[1], k2);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
    dist_join(m, s, m2, s2, k2);
  }
  m = dist_uniform(m);
  s = dist_uniform(s);
  const float c = a.coef ? a.coef[row] : 1.f;
  const float inv = 1.f / s, scale = c * a.tau, mul = scale * inv;
  bits* out = (bits*)a.dlogits + row * a.ldd;
  const int ex = piece == 0 && dense ? dist_extra<VEC>(w, t) : -1;
  if (!dense) {
    if (lane == 0) alive = any;
    if (piece == 0) {
      const float l = dist_loss(a, d, m, s, lane);
      if (lane == 0) a.loss[row] = any && c != 0.f ? c * a.tau * l : 0.f;
    }
  } else if (a.dlogits && c != 0.f) {
    for (int jb = j0; jb < j1; jb += DIST_CUT * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = jb + u * DIST_CUT + t;
        float x[VEC];
        raw[u].get(x);
#pragma unroll
        for (int v = 0; v < VEC; ++v) x[v] = dist_exp(x[v], m, k2) * mul;
        raw[u].put(x);
        if (j < j1) dist_store(raw[u], out + w.nh, j);
      }
      fetch(jb + DIST_CUT * U);
    }
    if (ex >= 0) {
      Raw<T, 1> e;
      e.load(p + ex);
      float x[1];
      e.get(x);
      x[0] = dist_exp(x[0], m, k2) * mul;
      e.put(x);
      e.store(out + ex);
    }
  }
  if (!a.dlogits) return;
  dist_drain();
  __syncthreads();
  if (alive && c != 0.f) {
    dist_fix<T>(a, row, d, m, inv, scale, w.nh + j0 * VEC, w.nh + j1 * VEC, t, DIST_CUT + 64);
    if (piece == 0) {
      dist_fix<T>(a, row, d, m, inv, scale, 0, w.nh, t, DIST_CUT + 64);
      dist_fix<T>(a, row, d, m, inv, scale, w.nh + w.nvec * VEC, a.V, t, DIST_CUT + 64);
    }
  } else if (dense) {                   // a row that is left out: zeros, whatever was written above
    Raw<T, VEC> zero;
    float x[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) x[v] = 0.f;
    zero.put(x);
    for (int j = j0 + t; j < j1; j += DIST_CUT) dist_store(zero, out + w.nh, j);
    if (ex >= 0) out[ex] = 0;
  }
}

// ---------------------------------------------------------------------------------------------------------- host side
// Pieces a row is cut into (1: a workgroup holds whole rows in registers).  Cutting costs a second launch and pays where few
// workgroups would hold very long rows: 64 x 131072 bf16 21.7 -> 16.0 us, but 64 x 65536 13.9 -> 16.8 us.
struct DistPlan { int pieces, piece_vecs; };
static int dist_vec(int type) { return type == SERL_F32 ? 4 : 8; }
static DistPlan dist_plan(int type, int R, int V) {
  const int n = cdiv(V, dist_vec(type));
  const int most = 1024 * 20;                                      // vectors of a row that fit the registers
  DistPlan p{1, n};
  int want = 1;
  if (n > most) want = cdiv(n, 4096);
  if (R < 128 && n > 8192) {                                       // few rows: share each among enough workgroups
    const int share = cdiv(512, R < 1 ? 1 : R), fit = cdiv(n, 1024);
    const int q = share < fit ? share : fit;
    want = want > q ? want : q;
  }
  if (want > 1) {
    p.piece_vecs = cdiv(n, want);
    p.pieces = cdiv(n, p.piece_vecs);
  }
  return p;
}

template <typename T, int VEC, int THREADS, int NV, bool STREAM, bool EARLY = false>
static void dist_go(const DistArgs& a, hipStream_t st) {
  // persistent: as many workgroups as 256 CUs hold at once (asked for once; 128 slots' tables in LDS); of one-wave workgroups 28 per CU
  // instead of 32: 65536 x 1000 bf16 87 -> 79 us, 200000 x 512 187 -> 166
  static const int fit = [] {
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, dist_row_kernel<T, VEC, THREADS, NV, STREAM, EARLY>, THREADS,
                                                     3 * 3 * 128 * sizeof(float)) != hipSuccess || n < 1) {
      (void)hipGetLastError();
      n = 1;
    }
    return 256 * (n > 28 ? 28 : n);
  }();
  hipLaunchKernelGGL((dist_row_kernel<T, VEC, THREADS, NV, STREAM, EARLY>), dim3(a.R < fit ? a.R : fit), dim3(THREADS),
                     3 * 3 * a.K * sizeof(float), st, a);
}
// Threads and vectors per thread.  Half the vectors for rows of 65 to 128 halve the exponentials: 20000 x 1000 bf16 30 -> 28 us; fp32
// has fewer per vector and lost by it (50000 x 512 61 -> 71 us).
template <typename T, int VEC, bool EARLY>
static void dist_wave(const DistArgs& a, int n, hipStream_t st) {
  if (n <= 64) return dist_go<T, VEC, 64, 1, false, EARLY>(a, st);
  if constexpr (VEC == 8) {
    if (n <= 128) return dist_go<T, VEC, 64, 2, false, EARLY>(a, st);
  }
  if (n <= 256) return dist_go<T, VEC, 64, 4, false, EARLY>(a, st);
  dist_go<T, VEC, 64, 8, false, EARLY>(a, st);
}
template <typename T, int VEC, bool STREAM>
static void dist_shape(const DistArgs& a, hipStream_t st) {
  const int n = cdiv(a.V, VEC);
  if constexpr (!STREAM) {
    if (n <= 512) return a.K <= 64 ? dist_wave<T, VEC, true>(a, n, st) : dist_wave<T, VEC, false>(a, n, st);
  }
  if (n <= 1024) dist_go<T, VEC, 128, 8, STREAM>(a, st);
  else if (n <= 2048) dist_go<T, VEC, 256, 8, STREAM>(a, st);
  else if (n <= 4096) dist_go<T, VEC, 512, 8, STREAM>(a, st);
  else if (n <= 8192) dist_go<T, VEC, 1024, 8, STREAM>(a, st);
  else if (n <= 16384) dist_go<T, VEC, 1024, 16, STREAM>(a, st);
  else dist_go<T, VEC, 1024, 20, STREAM>(a, st);
}
// Logits and gradient are streamed past the caches where a call moves more than they hold and rows are whole cache lines, more than
// 512 vectors: 2048 x 131072 bf16 242 -> 225 us, 16384 x 8192 124 -> 111; below that size 8192 x 8000 53 -> 57, of a wave's rows
// 65536 x 1024 107 -> 121.
static bool dist_stream(const DistArgs& a, int type) {
  const int e = sq_size(type);
  return a.V > 512 * 16 / e && a.V * (long long)e % 128 == 0 && a.ldl * e % 128 == 0 && a.ldd * e % 128 == 0 && sq_aligned(a.logits, 128) &&
         sq_aligned(a.dlogits, 128) && (long long)a.R * a.V * e * (a.dlogits ? 2 : 1) > SQ_STREAM;
}

template <typename T, int VEC>
static void dist_launch(const DistArgs& a, hipStream_t st) {
  if constexpr (VEC == 1) {
    if (a.K <= 64) dist_go<T, 1, 64, 1, false, true>(a, st);      // less than two vectors
    else dist_go<T, 1, 64, 1, false>(a, st);
  } else if (a.pieces > 1) {
    const dim3 grid((unsigned)(a.R * a.pieces));
    hipLaunchKernelGGL((dist_stats_kernel<T, VEC>), grid, dim3(DIST_CUT), 0, st, a);
    hipLaunchKernelGGL((dist_grad_kernel<T, VEC>), grid, dim3(DIST_CUT + 64), 3 * a.K * sizeof(float), st, a);
  } else if (dist_stream(a, T::code)) {
    dist_shape<T, VEC, true>(a, st);
  } else {
    dist_shape<T, VEC, false>(a, st);
  }
}

static long long dist_ws(const DistPlan& p, int R, int K) {
  return p.pieces > 1 ? (long long)R * p.pieces * 8 + (long long)R * K * 4 : 0;
}

extern "C" long long serl_topk_distill_workspace_bytes(int type, int R, int V, int K) {
  if (type < 0 || type > 2 || R < 0 || R > DIST_MAXR || V < 1 || K < 1 || K > DIST_MAXK) {
    serl_set_error("topk_distill: bad type or sizes");
    return -1;
  }
  return dist_ws(dist_plan(type, R, V), R, K);
}

extern "C" int serl_topk_distill(int type, int teacher_type, int index64, int R, int V, int K, const void* logits,
                                 long long ldl, const void* teacher, long long ldt, const void* index, long long ldi,
                                 float temperature, const float* coef, float* loss, void* dlogits, long long ldd,
                                 float* workspace, long long workspace_bytes, void* stream) {
  SERL_CHECK_ARG(type >= 0 && type <= 2, "topk_distill: type must be 0 (fp32), 1 (bf16) or 2 (fp16)");
  SERL_CHECK_ARG(teacher_type == type || teacher_type == SERL_F32, "topk_distill: the teacher's type must be the logits' or fp32");
  SERL_CHECK_ARG(R >= 0 && R <= DIST_MAXR && V >= 1 && V <= 0x3fffffff && K >= 1 && K <= DIST_MAXK,
                 "topk_distill: R in [0, %d], V in [1, 2^30) and K in [1, %d]", DIST_MAXR, DIST_MAXK);
  SERL_CHECK_ARG(temperature >= 0x1p-20f && temperature <= 0x1p20f, "topk_distill: the temperature must be in [2^-20, 2^20]");
  if (R == 0) return SERL_OK;
  SERL_CHECK_ARG(logits && teacher && index && loss, "topk_distill: null pointer");
  SERL_CHECK_ARG(ldl >= 0 && ldt >= 0 && ldi >= 0 && (!dlogits || R <= 1 || ldd >= V),
                 "topk_distill: negative row stride, or output rows overlap");
  SERL_CHECK_ARG(!dlogits || dlogits != logits || R <= 1 || ldl == ldd, "topk_distill: in place needs the same row stride");
  const bool wide = V >= 2 * dist_vec(type);
  const DistPlan p = dist_plan(type, R, V);
  const long long need = dist_ws(p, R, K);
  SERL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                 "topk_distill: workspace of %lld bytes needed, %lld available", need, workspace ? workspace_bytes : 0);
  SERL_CHECK_ARG(p.pieces == 1 || (long long)R * p.pieces * (DIST_CUT + 64) < (1ll << 32),      // a launch has less than 2^32 threads
                 "topk_distill: too many rows of this length: R at most %lld", ((1ll << 32) - 1) / (DIST_CUT + 64) / p.pieces);
  DistArgs a{};
  a.logits = logits; a.ldl = ldl; a.teacher = teacher; a.ldt = ldt; a.index = index; a.ldi = ldi; a.dlogits = dlogits;
  a.ldd = ldd; a.coef = coef; a.loss = loss; a.part = workspace;
  a.taken = workspace ? workspace + (long long)R * p.pieces * 2 : nullptr; a.R = R; a.V = V; a.K = K;
  a.teacher_f32 = teacher_type == SERL_F32; a.index64 = index64 != 0; a.tau = temperature; a.pieces = p.pieces;
  a.piece_vecs = p.piece_vecs;
  hipStream_t st = (hipStream_t)stream;
#define DIST_GO(T, W) (wide ? dist_launch<T, W>(a, st) : dist_launch<T, 1>(a, st))
  if (type == SERL_F32) DIST_GO(F32, 4);
  else if (type == SERL_BF16) DIST_GO(BF16, 8);
  else DIST_GO(F16, 8);
#undef DIST_GO
  SERL_CHECK_LAUNCH("topk_distill");
  return SERL_OK;
}
