// What a network's last layer is asked for and trained with, over rows of logits: log
// probabilities of given tokens with entropy and top alternatives, and the distillation loss
// against a teacher's top logits with its gradient.  No counterpart in the reference, whose
// row softmax (internal/cgo/metal_bridge_activation.m:300-321) is the nearest kin.
//
// A row is read once: every thread keeps the running maximum m and, relative to it, the
// sums S = sum e^(x-m) and U = sum e^(x-m) (x-m) of the elements it has seen, and pairs of
// (m, S, U) merge by
//   m' = max(m1, m2),  S' = sum_i S_i e^(m_i-m'),  U' = sum_i e^(m_i-m') (U_i + (m_i-m') S_i).
// log p(t) = (x_t - m) - log S, and the entropy is log S - U / S.
//
// Short rows (up to 1024 logits) are held in the registers of one warp.  Longer ones go through a
// ring of shared-memory stages of 4096 or 8192 logits: one warp of a block feeds it with bulk copies,
// ahead of the eight or sixteen warps that add (T threads), and into the next row; another one or two
// take care of what is little and slow, the tokens, targets and results of a row.  Few long rows are shared by the up to 8 blocks
// of a cluster.  All merges have a fixed order: results repeat bit for bit.
#include <algorithm>

#include "kernels.h"
#include "launch.cuh"
#include "ptx.cuh"
#include "status.cuh"

namespace gonn {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int BLOCK = 256;                          // adding threads of a ring kernel, and
constexpr int WIDE = 512;                           // of the step over wide rows
constexpr int ROWS_BLOCK = 256;                     // threads of a kernel with a warp per row
constexpr uint32_t QUADS = 4;                       // 16-byte pieces of an adding thread in one stage
constexpr uint32_t WARP_ROW = 1024;                 // longest row that one warp holds
constexpr uint32_t MAX_SHARE = 8;                   // blocks of a cluster

__device__ __forceinline__ void report_index(GemmStatus* st, uint32_t kind, uint64_t row, int index) {
  volatile GemmStatus* v = st;  // mapped host memory: plain stores, the first report wins
  if (v->code == 0u) {
    v->where = kind;
    v->tile = uint32_t(row);
    v->kblock = uint32_t(index);
    v->code = kStatusBadIndex;
  }
}

// 2^x for sums: results below 2^-126 become 0.
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- barriers of the T adding threads alone -------------------------------------------------
template <int T>
__device__ __forceinline__ void adders_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(T) : "memory");
}
template <int T>
__device__ __forceinline__ bool adders_or(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred P, Q;\n\t"
      "setp.ne.u32 P, %1, 0;\n\t"
      "bar.red.or.pred Q, 1, %2, P;\n\t"
      "selp.u32 %0, 1, 0, Q;\n\t"
      "}\n"
      : "=r"(r)
      : "r"(uint32_t(v)), "n"(T)
      : "memory");
  return r != 0;
}
// ---- statistics of (part of) a row ------------------------------------------------------
// What is summed beside S: nothing; U for the entropy; or the tempered sum e^((x-m)/T), with
// `c` = log2(e) / T.  With T = 2 or 4, e^(x-m) is the tempered exponential squared once or twice: one
// exponential an element instead of two, of which an SM does 16 a clock.
enum class Sum : int { Plain = 0, Entropy = 1, Tempered = 2, Tempered2 = 3, Tempered4 = 4 };
__host__ __device__ constexpr bool tempered(Sum s) { return s == Sum::Tempered || s == Sum::Tempered2 || s == Sum::Tempered4; }

struct RowStats {
  float m = -INFINITY;
  float s = 0.f;
  float u = 0.f;
};

// The maximum that differences are taken from: a part that has seen nothing but -inf takes
// them from 0, so that its elements still give e^-inf = 0 and not NaN.
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

// Plain: `c` = log2(e) / T gives S itself a temperature.
template <Sum SUM>
__device__ __forceinline__ void rescale(RowStats& r, float m_new, float c) {
  if (m_new == r.m) return;
  if (r.m != -INFINITY) {
    const float d = r.m - m_new;
    const float f = exp2f(d * (SUM == Sum::Plain ? c : kLog2e));
    // where f is 0 the limit keeps d S finite (the difference itself may be -inf)
    if (SUM == Sum::Entropy) r.u = f * (r.u + fmaxf(d, -1e4f) * r.s);
    if (tempered(SUM)) r.u *= exp2f(d * c);
    r.s *= f;
  }
  r.m = m_new;
}

template <Sum SUM>
__device__ __forceinline__ void add(RowStats& r, float x, float ref, float c) {
  const float d = x - ref;
  const float e = exp2_ftz(d * (SUM == Sum::Plain ? c : kLog2e));
  r.s += e;
  // a masked element (-inf) adds e = 0 times a finite number
  if (SUM == Sum::Entropy) r.u = fmaf(e, fmaxf(d, -1e30f), r.u);
  if (tempered(SUM)) r.u += exp2_ftz(d * c);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Orders like the values (NaN aside); -0 counts as 0.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t b) {
  return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}

// The statistics of the adding threads in every one of them, with one barrier: each warp's, then
// all warps' in every warp.  `smem`: another one for every other row, so that the next row's may be
// written while this one's are read.
template <Sum SUM, int T>
__device__ RowStats block_merge(RowStats r, float c, RowStats (&smem)[T / 32]) {
  constexpr uint32_t WARPS = T / 32;
  const uint32_t lane = threadIdx.x & 31;
  rescale<SUM>(r, order_value(__reduce_max_sync(0xffffffffu, order_bits(r.m))), c);
  r.s = warp_sum(r.s);
  if (SUM != Sum::Plain) r.u = warp_sum(r.u);
  if (lane == 0) smem[threadIdx.x >> 5] = r;
  adders_sync<T>();
  r = smem[lane % WARPS];
  rescale<SUM>(r, order_value(__reduce_max_sync(0xffffffffu, order_bits(r.m))), c);
#pragma unroll
  for (uint32_t o = WARPS / 2; o > 0; o >>= 1) {
    r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
    if (SUM != Sum::Plain) r.u += __shfl_xor_sync(0xffffffffu, r.u, o);
  }
  return r;
}

// log p of a logit: NaN for a row that holds a NaN or +inf, -inf for a masked token and for
// every token of a row that is masked as a whole.
__device__ __forceinline__ float log_prob(const RowStats& r, float x) {
  if (x == -INFINITY && r.s == r.s) return -INFINITY;
  return (x - r.m) - logf(r.s);
}

// ---- a block's part of a long row --------------------------------------------------------
// Whole 16-byte pieces of the row's memory, split evenly over the blocks of the cluster; the up to
// three logits before the first piece belong to the first block and those behind the last one to
// the last block, a thread each.
struct Part {
  const float4* quads;  // first piece of the row
  uint32_t lead;        // logits before it
  uint32_t q0, q1;      // this block's pieces
  uint32_t first, end;  // this block's logits
  uint32_t tail;        // first logit behind the row's pieces
};

__device__ __forceinline__ Part part_of(const float* x, uint32_t vocab, uint32_t rank, uint32_t shares) {
  Part p;
  p.lead = min(uint32_t((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / 4u, vocab);
  const uint32_t all = (vocab - p.lead) / 4u;
  p.quads = reinterpret_cast<const float4*>(x + p.lead);
  p.q0 = uint32_t(uint64_t(all) * rank / shares);
  p.q1 = uint32_t(uint64_t(all) * (rank + 1) / shares);
  p.tail = p.lead + all * 4u;
  p.first = rank == 0 ? 0u : p.lead + p.q0 * 4u;
  p.end = rank + 1 == shares ? vocab : p.lead + p.q1 * 4u;
  return p;
}
// This thread's logit outside the pieces, or -1.
__device__ __forceinline__ int extra_of(const Part& p) {
  const uint32_t t = threadIdx.x;
  if (t < 4) return p.first == 0 && t < p.lead ? int(t) : -1;
  return p.tail >= p.first && p.tail + t - 4u < p.end && t < 8 ? int(p.tail + t - 4u) : -1;
}

__device__ __forceinline__ float4 masked_quad() { return make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }

// ---- the ring ------------------------------------------------------------------------------
// full[s]: the feeder's arrival and the stage's bytes; empty[s]: the adding warps (or the storing one).
template <int T>
constexpr uint32_t kStage = QUADS * T;  // pieces of a stage: 16 or 32 KB
template <int T>
constexpr uint32_t kStages = T == WIDE ? 6 : 4;  // 192 KB and one block an SM, or 64 KB and two or three
template <int T>
struct RingBars {
  uint64_t full[kStages<T>], empty[kStages<T>];
  __device__ void init(uint32_t leavers) {
    for (uint32_t i = 0; i < kStages<T>; ++i) {
      ptx::mbar_init(ptx::smem_u32(&full[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty[i]), leavers);
    }
  }
};

// What all roles of a ring kernel share.  A wait that runs out is reported and the roles carry on
// without waiting (every index they use stays within the row): results are then undefined, the
// call fails, and all barriers are still met.
struct Waits {
  GemmStatus* status;
  volatile uint32_t* abort_flag;
  __device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, uint32_t where) const {
    if (!ptx::mbar_wait(ptx::smem_u32(bar), parity, abort_flag)) gave_up(where);
  }
  __device__ __forceinline__ void wait_cluster(uint64_t* bar, uint32_t parity, uint32_t where) const {
    if (!ptx::mbar_wait_cluster(ptx::smem_u32(bar), parity, abort_flag)) gave_up(where);
  }
  __device__ __noinline__ void gave_up(uint32_t where) const {
    if (first_to_give_up(abort_flag)) report(status, 1, where, blockIdx.x, 0);
  }
};
__device__ __forceinline__ void arrive(uint64_t* bar) { ptx::mbar_arrive(ptx::smem_u32(bar)); }

// Place and phase of a ring's next stage.
template <int T>
struct RingAt {
  uint32_t slot = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == kStages<T>) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// One lane feeds a part's stages; a part without pieces is one empty stage.
template <int T>
__device__ __forceinline__ void feed_part(const Part& p, float4* ring, RingBars<T>& bars, RingAt<T>& at,
                                          const Waits& w) {
  uint32_t q = p.q0;
  do {
    const uint32_t n = min(kStage<T>, p.q1 - q);
    w.wait(&bars.empty[at.slot], at.phase ^ 1u, 0x10u | at.slot);
    const uint32_t full = ptx::smem_u32(&bars.full[at.slot]);
    if (n) {
      ptx::mbar_arrive_expect_tx(full, n * 16);
      ptx::bulk_load(ptx::smem_u32(ring + at.slot * kStage<T>), p.quads + q, n * 16, full);
    } else {
      ptx::mbar_arrive(full);
    }
    at.next();
    q += kStage<T>;
  } while (q < p.q1);
}

// A thread's logits of the stage that holds the pieces from `q`; -inf past the part's end.
template <int T>
__device__ __forceinline__ void read_stage(const Part& p, uint32_t q, const float4* stage, float4 (&v)[QUADS]) {
  const float4* from = stage + threadIdx.x;
  if (q + kStage<T> <= p.q1) {
#pragma unroll
    for (uint32_t j = 0; j < QUADS; ++j) v[j] = from[j * T];
  } else {
#pragma unroll
    for (uint32_t j = 0; j < QUADS; ++j) v[j] = q + j * T + threadIdx.x < p.q1 ? from[j * T] : masked_quad();
  }
}
template <int T>
__device__ __forceinline__ void take_stage(const Part& p, uint32_t q, const float4* ring, RingBars<T>& bars,
                                           const RingAt<T>& at, const Waits& w, float4 (&v)[QUADS]) {
  w.wait(&bars.full[at.slot], at.phase, at.slot);
  read_stage<T>(p, q, ring + at.slot * kStage<T>, v);
}
// The warp does not need the stage any more.  What it has read must have been used by something that
// cannot move behind the arrival (a vote, a store): the arrival can overtake loads under way, and the
// next copy then lands in front of them (one backward pass in ten over 2048 x 32000 had 256 bytes of a
// row from the next copy).
template <int T>
__device__ __forceinline__ void leave_stage(RingBars<T>& bars, const RingAt<T>& at) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) arrive(&bars.empty[at.slot]);
}

__device__ __forceinline__ float max4(const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }

template <Sum SUM>
__device__ __forceinline__ void add_one(RowStats& r, float x, float c) {
  if (x > r.m) rescale<SUM>(r, x, c);
  add<SUM>(r, x, reference(r.m), c);
}

// A thread's running statistics while it streams a row, two elements an instruction.  An exponent
// is one fused multiply-add, x c - b with b = m c rounded (the same b for all elements, so its
// rounding is a common factor, which result() takes out again); logits beyond 1e37, where the
// products could overflow, take the difference first (`far`).
//
// m is a reference and need not be the maximum: it is the largest logit of the warp's first stage,
// and moves only when one comes whose exponential would be above 2^58 (the sums are then still far
// from overflow).  With the reference at each thread's running maximum some lane of a warp moved it
// at nearly every stage (1021 x 50001, top 5: 53 us instead of 50).
template <Sum SUM>
struct Stream {
  const float slack;
  float m = -INFINITY, top = -INFINITY, b = 0.f, bt = 0.f;
  float2 s = make_float2(0.f, 0.f), u = make_float2(0.f, 0.f);
  bool far = false;

  // scale of S itself; Plain: log2(e) / T
  static __device__ __forceinline__ float scale(float c) { return SUM == Sum::Plain ? c : kLog2e; }

  __device__ __forceinline__ explicit Stream(float c) : slack(58.f / (tempered(SUM) ? fmaxf(c, kLog2e) : scale(c))) {}

  __device__ __forceinline__ void raise(float most, float c) {
    const float k = scale(c), ref = reference(most);
    const bool far_new = !(fabsf(ref) < 1e37f);
    const float b_new = far_new ? 0.f : ref * k, bt_new = far_new ? 0.f : ref * c;
    if (m != -INFINITY) {
      const bool apart = far || far_new;
      const float d = apart ? (m - most) * k : b - b_new, dt = apart ? (m - most) * c : bt - bt_new;
      const float f = exp2f(d);
      if (SUM == Sum::Entropy) {
        const float by = fmaxf(d, -1e4f);  // where f is 0 the limit keeps the product finite
        u.x = f * (u.x + by * s.x);
        u.y = f * (u.y + by * s.y);
      }
      if (tempered(SUM)) {
        const float ft = exp2f(dt);
        u.x *= ft;
        u.y *= ft;
      }
      s.x *= f;
      s.y *= f;
    }
    m = most;
    b = b_new;
    bt = bt_new;
    far = far_new;
  }

  // The exponent of scale `by` (whose b is `off`) of two elements.
  __device__ __forceinline__ float2 exponent(float x, float y, float by, float off) const {
    if (far) return make_float2((x - m) * by, (y - m) * by);
    return ptx::fma2(make_float2(x, y), make_float2(by, by), make_float2(-off, -off));
  }
  // Adds two elements; returns their tempered exponentials (Plain, Entropy: those of S).
  __device__ __forceinline__ float2 add_pair(float x, float y, float c) {
    if (SUM == Sum::Tempered2 || SUM == Sum::Tempered4) {
      const float2 t = exponent(x, y, c, bt);
      const float2 e = make_float2(exp2_ftz(t.x), exp2_ftz(t.y));
      u = ptx::add2(u, e);
      if (SUM == Sum::Tempered2) {
        s = ptx::fma2(e, e, s);
      } else {
        const float2 sq = make_float2(e.x * e.x, e.y * e.y);
        s = ptx::fma2(sq, sq, s);
      }
      return e;
    }
    const float2 t = exponent(x, y, scale(c), b);
    const float2 e = make_float2(exp2_ftz(t.x), exp2_ftz(t.y));
    s = ptx::add2(s, e);
    // a masked element (-inf) adds e = 0 times a finite number
    if (SUM == Sum::Entropy) u = ptx::fma2(e, make_float2(fmaxf(t.x, -1e30f), fmaxf(t.y, -1e30f)), u);
    if (SUM == Sum::Tempered) {
      const float2 w = exponent(x, y, c, bt);
      u = ptx::add2(u, make_float2(exp2_ftz(w.x), exp2_ftz(w.y)));
    }
    return e;
  }

  // Adds a thread's logits of a stage and leaves their exponentials, relative to m as it is then, in
  // their place.  Returns their maximum.
  __device__ __forceinline__ float add(float4 (&v)[QUADS], float c) {
    float most = max4(v[0]);
#pragma unroll
    for (uint32_t j = 1; j < QUADS; ++j) most = fmaxf(most, max4(v[j]));
    // (the whole warp moves together: its lanes hold logits of one row)
    if (__any_sync(0xffffffffu, most > m + slack)) raise(fmaxf(m, order_value(__reduce_max_sync(0xffffffffu, order_bits(most)))), c);
    top = fmaxf(top, most);
#pragma unroll
    for (uint32_t j = 0; j < QUADS; ++j) {
      const float2 a = add_pair(v[j].x, v[j].y, c), z = add_pair(v[j].z, v[j].w, c);
      v[j] = make_float4(a.x, a.y, z.x, z.y);
    }
    return most;
  }

  __device__ __forceinline__ RowStats result(float c) const {
    RowStats r;
    r.m = m;
    const float ref = reference(m);
    // m c - b, exactly
    const float off = far ? 0.f : fmaf(ref, scale(c), -b), off_t = far ? 0.f : fmaf(ref, c, -bt);
    const float f = exp2f(-off);
    r.s = (s.x + s.y) * f;
    if (SUM == Sum::Entropy) r.u = ((u.x + u.y) - off * (s.x + s.y)) * f * 0.6931471805599453f;
    if (tempered(SUM)) r.u = (u.x + u.y) * exp2f(-off_t);
    rescale<SUM>(r, fmaxf(m, top), c);  // (m is one of the row's logits too)
    return r;
  }
};

// ---- alternatives -------------------------------------------------------------------------
// Orders like (value, lowest index first): larger keys come first among the alternatives.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) {
  return (uint64_t(order_bits(x)) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - uint32_t(key); }
__device__ __forceinline__ float key_value(uint64_t key) { return order_value(uint32_t(key >> 32)); }
constexpr uint32_t kMaskedBits = 0x007fffffu;  // order_bits(-inf); below it only NaN

// The largest `want` keys a block has met.  A key is kept when it lies above a floor that is known
// to have `want` keys above it.  The first floor comes from the threads' maxima of their first 32
// logits (as many of those as wanted lie above it, so as many logits do).  Before the
// buffer can have filled up (in rows without an order), the threads look whether there are more than
// kCrowd keys; then the surplus is thrown out and the floor rises.  (With a look every 16 stages
// the buffer did fill up: 2048 x 64000, top 128, 349 us instead of 193.)
struct Selection {
  static constexpr uint32_t CAP = 1024;
  uint64_t key[CAP];
  uint64_t floor;
  uint32_t count;
  uint32_t part[2][BLOCK / 32];
};

constexpr uint32_t kCrowd = 2 * kMaxTop + 64;  // more keys than that are thinned out

// Throws out the smallest of the n > want + want / 2 + 16 keys (all different): the `want` largest
// stay and up to want / 2 + 16 more.  All threads look for a bound, two bits a round, with a barrier
// a round; they stop at the first that leaves few enough.  (The exact bound, a bit a round, took
// 11000 clocks of a row's 50000; this takes about 2500.)  Ends with a barrier.
__device__ __noinline__ void keep_largest(Selection& s, uint32_t n, uint32_t want) {
  constexpr uint32_t PER = Selection::CAP / BLOCK, WARPS = BLOCK / 32;
  const uint32_t most = want + want / 2 + 16;
  uint64_t mine[PER];
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i) {
    const uint32_t at = i * BLOCK + threadIdx.x;
    mine[i] = at < n ? s.key[at] : 0ull;
  }
  uint64_t floor = 0;
  uint32_t turn = 0;
  for (int bit = 62; bit >= 0; bit -= 2) {
    // keys at or above the three bounds, 10 bits each: a warp has at most 128 keys
    uint32_t above = 0;
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i)
#pragma unroll
      for (uint32_t k = 0; k < 3; ++k) above += uint32_t(mine[i] >= (floor | (uint64_t(k + 1) << bit))) << (10 * k);
    above = __reduce_add_sync(0xffffffffu, above);
    if ((threadIdx.x & 31) == 0) s.part[turn][threadIdx.x >> 5] = above;
    adders_sync<BLOCK>();
    uint32_t c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
    for (uint32_t w = 0; w < WARPS; ++w) {
      above = s.part[turn][w];
      c1 += above & 1023u;
      c2 += above >> 10 & 1023u;
      c3 += above >> 20;
    }
    turn ^= 1u;
    const uint32_t digit = c3 >= want ? 3u : c2 >= want ? 2u : c1 >= want ? 1u : 0u;
    floor |= uint64_t(digit) << bit;
    const uint32_t left = digit == 3 ? c3 : digit == 2 ? c2 : c1;
    if (digit && left <= most) break;
  }
  if (threadIdx.x == 0) {
    s.count = 0;
    s.floor = floor;
  }
  adders_sync<BLOCK>();
#pragma unroll
  for (uint32_t i = 0; i < PER; ++i)
    if (mine[i] >= floor && mine[i] != 0) s.key[atomicAdd(&s.count, 1u)] = mine[i];
  adders_sync<BLOCK>();
}

// The first floor from the threads' maxima, 18 bits of it: one warp looks for the largest bound
// with `want` maxima at or above it, two bits a round, with the three counts of a round in one
// word.  (All threads counting together, a barrier a bit, took 2100 clocks of a row's 27000.)
// `maxima`: room for BLOCK words.
__device__ void first_floor(Selection& s, uint32_t* maxima, float most, uint32_t want) {
  maxima[threadIdx.x] = order_bits(most);
  adders_sync<BLOCK>();
  if (threadIdx.x < 32) {
    uint32_t mine[BLOCK / 32];
#pragma unroll
    for (uint32_t i = 0; i < BLOCK / 32; ++i) mine[i] = maxima[i * 32 + threadIdx.x];
    uint32_t floor = 0;
    for (int bit = 30; bit >= 14; bit -= 2) {
      uint32_t above = 0;
#pragma unroll
      for (uint32_t i = 0; i < BLOCK / 32; ++i)
#pragma unroll
        for (uint32_t k = 0; k < 3; ++k) above += uint32_t(mine[i] >= (floor | ((k + 1) << bit))) << (10 * k);
      above = __reduce_add_sync(0xffffffffu, above);
      const uint32_t c1 = above & 1023u, c2 = above >> 10 & 1023u, c3 = above >> 20;
      const uint32_t digit = c3 >= want ? 3u : c2 >= want ? 2u : c1 >= want ? 1u : 0u;
      floor |= digit << bit;
    }
    if (threadIdx.x == 0) {
      s.floor = uint64_t(floor) << 32;
      s.count = 0;
    }
  }
  adders_sync<BLOCK>();
}

// The floor's value as a bound on logits; one below the order of -inf lets everything pass.
__device__ __forceinline__ float floor_value(uint64_t floor) {
  return uint32_t(floor >> 32) <= kMaskedBits ? -INFINITY : key_value(floor);
}
constexpr uint32_t FIRST = 2;  // stages that the first floor is taken from

// Which of a thread's 16 logits from piece `q` may lie above the floor, a bit each.
__device__ __forceinline__ uint32_t above_floor(const Part& p, uint32_t q, const float4 (&v)[QUADS], float low) {
  uint32_t hits = 0;
#pragma unroll
  for (uint32_t j = 0; j < QUADS; ++j) {
    const uint32_t four = uint32_t(v[j].x >= low) | uint32_t(v[j].y >= low) << 1 | uint32_t(v[j].z >= low) << 2 |
                          uint32_t(v[j].w >= low) << 3;
    if (q + j * BLOCK + threadIdx.x < p.q1) hits |= four << (4 * j);
  }
  return hits;
}

// Where a thread stands since the last look: the first of its logits of the step that found no room
// (`left`, 16 to a stage; the count only grows between two looks, so none after it did either),
// whether that is so of the logit outside the pieces, and whether it saw the buffer fill up.
struct Offer {
  uint32_t left = 0xffffffffu;
  bool outside = false, over = false;
};

// Stores a logit's key unless it lies below the floor; false when there is no room.
__device__ __forceinline__ bool store_key(Selection& s, uint64_t floor, float x, uint32_t index, Offer& o) {
  const uint64_t key = order_key(x, index);
  if (key < floor) return true;
  const uint32_t at = atomicAdd(&s.count, 1u);
  o.over = o.over || at >= kCrowd;
  if (at >= Selection::CAP) return false;
  s.key[at] = key;
  return true;
}

// Offers the marked ones of a thread's logits of the k-th stage of a step, which is still in shared
// memory.
__device__ __forceinline__ void offer_stage(Selection& s, const Part& p, uint32_t q, uint32_t k, const float4* stage,
                                            uint32_t hits, uint64_t floor, Offer& o) {
  while (hits && o.left == 0xffffffffu) {
    const uint32_t i = uint32_t(__ffs(int(hits))) - 1u;
    const uint32_t piece = (i >> 2) * BLOCK + threadIdx.x;
    const float x = reinterpret_cast<const float*>(stage + piece)[i & 3u];
    if (!store_key(s, floor, x, p.lead + (q + piece) * 4u + (i & 3u), o)) o.left = k * 16u + i;
    hits &= hits - 1u;
  }
}

// The look after a step of `stages` stages from piece `q`: throws out the surplus when there is one,
// and goes on with what had found no room (from the row itself: that is rare).  At the row's end a
// surplus that the sort can do with may stay.  All adding threads call it.
__device__ __forceinline__ void settle(Selection& s, const float* x, const Part& p, uint32_t q, uint32_t stages,
                                       int extra, uint32_t want, bool last, Offer& o) {
  if (last) o.over = o.left != 0xffffffffu || o.outside;
  while (adders_or<BLOCK>(o.over)) {
    keep_largest(s, min(s.count, Selection::CAP), want);
    if (!adders_or<BLOCK>(o.left != 0xffffffffu || o.outside)) break;
    o.over = false;
    const uint64_t floor = s.floor;
    const float low = floor_value(floor);
    if (o.outside) o.outside = !store_key(s, floor, x[extra], uint32_t(extra), o);
    uint32_t i = o.left;
    o.left = 0xffffffffu;
    for (; i < stages * 16u; ++i) {
      const uint32_t piece = q + (i >> 4) * kStage<BLOCK> + (i >> 2 & 3u) * BLOCK + threadIdx.x;
      if (piece >= p.q1) continue;
      const uint32_t index = p.lead + piece * 4u + (i & 3u);
      const float v = x[index];
      if (v >= low && !store_key(s, floor, v, index, o)) {
        o.left = i;
        break;
      }
    }
  }
  o = Offer{};
}

// Sorts the selection's keys: sorted[0 .. min(n, want)) in descending order.  Returns how many.
// The caller sees to it that `sorted` is complete before it is read.
__device__ uint32_t sort_selection(Selection& s, uint64_t* sorted, uint32_t want) {
  adders_sync<BLOCK>();
  uint32_t n = s.count;
  if (n > kCrowd) {  // the alternatives of several blocks
    keep_largest(s, n, want);
    n = s.count;
  }
  // a key's place is the number of keys above it
  for (uint32_t i = threadIdx.x; i < n; i += BLOCK) {
    const uint64_t mine = s.key[i];
    uint32_t place = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < n; ++j) place += s.key[j] > mine;
    if (place < want) sorted[place] = mine;
  }
  return min(n, want);
}

// ---- log probabilities ----------------------------------------------------------------------
__device__ __forceinline__ float token_logprob(const LogprobArgs& a, const RowStats& r, uint64_t row, const float* x,
                                               uint32_t t) {
  const int token = a.tokens[row * a.n_tokens + t];
  if (token < 0) return 0.f;  // none
  if (uint64_t(token) >= a.vocab) {
    report_index(a.status, INDEX_TOKEN, row, token);
    return NAN;
  }
  return log_prob(r, x[token]);
}
__device__ __forceinline__ float row_entropy(const RowStats& r) {
  return r.s == 0.f ? 0.f : logf(r.s) - r.u / r.s;
}

// The results of one row, by one warp.
__device__ __forceinline__ void write_logprobs(const LogprobArgs& a, const RowStats& r, uint64_t row, const float* x,
                                               const uint64_t* sorted) {
  const uint32_t lane = threadIdx.x & 31;
  for (uint32_t t = lane; t < a.n_tokens; t += 32) a.logprobs[row * a.n_tokens + t] = token_logprob(a, r, row, x, t);
  if (a.entropy && lane == 0) a.entropy[row] = row_entropy(r);
  const bool nan = !(r.s == r.s);
  for (uint32_t k = lane; k < a.top_n; k += 32) {
    const uint64_t key = sorted[k];
    a.top_tokens[row * a.top_n + k] = nan ? -1 : int(key_index(key));
    a.top_logprobs[row * a.top_n + k] = nan ? NAN : log_prob(r, key_value(key));
  }
}

// Long rows.  With shares > 1 a cluster has exactly one row.
template <bool TOP>
__global__ void __launch_bounds__(BLOCK + 64, 3)
logprobs_ring_kernel(const LogprobArgs a, uint32_t shares) {
  constexpr int T = BLOCK, WARPS = T / 32;
  extern __shared__ float4 ring[];
  __shared__ RingBars<T> bars;
  __shared__ uint64_t ready[2], freed[2];  // a row's results: written by the adders, read by the server
  __shared__ uint32_t abort_word;
  __shared__ RowStats result[2], merged[2][WARPS];
  __shared__ uint64_t sorted[2][TOP ? kMaxTop : 1];
  __shared__ Selection sel;
  const uint32_t warp = threadIdx.x >> 5, rank = blockIdx.x % shares, vocab = uint32_t(a.vocab);
  const uint64_t first_row = blockIdx.x / shares, step = gridDim.x / shares;
  if (threadIdx.x == 0) {
    bars.init(WARPS);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(ptx::smem_u32(&ready[i]), WARPS);
      ptx::mbar_init(ptx::smem_u32(&freed[i]), 1);
    }
    abort_word = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  __syncthreads();
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  const Waits w{a.status, &abort_word};

  if (warp == WARPS) {  // feeder
    if ((threadIdx.x & 31) == 0) {
      RingAt<T> at;
      for (uint64_t row = first_row; row < a.rows; row += step)
        feed_part<T>(part_of(a.x + row * a.ld, vocab, rank, shares), ring, bars, at, w);
    }
    __syncwarp();
  } else if (warp == WARPS + 1) {  // server
    if (shares == 1) {
      uint32_t i = 0;
      for (uint64_t row = first_row; row < a.rows; row += step, ++i) {
        w.wait(&ready[i & 1], (i >> 1) & 1u, 0x20u);
        write_logprobs(a, result[i & 1], row, a.x + row * a.ld, sorted[i & 1]);
        __syncwarp();
        if ((threadIdx.x & 31) == 0) arrive(&freed[i & 1]);
      }
    }
  } else {  // adders
    RingAt<T> at;
    uint32_t i = 0;
    for (uint64_t row = first_row; row < a.rows; row += step, ++i) {
      const float* x = a.x + row * a.ld;
      const Part p = part_of(x, vocab, rank, shares);
      const int extra_at = extra_of(p);
      const float extra = extra_at >= 0 ? x[extra_at] : -INFINITY;
      Stream<Sum::Entropy> stream(kLog2e);
      Offer mine;
      uint32_t q = p.q0;
      if (TOP) {  // the first stages stay until there is a floor
        RingAt<T> again = at;
        float most = extra;
#pragma unroll 1
        for (uint32_t k = 0; k < FIRST && (k == 0 || q + k * kStage<T> < p.q1); ++k) {
          float4 v[QUADS];
          take_stage<T>(p, q + k * kStage<T>, ring, bars, at, w, v);
          most = fmaxf(most, stream.add(v, kLog2e));
          at.next();
        }
        // the place of this row's result: the server has read the one of two rows ago
        w.wait(&freed[i & 1], ((i >> 1) & 1u) ^ 1u, 0x21u);
        static_assert(!TOP || sizeof(sorted[0]) >= BLOCK * 4, "room for the maxima");
        first_floor(sel, reinterpret_cast<uint32_t*>(sorted[i & 1]), most, a.top_n);
        const uint64_t floor = sel.floor;
        const float low = floor_value(floor);
        if (extra_at >= 0 && extra >= low)
          mine.outside = !store_key(sel, floor, extra, uint32_t(extra_at), mine);
#pragma unroll 1
        for (uint32_t k = 0; k < FIRST && (k == 0 || q + k * kStage<T> < p.q1); ++k) {
          const float4* stage = ring + again.slot * kStage<T>;
          if (most >= low) {
            float4 v[QUADS];
            read_stage<T>(p, q + k * kStage<T>, stage, v);
            const uint32_t hits = above_floor(p, q + k * kStage<T>, v, low);
            offer_stage(sel, p, q + k * kStage<T>, k, stage, hits, floor, mine);
          }
          leave_stage<T>(bars, again);
          again.next();
        }
        settle(sel, x, p, q, FIRST, extra_at, a.top_n, q + FIRST * kStage<T> >= p.q1, mine);
        q += FIRST * kStage<T>;
      }
      // stages of the next step: as many as bring at most about half of CAP keys, and at least three
      // times as many as have been seen (`want` is at most 128)
      const uint32_t grow = TOP ? Selection::CAP / 2 / a.top_n - 1 : 1;
      uint32_t stages = FIRST * grow;
      while (q < p.q1 || (!TOP && q == p.q0)) {
        const uint64_t floor = TOP ? sel.floor : 0;
        const float low = TOP ? floor_value(floor) : INFINITY;
#pragma unroll 1
        for (uint32_t k = 0; k < stages && (k == 0 || q + k * kStage<T> < p.q1); ++k) {
          float4 v[QUADS];
          take_stage<T>(p, q + k * kStage<T>, ring, bars, at, w, v);
          float4 raw[QUADS];
#pragma unroll
          for (uint32_t j = 0; j < QUADS; ++j) raw[j] = v[j];
          if (stream.add(raw, kLog2e) >= low && TOP) {
            const float4* stage = ring + at.slot * kStage<T>;
            const uint32_t hits = above_floor(p, q + k * kStage<T>, v, low);
            offer_stage(sel, p, q + k * kStage<T>, k, stage, hits, floor, mine);
          }
          leave_stage<T>(bars, at);
          at.next();
        }
        if (TOP) settle(sel, x, p, q, stages, -1, a.top_n, q + stages * kStage<T> >= p.q1, mine);
        q += stages * kStage<T>;
        stages = min((q - p.q0) / kStage<T> * grow, 1u << 20);
      }
      RowStats r = stream.result(kLog2e);
      add_one<Sum::Entropy>(r, extra, 0.f);
      r = block_merge<Sum::Entropy, T>(r, 0.f, merged[i & 1]);
      if (!TOP) w.wait(&freed[i & 1], ((i >> 1) & 1u) ^ 1u, 0x21u);
      uint32_t found = 0;
      if (TOP) found = sort_selection(sel, sorted[i & 1], a.top_n);
      if (threadIdx.x == 0) result[i & 1] = r;
      if (TOP && shares > 1) {  // for the first block of the cluster
        adders_sync<T>();
        if (threadIdx.x == 0) sel.count = found;
      }
      // (the next row's first floor comes behind barriers that all threads reach after this)
      __syncwarp();
      if ((threadIdx.x & 31) == 0) arrive(&ready[i & 1]);
    }
  }

  if (shares > 1) {
    __syncthreads();
    ptx::cluster_sync_all();  // every block's results are in place
    if (rank == 0 && warp < WARPS) {
      // All peers are asked at once, a lane each (a word from another block's shared memory takes
      // up to a thousand clocks).
      const uint32_t lane = threadIdx.x & 31, peer = min(lane, shares - 1);
      const uint32_t at = ptx::mapa_shared(ptx::smem_u32(&result[0]), peer);
      RowStats r;
      r.m = ptx::ld_shared_cluster(at);
      r.s = ptx::ld_shared_cluster(at + 4);
      r.u = ptx::ld_shared_cluster(at + 8);
      if (lane >= shares) r = RowStats{};
      rescale<Sum::Entropy>(r, order_value(__reduce_max_sync(0xffffffffu, order_bits(r.m))), 0.f);
      r.s = warp_sum(r.s);
      r.u = warp_sum(r.u);
      if (TOP) {  // the blocks' own alternatives, at most 8 x 128, behind one another
        uint32_t theirs = ptx::ld_shared_cluster_u32(ptx::mapa_shared(ptx::smem_u32(&sel.count), peer));
        if (lane >= shares) theirs = 0;
        uint32_t before = 0;  // keys of the peers below this lane's
        for (uint32_t k = 0; k + 1 < shares; ++k) {
          const uint32_t n = __shfl_sync(0xffffffffu, theirs, k);
          if (k < lane) before += n;
        }
        const uint32_t all = __shfl_sync(0xffffffffu, before + theirs, shares - 1);
        uint64_t key[kMaxTop * MAX_SHARE / T];
        uint32_t to[kMaxTop * MAX_SHARE / T];
#pragma unroll
        for (uint32_t i = 0; i < kMaxTop * MAX_SHARE / T; ++i) {
          const uint32_t from = (i * T + threadIdx.x) / kMaxTop, k = threadIdx.x % kMaxTop;
          const uint32_t n = __shfl_sync(0xffffffffu, theirs, from), base = __shfl_sync(0xffffffffu, before, from);
          const bool there = from < shares && k < n;
          to[i] = there ? base + k : 0xffffffffu;
          if (there) key[i] = ptx::ld_shared_cluster_u64(ptx::mapa_shared(ptx::smem_u32(&sorted[0][k]), from));
        }
#pragma unroll
        for (uint32_t i = 0; i < kMaxTop * MAX_SHARE / T; ++i)
          if (to[i] != 0xffffffffu) sel.key[to[i]] = key[i];
        adders_sync<T>();
        if (threadIdx.x == 0) sel.count = all;
        sort_selection(sel, sorted[1], a.top_n);
        adders_sync<T>();
      }
      if (warp == 0) write_logprobs(a, r, first_row, a.x + first_row * a.ld, sorted[1]);
    }
    ptx::cluster_sync_all();  // no block leaves while another still reads its shared memory
  }
  __syncthreads();
  wait_out(&abort_word);
}

// One warp a row, PER logits a lane in registers.
template <int PER>
__device__ __forceinline__ void load_row(const float* x, uint32_t vocab, uint32_t lane, float (&v)[PER]) {
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t i = uint32_t(j) * 32u + lane;
    v[j] = i < vocab ? x[i] : -INFINITY;
  }
}
template <Sum SUM, int PER>
__device__ __forceinline__ RowStats stats_of(const float (&v)[PER], float c) {
  RowStats r;
#pragma unroll
  for (int j = 0; j < PER; ++j) r.m = fmaxf(r.m, v[j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r.m = fmaxf(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
  const float ref = reference(r.m);
#pragma unroll
  for (int j = 0; j < PER; ++j) add<SUM>(r, v[j], ref, c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
    r.u += __shfl_xor_sync(0xffffffffu, r.u, o);
  }
  return r;
}

template <int PER>
__global__ void __launch_bounds__(ROWS_BLOCK) logprobs_warp_kernel(const LogprobArgs a) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  const uint32_t lane = threadIdx.x & 31, vocab = uint32_t(a.vocab);
  const uint64_t row = uint64_t(blockIdx.x) * (ROWS_BLOCK / 32) + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const float* x = a.x + row * a.ld;
  float v[PER];
  load_row<PER>(x, vocab, lane, v);
  const RowStats r = stats_of<Sum::Entropy, PER>(v, 0.f);
  for (uint32_t t = lane; t < a.n_tokens; t += 32) a.logprobs[row * a.n_tokens + t] = token_logprob(a, r, row, x, t);
  if (a.entropy && lane == 0) a.entropy[row] = row_entropy(r);
  if (a.top_n == 0) return;
  const bool nan = !(r.s == r.s);
  // every round takes the largest logit that is left, the lowest index among equal ones; `taken`
  // marks the lane's logits that are gone
  uint32_t taken = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (uint32_t(j) * 32u + lane >= vocab) taken |= 1u << j;
  uint32_t best = 0, best_j = 0;  // the lane's largest order bits (0: none left) and which logit has them
  auto look = [&] {
    best = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t b = order_bits(v[j]);
      if (!(taken >> j & 1u) && b > best) {  // ascending j: equal logits keep the lowest index
        best = b;
        best_j = uint32_t(j);
      }
    }
  };
  look();
  for (uint32_t k = 0; k < a.top_n; ++k) {
    const uint32_t most = __reduce_max_sync(0xffffffffu, best);
    const uint32_t index = __reduce_min_sync(0xffffffffu, best == most ? best_j * 32u + lane : 0xffffffffu);
    if (lane == (k & 31u)) {
      const float value = key_value(uint64_t(most) << 32);
      a.top_tokens[row * a.top_n + k] = nan ? -1 : int(index);
      a.top_logprobs[row * a.top_n + k] = nan ? NAN : log_prob(r, value);
    }
    if ((index & 31u) == lane) {
      taken |= 1u << (index >> 5);
      look();
    }
    __syncwarp();
  }
}

// ---- distillation ---------------------------------------------------------------
// q = softmax(z / T) over the teacher's tokens of the row that are there (index in the
// vocabulary, logit above -inf), p_T = softmax(x / T), p = softmax(x):
//   loss = w T^2 sum_k q_k (log q_k - log p_T[idx_k]) + (1-w) (-log p[label])
//   dx_j = g (w T (p_T[j] - sum_{k: idx_k = j} q_k) + (1-w) (p[j] - [j = label]))
// The statistics keep S_1 = sum e^(x-m) in `s` and S_T = sum e^((x-m)/T) in `u`; where only one of
// them is wanted, or T is 1, only that one is summed.
// One warp takes care of a row's teacher and label, before the row is streamed: what it finds waits
// in shared memory.
struct Targets {
  int index[kMaxTop + 1];   // teacher tokens, then the label; -1: not there
  float take[kMaxTop + 1];  // q_k, then 1 for the label
  float x_at[kMaxTop + 1];  // the student's logit there
  float log_q[kMaxTop];
  float scale;              // of the row's gradient
  float saved[3];           // the statistics that the forward pass has left: m, u, s (Backward)
  float soft;               // 1: there is a teacher, 0: there is none, NaN: it is spoiled
};

// Reads the row's targets, the student's logits at them included: before anyone may overwrite the
// row with its gradient.  Called by one warp; `tell`: one warp of a row reports bad indices; LOSS:
// the student's logits are wanted.
template <bool LOSS>
__device__ void read_targets(const DistillArgs& a, uint64_t row, const float* x, bool tell, Targets& t) {
  constexpr int PER = kMaxTop / 32;
  const uint32_t lane = threadIdx.x & 31;
  const float inv_t = 1.f / a.temperature;
  int index[PER];
  float z[PER], x_at[PER], zm = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t k = uint32_t(i) * 32u + lane;
    index[i] = -1;
    x_at[i] = 0.f;
    z[i] = -INFINITY;
    if (k < a.top_n) {
      index[i] = a.teacher_tokens[row * a.top_n + k];
      z[i] = a.teacher_logits[row * a.top_n + k] * inv_t;
    }
  }
  int label = lane == 0 && a.labels ? a.labels[row] : -1;
  if (label >= 0 && uint64_t(label) >= a.vocab) {
    if (tell) report_index(a.status, INDEX_LABEL, row, label);
    label = -1;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (index[i] >= 0 && uint64_t(index[i]) >= a.vocab) {
      if (tell) report_index(a.status, INDEX_TEACHER, row, index[i]);
      index[i] = -1;
    }
    if (z[i] == -INFINITY) index[i] = -1;
    if (index[i] < 0) z[i] = -INFINITY;
    else if (LOSS) x_at[i] = x[index[i]];
    zm = fmaxf(zm, z[i]);
  }
  const float x_label = LOSS && label >= 0 ? x[label] : 0.f;
  zm = warp_max(zm);
  float q[PER], total = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    q[i] = index[i] >= 0 ? exp2f((z[i] - zm) * kLog2e) : 0.f;
    total += q[i];
  }
  total = warp_sum(total);
  const float inv_total = total == 0.f ? 0.f : 1.f / total, log_total = logf(total);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t k = uint32_t(i) * 32u + lane;
    if (k < a.top_n) {
      t.index[k] = index[i];
      t.take[k] = q[i] * inv_total;
      t.x_at[k] = x_at[i];
      t.log_q[k] = (z[i] - zm) - log_total;
    }
  }
  if (lane == 0) {
    t.index[a.top_n] = label;
    t.take[a.top_n] = 1.f;
    t.x_at[a.top_n] = x_label;
    t.scale = a.grad_loss ? a.grad_scale * a.grad_loss[row] : a.grad_scale;
    // a NaN among the teacher's logits spoils the whole row, not only the tokens it names
    t.soft = total == 0.f ? 0.f : total == total ? 1.f : NAN;
  }
  __syncwarp();
}

// The row's loss, in every lane of the warp that read the targets.
__device__ float row_loss(const DistillArgs& a, const RowStats& r, const Targets& t) {
  const float inv_t = 1.f / a.temperature, w = a.soft_weight;
  float far = 0.f;
  if (a.top_n) {
    const float log_u = logf(r.u);
    for (uint32_t k = threadIdx.x & 31; k < a.top_n; k += 32)
      // q_k = 0 (an underflow) contributes 0 whatever the student says
      if (t.index[k] >= 0 && t.take[k] != 0.f)
        far += t.take[k] * (t.log_q[k] - ((t.x_at[k] - r.m) * inv_t - log_u));
    far = warp_sum(far);
  }
  if (r.m == -INFINITY && r.s == 0.f && r.u == 0.f) return 0.f;  // masked as a whole: no distribution
  float loss = 0.f;
  if (!(t.soft == 0.f)) loss += w * a.temperature * a.temperature * far;
  if (t.index[a.top_n] >= 0) loss += (1.f - w) * (logf(r.s) - (t.x_at[a.top_n] - r.m));
  return loss;
}

// Factors of a row's gradient: dx = e^((x-m)/T) ks + e^(x-m) kh, minus soft q_k and hard at the
// named places.  Exponents as in Stream; what the rounding of b adds is taken out of ks and kh.
// With T = 1 both parts share an exponential, and a loss with one part has one (Plain).
struct GradFactors {
  float m, b, bt, ks, kh, soft, hard;
  bool empty, far;
};
template <Sum SUM>
__device__ __forceinline__ GradFactors grad_factors(const DistillArgs& a, const RowStats& r, const Targets& t, float c) {
  GradFactors f;
  const float scale = t.scale, soft = t.soft;
  const int label = t.index[a.top_n];
  f.empty = r.m == -INFINITY && r.s == 0.f && r.u == 0.f;
  f.m = reference(r.m);
  f.far = !(fabsf(f.m) < 1e37f);
  f.b = f.far ? 0.f : f.m * kLog2e;
  f.bt = f.far ? 0.f : f.m * c;
  const float off = f.far ? 0.f : fmaf(f.m, kLog2e, -f.b), off_t = f.far ? 0.f : fmaf(f.m, c, -f.bt);
  f.soft = soft * scale * (a.soft_weight * a.temperature);
  f.hard = label >= 0 ? scale * (1.f - a.soft_weight) : 0.f;
  f.ks = soft == 0.f || a.soft_weight == 0.f ? 0.f : f.soft / r.u * exp2f(-off_t);
  f.kh = label < 0 ? 0.f : f.hard / r.s * exp2f(-(tempered(SUM) ? off : off_t));
  if (SUM == Sum::Plain) f.ks += f.kh;
  if (f.empty) f.ks = f.kh = 0.f;
  return f;
}
// e: the tempered exponentials of two elements, e1: those of T = 1 (Tempered alone).
template <Sum SUM>
__device__ __forceinline__ float2 grad_of(float ks, float kh, float2 e, float2 e1) {
  float2 g = make_float2(e.x * ks, e.y * ks);
  if (SUM == Sum::Tempered) g = ptx::fma2(e1, make_float2(kh, kh), g);
  if (SUM == Sum::Tempered2) g = ptx::fma2(make_float2(e.x * e.x, e.y * e.y), make_float2(kh, kh), g);
  if (SUM == Sum::Tempered4) {
    const float2 sq = make_float2(e.x * e.x, e.y * e.y);
    g = ptx::fma2(make_float2(sq.x * sq.x, sq.y * sq.y), make_float2(kh, kh), g);
  }
  return g;
}
// A probability below 2^-126 gives 0.
template <Sum SUM>
__device__ __forceinline__ float2 grad_pair(const GradFactors& f, float x, float y, float c) {
  auto exponential = [&](float by, float off) {
    float2 t;
    if (f.far) t = make_float2((x - f.m) * by, (y - f.m) * by);
    else t = ptx::fma2(make_float2(x, y), make_float2(by, by), make_float2(-off, -off));
    return make_float2(exp2_ftz(t.x), exp2_ftz(t.y));
  };
  const float2 e = exponential(c, f.bt);
  return grad_of<SUM>(f.ks, f.kh, e, SUM == Sum::Tempered ? exponential(kLog2e, f.b) : e);
}
template <Sum SUM>
__device__ __forceinline__ float grad_at(const GradFactors& f, float x, float c) {
  return f.empty ? 0.f : grad_pair<SUM>(f, x, x, c).x;
}
// A thread's logits of a stage -> their gradients.
template <Sum SUM>
__device__ __forceinline__ void grad_stage(const GradFactors& f, float4 (&v)[QUADS], float c) {
#pragma unroll
  for (uint32_t j = 0; j < QUADS; ++j) {
    const float2 a = grad_pair<SUM>(f, v[j].x, v[j].y, c), b = grad_pair<SUM>(f, v[j].z, v[j].w, c);
    v[j] = f.empty ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(a.x, a.y, b.x, b.y);
  }
}
// The same from the exponentials that Stream::add left when its reference was m (<= the row's
// maximum).
template <Sum SUM>
__device__ __forceinline__ void scale_stage(const GradFactors& f, float4 (&v)[QUADS], float m, float c) {
  const float ref = reference(m);
  const bool apart = f.far || !(fabsf(ref) < 1e37f);
  // nothing but masked logits: the exponentials are 0 whatever the reference is
  const float by = m == -INFINITY ? 0.f : 1.f;
  const float ks = by * f.ks * (by == 0.f ? 0.f : exp2f(apart ? (ref - f.m) * c : ref * c - f.bt));
  const float kh = by * f.kh * (by == 0.f ? 0.f : exp2f(apart ? (ref - f.m) * kLog2e : ref * kLog2e - f.b));
#pragma unroll
  for (uint32_t j = 0; j < QUADS; ++j) {
    const float2 p = make_float2(v[j].x, v[j].y), q = make_float2(v[j].z, v[j].w);
    const float2 a = grad_of<SUM>(ks, kh, p, p), b = grad_of<SUM>(ks, kh, q, q);
    v[j] = make_float4(a.x, a.y, b.x, b.y);
  }
}

// Takes the targets' part from the gradient at the places that they name, among [first, end).
// Called by one warp.  Entries that name the same place are added up before they are taken off
// where they are in one group of 32, and are taken off one group after the other where they are not
// (same-address reductions of a warp stay in order): the result does not depend on timing.  The
// reductions leave without waiting for the gradient to come back; with loads, and a loop over all
// entries for those that name a place again, this took 10000 to 17000 clocks for 65 entries, longer
// than all else that happens to a block's part of a row.
__device__ void take_targets(const DistillArgs& a, float* g, const Targets& t, const GradFactors& f, uint32_t first,
                             uint32_t end) {
  if (f.empty) return;
  const uint32_t n = a.top_n + 1, lane = threadIdx.x & 31;
  for (uint32_t k0 = 0; k0 < n; k0 += 32) {
    const uint32_t k = k0 + lane;
    const int index = k < n ? t.index[k] : -1;
    const bool here = index >= int(first) && uint32_t(index) < end;
    float by = here ? t.take[k] * (k == a.top_n ? f.hard : f.soft) : 0.f;
    const uint32_t same = __match_any_sync(0xffffffffu, here ? index : -1 - int(lane));
    const bool lead = uint32_t(__ffs(int(same))) == lane + 1;
    if (!__all_sync(0xffffffffu, lead)) {
      float sum = 0.f;
      for (uint32_t j = 0; j < 32; ++j) {
        const float other = __shfl_sync(0xffffffffu, by, int(j));
        if ((same >> j) & 1u) sum += other;
      }
      by = sum;
    }
    if (here && lead) ptx::red_add(g + index, -by);
    __syncwarp();
  }
}

__device__ __forceinline__ RowStats saved_stats(const DistillArgs& a, uint64_t row) {
  RowStats r;
  r.m = a.stats_in[row * 3];
  r.u = a.stats_in[row * 3 + 1];
  r.s = a.stats_in[row * 3 + 2];
  return r;
}
// Plain sums one of the two; with T = 1 it is both.
template <Sum SUM>
__device__ __forceinline__ void complete(RowStats& r) {
  if (SUM == Sum::Plain) r.u = r.s;
}
__device__ __forceinline__ void save_stats(const DistillArgs& a, uint64_t row, const RowStats& r) {
  a.stats[row * 3] = r.m;
  a.stats[row * 3 + 1] = r.u;
  a.stats[row * 3 + 2] = r.s;
}

// Long rows.  The step reads a row twice, the second time from L2 (see launch_step).  Parts of a row
// that leave room in the ring for the next row's first stages are read once (`keep`): their
// exponentials wait in the ring for the gradient.  (2048 x 32000: 100 us, read twice 104; in 2 to 8
// blocks' rings, 4096 x 128000 took 823 to 1142 us, read twice 683.)
//
// The serving warps read a row's targets while rows before it are being added (tfull, tempty), write
// its loss (done) and correct the gradient at the targets (written); with two of them in the step,
// each may take as long as two rows.  The blocks of a cluster send each other their statistics
// (peers).
//
// BULK: the gradient takes the logits' place in the ring and a storing warp sends each stage off
// with a bulk copy (stored[s] says that it is there) while the next is added; it also gives back
// the stages of the first reading.  (16-byte stores of the adding warps left an SM at 20 bytes a
// clock and took 6200 of a row's 13500 clocks.)  `written` comes when the next row's first stage
// does: until then the row's bytes had time to arrive.
template <DistillPass PASS>
constexpr int kServers = PASS == DistillPass::Step ? 2 : 1;  // warps that take care of the targets
template <DistillPass PASS, int T>
constexpr int kRingThreads = T + 32 + 32 * kServers<PASS> + (PASS == DistillPass::Step ? 32 : 0);
template <DistillPass PASS, int T>
constexpr int kRingBlocks = PASS != DistillPass::Step ? 3 : T == WIDE ? 1 : 2;  // an SM
template <DistillPass PASS, Sum SUM, bool BULK, int T>
__global__ void __launch_bounds__((kRingThreads<PASS, T>), (kRingBlocks<PASS, T>))
distill_ring_kernel(const DistillArgs a, uint32_t shares, bool keep) {
  constexpr int WARPS = T / 32, SERVERS = kServers<PASS>, SLOTS = 2 * SERVERS;
  extern __shared__ float4 ring[];
  __shared__ RingBars<T> bars;
  __shared__ uint64_t tfull[SLOTS], tempty[SLOTS], done[SLOTS], written[SLOTS], peers[2], stored[BULK ? kStages<T> : 1];
  __shared__ uint32_t abort_word;
  __shared__ RowStats result[SLOTS], merged[2][WARPS];
  __shared__ float4 parts[2][MAX_SHARE];  // of a row: m, s, u of every block
  __shared__ float kept_at[PASS == DistillPass::Step ? kStages<T> : 1][PASS == DistillPass::Step ? T : 1];
  __shared__ Targets targets[SLOTS];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x % shares;
  const uint32_t vocab = uint32_t(a.vocab);
  const uint64_t first_row = blockIdx.x / shares, step = gridDim.x / shares;
  const float c = kLog2e / a.temperature;
  if (threadIdx.x == 0) {
    bars.init(BULK ? 1 : WARPS);
    for (uint32_t i = 0; BULK && i < kStages<T>; ++i) ptx::mbar_init(ptx::smem_u32(&stored[i]), WARPS);
    for (int i = 0; i < SLOTS; ++i) {
      ptx::mbar_init(ptx::smem_u32(&tfull[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&tempty[i]), WARPS);
      ptx::mbar_init(ptx::smem_u32(&done[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&written[i]), BULK ? 1 : WARPS);
    }
    for (int i = 0; i < 2; ++i) ptx::mbar_init(ptx::smem_u32(&peers[i]), 1);
    abort_word = 0;
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_smem();
  }
  __syncthreads();
  if (shares > 1) ptx::cluster_sync_all();  // the peers' barriers exist
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  const Waits w{a.status, &abort_word};

  if (warp == WARPS) {  // feeder
    if (lane == 0) {
      RingAt<T> at;
      for (uint64_t row = first_row; row < a.rows; row += step) {
        const Part p = part_of(a.x + row * a.ld, vocab, rank, shares);
        feed_part<T>(p, ring, bars, at, w);
        if (PASS == DistillPass::Step && !keep) feed_part<T>(p, ring, bars, at, w);
      }
    }
    __syncwarp();
  } else if (warp > WARPS && warp <= WARPS + SERVERS) {  // servers, each with every SERVERS-th row
    const uint32_t me = warp - WARPS - 1;
    auto publish = [&](uint32_t k) {
      const uint64_t row = first_row + uint64_t(k) * step;
      if (row >= a.rows) return;
      w.wait(&tempty[k % SLOTS], ((k / SLOTS) & 1u) ^ 1u, 0x30u);
      if (PASS == DistillPass::Backward) {
        read_targets<false>(a, row, a.x + row * a.ld, rank == 0, targets[k % SLOTS]);
        if (lane < 3) targets[k % SLOTS].saved[lane] = a.stats_in[row * 3 + lane];
      }
      else if (rank == 0) read_targets<true>(a, row, a.x + row * a.ld, true, targets[k % SLOTS]);
      else if (PASS == DistillPass::Step) read_targets<false>(a, row, a.x + row * a.ld, false, targets[k % SLOTS]);
      __syncwarp();
      if (lane == 0) arrive(&tfull[k % SLOTS]);
    };
    publish(me);
    for (uint32_t i = me;; i += SERVERS) {
      const uint64_t row = first_row + uint64_t(i) * step;
      if (row >= a.rows) break;
      publish(i + SERVERS);
      const uint32_t turn = i % SLOTS, phase = (i / SLOTS) & 1u;
      w.wait(&done[turn], phase, 0x31u);
      const RowStats r = result[turn];
      if (PASS != DistillPass::Backward && rank == 0) {
        const float loss = row_loss(a, r, targets[turn]);
        if (lane == 0) {
          a.loss[row] = loss;
          if (PASS == DistillPass::Forward && a.stats) save_stats(a, row, r);
        }
      }
      if (PASS != DistillPass::Forward) {
        const GradFactors f = grad_factors<SUM>(a, r, targets[turn], c);
        const Part p = part_of(a.x + row * a.ld, vocab, rank, shares);
        w.wait(&written[turn], phase, 0x34u);
        take_targets(a, a.grad + row * a.ld_grad, targets[turn], f, p.first, p.end);
      }
      __syncwarp();
    }
  } else if (warp > WARPS + SERVERS) {  // storer
    if (BULK && lane == 0) {
      RingAt<T> at;
      int sent = -1;  // a stage whose memory may still be read
      uint32_t i = 0;
      for (uint64_t row = first_row; row < a.rows; row += step, ++i) {
        const Part p = part_of(a.x + row * a.ld, vocab, rank, shares);
        float4* gq = reinterpret_cast<float4*>(a.grad + row * a.ld_grad + p.lead);
        bool first = i > 0;
        if (!keep) {  // the stages of the first reading have only to be given back
          uint32_t q = p.q0;
          do {
            w.wait(&stored[at.slot], at.phase, 0x50u | at.slot);
            if (first) {
              ptx::bulk_wait<0>();
              arrive(&bars.empty[sent]);
              arrive(&written[(i - 1) % SLOTS]);
              sent = -1;
              first = false;
            }
            arrive(&bars.empty[at.slot]);
            at.next();
            q += kStage<T>;
          } while (q < p.q1);
        }
        uint32_t q = p.q0;
        do {
          w.wait(&stored[at.slot], at.phase, 0x40u | at.slot);
          const uint32_t n = min(kStage<T>, p.q1 - q);
          if (n) ptx::bulk_store(gq + q, ptx::smem_u32(ring + at.slot * kStage<T>), n * 16);
          ptx::bulk_commit();
          if (sent >= 0) {
            ptx::bulk_wait_read<1>();
            arrive(&bars.empty[sent]);
          }
          if (first) {
            ptx::bulk_wait<1>();  // the row before is in memory: its targets may be corrected
            arrive(&written[(i - 1) % SLOTS]);
            first = false;
          }
          sent = int(at.slot);
          at.next();
          q += kStage<T>;
        } while (q < p.q1);
      }
      if (i) {
        ptx::bulk_wait<0>();
        arrive(&written[(i - 1) % SLOTS]);
      }
    }
    __syncwarp();
  } else {  // adders
    RingAt<T> at;
    uint32_t i = 0;
    for (uint64_t row = first_row; row < a.rows; row += step, ++i) {
      RingAt<T> start = at;
      const uint32_t turn = i % SLOTS, phase = (i / SLOTS) & 1u;
      const float* x = a.x + row * a.ld;
      const Part p = part_of(x, vocab, rank, shares);
      const int extra_at = extra_of(p);
      const float extra = extra_at >= 0 ? x[extra_at] : -INFINITY;
      RowStats r;
      if (PASS != DistillPass::Backward) {
        Stream<SUM> stream(c);
        uint32_t q = p.q0;
        do {
          float4 v[QUADS];
          take_stage<T>(p, q, ring, bars, at, w, v);
          stream.add(v, c);
          if (PASS == DistillPass::Step && keep) {
            if (SUM != Sum::Tempered) {
              // the exponentials take the logits' place: the gradient has only to scale them
              float4* to = ring + at.slot * kStage<T> + threadIdx.x;
#pragma unroll
              for (uint32_t j = 0; j < QUADS; ++j) to[j * T] = v[j];
              kept_at[at.slot][threadIdx.x] = stream.m;
            }
          } else if (BULK) {
            __syncwarp();
            if (lane == 0) arrive(&stored[at.slot]);
          } else {
            leave_stage<T>(bars, at);
          }
          at.next();
          q += kStage<T>;
        } while (q < p.q1);
        r = stream.result(c);
        add_one<SUM>(r, extra, c);
        r = block_merge<SUM, T>(r, c, merged[i & 1]);
      }
      // From here on the targets have been read, in every block of the cluster once its
      // statistics have arrived: the row may be overwritten.  The wait also says that the server
      // is done with the result of SLOTS rows ago.
      w.wait(&tfull[turn], phase, 0x32u);
      if (PASS == DistillPass::Backward) {
        r.m = targets[turn].saved[0];
        r.u = targets[turn].saved[1];
        r.s = targets[turn].saved[2];
      } else {
        if (shares > 1) {
          const uint32_t bar = ptx::smem_u32(&peers[i & 1]);
          if (threadIdx.x == 0) ptx::mbar_arrive_expect_tx(bar, shares * 16);
          if (threadIdx.x < shares)
            ptx::st_async(ptx::mapa_shared(ptx::smem_u32(&parts[i & 1][rank]), threadIdx.x),
                          make_float4(r.m, r.s, r.u, 0.f), ptx::mapa_shared(bar, threadIdx.x));
          w.wait_cluster(&peers[i & 1], (i >> 1) & 1u, 0x33u);
          const float4 part = parts[i & 1][lane & (shares - 1)];
          r.m = part.x;
          r.s = part.y;
          r.u = part.z;
          rescale<SUM>(r, order_value(__reduce_max_sync(0xffffffffu, order_bits(r.m))), c);
          for (uint32_t o = shares / 2; o > 0; o >>= 1) {
            r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
            if (SUM != Sum::Plain) r.u += __shfl_xor_sync(0xffffffffu, r.u, o);
          }
        }
        complete<SUM>(r);
      }
      if (threadIdx.x == 0) {
        result[turn] = r;
        arrive(&done[turn]);
      }
      if (PASS != DistillPass::Forward) {
        const GradFactors f = grad_factors<SUM>(a, r, targets[turn], c);
        float* g = a.grad + row * a.ld_grad;
        if (extra_at >= 0) g[extra_at] = grad_at<SUM>(f, extra, c);
        // the same distance to a 16-byte boundary in both rows: 16-byte stores
        const bool vec = ((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(x)) & 15u) == 0;
        float4* gq = reinterpret_cast<float4*>(g + p.lead);
        uint32_t q = p.q0;
        do {
          float4 v[QUADS];
          const bool kept = PASS == DistillPass::Step && keep;
          RingAt<T>& now_at = kept ? start : at;
          if (kept) {
            read_stage<T>(p, q, ring + start.slot * kStage<T>, v);
            if (SUM == Sum::Tempered) grad_stage<SUM>(f, v, c);
            else scale_stage<SUM>(f, v, kept_at[start.slot][threadIdx.x], c);
          } else {
            take_stage<T>(p, q, ring, bars, at, w, v);
            grad_stage<SUM>(f, v, c);
          }
          if (BULK) {
            float4* to = ring + now_at.slot * kStage<T> + threadIdx.x;
#pragma unroll
            for (uint32_t j = 0; j < QUADS; ++j) to[j * T] = v[j];
          }
          // what was written here comes before the copy that sends the stage off, or fills it
          if (BULK || (kept && SUM != Sum::Tempered)) ptx::fence_proxy_async_smem();
          if (BULK) {
            __syncwarp();
            if (lane == 0) arrive(&stored[now_at.slot]);
          }
          if (BULK) {
            // sent by the storing warp
          } else if (vec && q + kStage<T> <= p.q1) {
#pragma unroll
            for (uint32_t j = 0; j < QUADS; ++j) __stcs(gq + q + threadIdx.x + j * T, v[j]);
          } else {
#pragma unroll
            for (uint32_t j = 0; j < QUADS; ++j) {
              const uint32_t piece = q + j * T + threadIdx.x;
              if (piece < p.q1) {
                const float4 o = v[j];
                if (vec) {
                  __stcs(gq + piece, o);
                } else {
                  float* out = g + p.lead + uint64_t(piece) * 4;
                  out[0] = o.x;
                  out[1] = o.y;
                  out[2] = o.z;
                  out[3] = o.w;
                }
              }
            }
          }
          if (!BULK) leave_stage<T>(bars, now_at);  // after the stores, which wait for what was read
          now_at.next();
          q += kStage<T>;
        } while (q < p.q1);
      }
      __syncwarp();
      if (lane == 0) {
        if (PASS != DistillPass::Forward && !BULK) arrive(&written[turn]);
        arrive(&tempty[turn]);
      }
    }
  }
  __syncthreads();
  if (shares > 1) ptx::cluster_sync_all();  // no block leaves while another may still write to it
  wait_out(&abort_word);
}

// Short rows, one warp each.
template <DistillPass PASS, Sum SUM, int PER>
__global__ void __launch_bounds__(ROWS_BLOCK) distill_warp_kernel(const DistillArgs a) {
  ptx::grid_dependency_release();  // programmatic dependent launch: see launch.cuh
  ptx::grid_dependency_wait();
  __shared__ Targets targets[ROWS_BLOCK / 32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, vocab = uint32_t(a.vocab);
  const uint64_t row = uint64_t(blockIdx.x) * (ROWS_BLOCK / 32) + warp;
  if (row >= a.rows) return;
  const float* x = a.x + row * a.ld;
  const float c = kLog2e / a.temperature;
  float v[PER];
  load_row<PER>(x, vocab, lane, v);
  RowStats r;
  if (PASS == DistillPass::Backward) {
    r = saved_stats(a, row);
  } else {
    r = stats_of<SUM, PER>(v, c);
    complete<SUM>(r);
  }
  read_targets<PASS != DistillPass::Backward>(a, row, x, true, targets[warp]);
  if (PASS != DistillPass::Backward) {
    const float loss = row_loss(a, r, targets[warp]);
    if (lane == 0) {
      a.loss[row] = loss;
      if (PASS == DistillPass::Forward && a.stats) save_stats(a, row, r);
    }
  }
  if (PASS != DistillPass::Forward) {
    const GradFactors f = grad_factors<SUM>(a, r, targets[warp], c);
    float* g = a.grad + row * a.ld_grad;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t i = uint32_t(j) * 32u + lane;
      if (i < vocab) g[i] = grad_at<SUM>(f, v[j], c);
    }
    __syncwarp();
    take_targets(a, g, targets[warp], f, 0, vocab);
  }
}

// ---- host side -----------------------------------------------------------------------------
// Blocks per row: few rows are shared so that the GPU is full, each block with at least 4096 logits.
uint32_t shares_for(uint64_t rows, uint64_t vocab, int sm_count) {
  uint32_t n = 1;
  while (n < MAX_SHARE && rows * n * 2 <= uint64_t(sm_count) * 2 && vocab / (n * 2) >= 4096) n *= 2;
  return n;
}
uint32_t rows_grid(uint64_t rows) { return uint32_t((rows + ROWS_BLOCK / 32 - 1) / (ROWS_BLOCK / 32)); }

// A ring kernel's clusters of `shares` blocks each take every so-many-th row.  As many as run at
// once: a cluster lies within one GPC, so that is fewer than the SMs would hold, and one more would
// start when the first are done (the step over 1024 x 128000 took 479 us with 37 clusters of 4 on
// 148 SMs, 263 us with those that fit).
template <auto KERN, int T, int THREADS = T + 64>
cudaError_t launch_ring(uint64_t rows, uint32_t shares, cudaStream_t stream, auto... args) {
  constexpr size_t smem = size_t(kStages<T>) * kStage<T> * 16;
  static int fit[64][MAX_SHARE + 1] = {};  // per kernel and device: clusters that run at once
  int dev = 0;
  cudaGetDevice(&dev);
  int& at_once = fit[dev & 63][shares];
  if (!at_once) {
    cudaError_t e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(shares);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = shares;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, KERN, &cfg);
    if (e != cudaSuccess) return e;
    if (n < 1) return cudaErrorInvalidConfiguration;
    at_once = n;
  }
  const uint64_t clusters = std::min<uint64_t>(rows, at_once);
  return launch_kernel_cluster(KERN, shares, dim3(uint32_t(clusters) * shares), dim3(THREADS), smem, stream, args...);
}

// The step over long rows with T adding threads a block.  What is read twice should come from L2 the
// second time, so the rows in flight are kept below kInFlight by giving a row to more blocks
// (4096 x 128000, one block a row and 76 MB in flight: 940 us; two and 38 MB: 683; four and 19 MB:
// 801, since each row costs a block some 3000 clocks besides its logits).
constexpr uint64_t kInFlight = 48ull << 20;
template <Sum SUM, int T>
cudaError_t launch_step(const DistillArgs& a, int sm_count, cudaStream_t stream) {
  constexpr DistillPass PASS = DistillPass::Step;
  uint32_t shares = shares_for(a.rows, a.vocab, sm_count);
  auto in_flight = [&] {
    return std::min<uint64_t>(a.rows, uint64_t(sm_count) * kRingBlocks<PASS, T> / shares) * a.vocab * 4;
  };
  while (shares < MAX_SHARE && in_flight() > kInFlight) shares *= 2;
  // a part that leaves the next row's loads two stages of the ring is kept there
  const bool keep = a.vocab / 4 / shares + 1 <= (kStages<T> - 2) * kStage<T>;
  // bulk stores need the rows of both matrices at the same distance from a 16-byte boundary
  const bool bulk = ((reinterpret_cast<uintptr_t>(a.grad) ^ reinterpret_cast<uintptr_t>(a.x)) & 15u) == 0 &&
                    (a.ld_grad - a.ld) % 4 == 0;
  constexpr int THREADS = kRingThreads<PASS, T>;
  return bulk ? launch_ring<distill_ring_kernel<PASS, SUM, true, T>, T, THREADS>(a.rows, shares, stream, a, shares, keep)
              : launch_ring<distill_ring_kernel<PASS, SUM, false, T>, T, THREADS>(a.rows, shares, stream, a, shares, keep);
}

template <DistillPass PASS, Sum SUM>
cudaError_t launch_distill_sum(const DistillArgs& a, int sm_count, cudaStream_t stream) {
  if (a.vocab <= WARP_ROW) {
    auto kern = a.vocab <= 32    ? distill_warp_kernel<PASS, SUM, 1>
                : a.vocab <= 128 ? distill_warp_kernel<PASS, SUM, 4>
                : a.vocab <= 512 ? distill_warp_kernel<PASS, SUM, 16>
                                 : distill_warp_kernel<PASS, SUM, 32>;
    return launch_kernel(kern, dim3(rows_grid(a.rows)), dim3(ROWS_BLOCK), 0, stream, a);
  }
  if constexpr (PASS == DistillPass::Step) {
    // Two narrow blocks an SM hide each other's waits between rows, a wide one has more of them in
    // flight: 2000 x 8000 41 and 55 us, x 12000 53 and 64, x 16000 68 and 66, x 24000 88 and 82.
    return a.vocab <= 3 * 4 * kStage<BLOCK> ? launch_step<SUM, BLOCK>(a, sm_count, stream)
                                            : launch_step<SUM, WIDE>(a, sm_count, stream);
  } else {
    const uint32_t shares = shares_for(a.rows, a.vocab, sm_count);
    return launch_ring<distill_ring_kernel<PASS, SUM, false, BLOCK>, BLOCK, kRingThreads<PASS, BLOCK>>(
        a.rows, shares, stream, a, shares, false);
  }
}

template <DistillPass PASS>
cudaError_t launch_distill_pass(const DistillArgs& given, int sm_count, cudaStream_t stream) {
  DistillArgs a = given;
  const bool soft = a.soft_weight > 0.f, hard = a.soft_weight < 1.f;
  // the saved statistics hold both sums
  const bool both = (soft && hard) || (PASS == DistillPass::Forward && a.stats);
  if (both && a.temperature == 2.f) return launch_distill_sum<PASS, Sum::Tempered2>(a, sm_count, stream);
  if (both && a.temperature == 4.f) return launch_distill_sum<PASS, Sum::Tempered4>(a, sm_count, stream);
  if (both && a.temperature != 1.f) return launch_distill_sum<PASS, Sum::Tempered>(a, sm_count, stream);
  if (!soft && !both) a.temperature = 1.f;  // a loss of the labels alone has no temperature
  return launch_distill_sum<PASS, Sum::Plain>(a, sm_count, stream);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, int sm_count, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  if (a.vocab <= WARP_ROW) {
    auto kern = a.vocab <= 32    ? logprobs_warp_kernel<1>
                : a.vocab <= 128 ? logprobs_warp_kernel<4>
                : a.vocab <= 512 ? logprobs_warp_kernel<16>
                                 : logprobs_warp_kernel<32>;
    return launch_kernel(kern, dim3(rows_grid(a.rows)), dim3(ROWS_BLOCK), 0, stream, a);
  }
  const uint32_t shares = shares_for(a.rows, a.vocab, sm_count);
  return a.top_n ? launch_ring<logprobs_ring_kernel<true>, BLOCK>(a.rows, shares, stream, a, shares)
                 : launch_ring<logprobs_ring_kernel<false>, BLOCK>(a.rows, shares, stream, a, shares);
}

cudaError_t launch_distill(DistillPass pass, const DistillArgs& a, int sm_count, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  switch (pass) {
    case DistillPass::Forward: return launch_distill_pass<DistillPass::Forward>(a, sm_count, stream);
    case DistillPass::Backward: return launch_distill_pass<DistillPass::Backward>(a, sm_count, stream);
    default: return launch_distill_pass<DistillPass::Step>(a, sm_count, stream);
  }
}

}  // namespace gonn
