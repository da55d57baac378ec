// Logit adjustments and the choice of the next token.
//
// A row of V logits is read once, by one CTA when the rows alone fill the
// GPU, by several when they do not (a cluster of up to 8 where their results
// have to meet).  What bounds it is the read (and write) of the logits for
// many rows, and the chain launch - load - combine for few; so a thread works
// on its own from the first load to the last, in runs of 8 logits with two
// more in flight, and the CTA meets at the end.
//
//   * The history of a row marks its tokens in a bitmap in shared memory and
//     counts them in 16-bit counters (32-bit ones for more than 65,535
//     tokens) beside it.  A counter is cleared by the token that marks it, so
//     nothing of the vocabulary's size is swept but the bitmap, and a logit
//     that was never seen, nearly every one, costs one bit.
//   * Rows of an odd length start anywhere.  A row is therefore counted from
//     the 16-byte boundary at or before its start: place q of a row is its
//     logit q - shift, shift < 8, so that every run but the first and the
//     last is one or two vector loads, in all rows (256 x 50,277 bf16 adjusted
//     in 14 us, 41 element by element).  Draws count from the logit itself,
//     whose index the generator's blocks go by, and load odd rows element by
//     element.  Where every row starts on a boundary all that is left out
//     (greedy, 256 x 50,280 bf16: 12 against 14 us).
//   * Penalties, bias and mask are applied in fp32 operation by operation (no
//     contraction), so the adjusted logit is that of the written formula.
//   * Largest logit and sum of exponentials are kept per thread, the sum
//     relative to the thread's largest, and joined in a fixed order.  Of the
//     largest logit a thread remembers the run it was in; its index is looked
//     up at the end, by the threads that hold the row's largest.
//   * A draw takes the largest z / T - log(-log u).  Since e = -log u >= v =
//     1 - u, z / T - log v bounds it from above, with v from the generator's
//     upper 23 bits and in units of log 2: a multiply-add and a hardware
//     logarithm.  A thread keeps the run with its highest bound and the second
//     highest; at the end the CTA's highest gives a score that is reached, and
//     the few logits whose bound is not below it are scored and compared in
//     64 bits.
#include <cuda_bf16.h>
#include <float.h>
#include <limits.h>
#include <math_constants.h>
#include <stddef.h>
#include <stdint.h>

#include "m3_kernels.cuh"
#include "m3_lm.cuh"

namespace m3 {

namespace {

constexpr int kVec = 8;       // consecutive logits of a thread
constexpr int kRuns = 2;      // such runs a thread loads at a time
constexpr int kTokens = 4;    // tokens of the history a thread holds
// Threads of a CTA, two CTAs an SM: draws want the registers of fewer threads
// (256 rows of bf16 44 against 50 us), the others the loads of more.
template <int MODE>
constexpr int logit_threads() { return MODE == 2 ? 384 : 512; }
constexpr int kWindow = 51200;   // logits whose 16-bit counters a CTA holds: two CTAs per SM
constexpr int kCountMax = 65535;
constexpr float kLog2e = 1.4426950408889634f;

enum { kProcess = 0, kGreedy = 1, kDraw = 2 };

struct LogitsParams {
  m3_logits_args a;
  int slices;  // CTAs of a row
  int slice;   // places of a CTA, a multiple of 32
  int window;  // places of a CTA at a time, a multiple of 32
  int history, wide;  // counters are needed; of 32 bits
};

__device__ __forceinline__ void logits_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t logits_peer(const void *smem, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(a)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t peer_load(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int64_t load_int(const void *p, int64_t i, int i64) {
  return i64 ? static_cast<const int64_t *>(p)[i] : (int64_t)static_cast<const int32_t *>(p)[i];
}

// Block i / 4 of the row's generator: four words.
struct RowNoise {
  uint32_t k0, k1, c1, c2;
  __device__ __forceinline__ uint4 block(uint32_t i) const {
    constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u, kW0 = 0x9E3779B9u, kW1 = 0xBB67AE85u;
    uint4 c = make_uint4(i, c1, c2, 0u);
#pragma unroll
    for (int r = 0; r < 7; ++r) {
      uint32_t ah, al, bh, bl;
      asm("{\n\t.reg .u64 t;\n\tmul.wide.u32 t, %2, %3;\n\tmov.b64 {%0, %1}, t;\n\t}" : "=r"(al), "=r"(ah) : "r"(c.x), "r"(kM0));
      asm("{\n\t.reg .u64 t;\n\tmul.wide.u32 t, %2, %3;\n\tmov.b64 {%0, %1}, t;\n\t}" : "=r"(bl), "=r"(bh) : "r"(c.z), "r"(kM1));
      c = make_uint4(bh ^ c.y ^ (k0 + r * kW0), bl, ah ^ c.w ^ (k1 + r * kW1), al);
    }
    return c;
  }
};

__device__ __forceinline__ uint32_t pick(const uint4 &c, int i) { return i == 0 ? c.x : i == 1 ? c.y : i == 2 ? c.z : c.w; }

// log2 of a lower bound of (w + 1/2) 2^-32, its truncation to 23 bits
__device__ __forceinline__ float noise_log2(uint32_t w) {
  return log2_approx(__uint_as_float(w >> 9 | 0x3f800000u) - 1.f);
}

__device__ __noinline__ double draw_noise(uint32_t w) { return -log(-log1p(-((double)w + 0.5) * 0x1p-32)); }

// An element of a row with its noise; id INT_MAX: none.
struct Drawn {
  double g;
  float z;
  int id;
};

// Whether a beats b: by the difference of the two, in 64 bits, so that large
// logits do not swallow the noise, and times the temperature, which is above
// 0 (a product where a quotient of 64 bits takes ten times as long).  Of two
// infinite ones b stays.
__device__ __forceinline__ bool draw_beats(const Drawn &a, const Drawn &b, float temperature) {
  if (b.id == INT_MAX) return a.id != INT_MAX;
  if (a.id == INT_MAX) return false;
  const double d = fma(a.g - b.g, (double)temperature, (double)a.z - (double)b.z);
  return d > 0.0 || (d == 0.0 && a.id < b.id);
}

// A sum of exponentials relative to `from`, relative to `to` (at least as
// large); equal ones, also infinite ones, leave it.
__device__ __forceinline__ float rebase(float sum, float from, float to, float scale) {
  return from == to ? sum : sum * exp2_approx((from - to) * scale);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFullMask, v, o));
  return v;
}
__device__ __forceinline__ Drawn warp_best(Drawn b, float temperature) {
  if (!__any_sync(kFullMask, b.id != INT_MAX)) return b;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Drawn c = {__shfl_xor_sync(kFullMask, b.g, o), __shfl_xor_sync(kFullMask, b.z, o),
                     __shfl_xor_sync(kFullMask, b.id, o)};
    if (draw_beats(c, b, temperature)) b = c;
  }
  return b;
}

// How far below a score a bound may be computed of an element that reaches
// it: the hardware logarithm and the product with the scale, which is at
// most about 33 larger than the score.
__device__ __forceinline__ float slack(float score) { return 1e-3f + 2e-6f * fabsf(score); }

struct Choice {  // of a CTA, read by the cluster's first
  float top, sum;
  uint32_t noise_hi, noise_lo;
  float z;
  int id;      // or INT_MAX
  int nan_id;  // first NaN, or INT_MAX
};

// A run as it lies in memory: elements [from, n) of it are the row's, the
// others -infinity.  vec: whole runs start on 16 bytes.
template <typename T>
struct Run {
  static constexpr int kWords = sizeof(T) * kVec / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const char *at, int from, int n, bool vec) {
    if (vec && from <= 0 && n >= kVec) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 q = reinterpret_cast<const uint4 *>(at)[i];
        w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
      }
    } else if (sizeof(T) == 2) {
      const uint16_t *h = reinterpret_cast<const uint16_t *>(at);
      auto get = [&](int i) -> uint32_t { return i >= from && i < n ? h[i] : 0xff80u; };
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = get(2 * i) | get(2 * i + 1) << 16;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        w[i] = i >= from && i < n ? reinterpret_cast<const uint32_t *>(at)[i] : 0xff800000u;
    }
  }
  __device__ __forceinline__ void get(float (&z)[kVec]) const {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      z[i] = __uint_as_float(sizeof(T) == 2 ? (i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16) : w[i % kWords]);
  }
};

// elements [from, n) of a run to `row` + place q
__device__ __forceinline__ void store_run(const float (&z)[kVec], char *row, int bf16, int q, int from, int n,
                                          bool vec) {
  if (!vec || n < kVec || from > 0) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (i >= from && i < n) st_any(row, q + i, z[i], bf16 ? M3_BF16 : M3_F32);
  } else if (bf16) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(z[2 * i], z[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&v);
    }
    *reinterpret_cast<uint4 *>(row + (int64_t)q * 2) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    float4 *p = reinterpret_cast<float4 *>(row + (int64_t)q * 4);
    p[0] = make_float4(z[0], z[1], z[2], z[3]);
    p[1] = make_float4(z[4], z[5], z[6], z[7]);
  }
}

// What a CTA needs to adjust its logits.  Offsets o are in the window, places
// q in the row.
struct Row {
  const float *bias;       // of place 0
  const uint32_t *seen;    // the window's bitmap, or NULL without a history
  const uint32_t *counts;  // its counters
  float rep, pres, freq;
  int wide;
  bool vec_bias;

  __device__ __forceinline__ uint32_t count(int o) const {
    return wide ? counts[o] : counts[o >> 1] >> ((o & 1) * 16) & 0xffffu;
  }
  // which of the run at o have been seen
  __device__ __forceinline__ uint32_t hits(int o) const { return seen ? seen[o >> 5] >> (o & 31) & 0xffu : 0u; }
  __device__ __forceinline__ float penalized(float v, int o) const {
    v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    const uint32_t c = count(o);
    return c ? __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)c)), pres) : v;
  }
  __device__ __forceinline__ void penalize(float (&z)[kVec], int o, uint32_t hit) const {
    while (hit) {
      const int at = __ffs(hit) - 1;
      hit &= hit - 1;
      float v = z[0];
#pragma unroll
      for (int i = 1; i < kVec; ++i) v = i == at ? z[i] : v;
      v = penalized(v, o + at);
#pragma unroll
      for (int i = 0; i < kVec; ++i) z[i] = i == at ? v : z[i];
    }
  }
  // bias and mask of elements [from, n) of the run at place q; ok: its bits of the mask
  __device__ __forceinline__ void finish(float (&z)[kVec], int q, int from, int n, uint32_t ok) const {
    if (bias) {
      if (vec_bias && n >= kVec && from <= 0) {
        const float4 b0 = reinterpret_cast<const float4 *>(bias + q)[0];
        const float4 b1 = reinterpret_cast<const float4 *>(bias + q)[1];
        z[0] += b0.x, z[1] += b0.y, z[2] += b0.z, z[3] += b0.w;
        z[4] += b1.x, z[5] += b1.y, z[6] += b1.z, z[7] += b1.w;
      } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          if (i >= from && i < n) z[i] += bias[q + i];
      }
    }
    if (ok != 0xffu) {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (!(ok >> i & 1u)) z[i] = -CUDART_INF_F;
    }
  }
};

// Marks and counts the history's tokens in the n logits from e0; held: the
// first kTokens of every thread, read already (INT_MIN: not in the vocabulary).
// The bitmap is clear.
__device__ __forceinline__ void mark_history(const LogitsParams &p, int row, int len, int prompt, int e0, int n,
                                             const int (&held)[kTokens], uint32_t *seen, uint32_t *counts) {
  const m3_logits_args &a = p.a;
  const int tid = threadIdx.x, nt = blockDim.x;
  const int64_t at = (int64_t)row * a.tokens_stride;
  auto token = [&](int64_t i) -> int64_t {  // outside the vocabulary: outside every window
    const int64_t t = load_int(a.tokens, at + i, a.tokens_i64);
    return t >= 0 && t < a.V ? t : INT_MIN;
  };
  auto mark = [&](int64_t o) {
    if (o < 0 || o >= n) return;
    if (p.wide)
      counts[o] = 0u;
    else
      reinterpret_cast<uint16_t *>(counts)[o] = 0;
    atomicOr(&seen[o >> 5], 1u << (o & 31));
  };
  auto count = [&](int64_t o) {
    if (o < 0 || o >= n) return;
    if (p.wide)
      atomicAdd(&counts[o], 1u);
    else
      atomicAdd(&counts[o >> 1], 1u << ((o & 1) * 16));
  };
#pragma unroll
  for (int k = 0; k < kTokens; ++k)
    if (tid + k * nt < len) mark((int64_t)held[k] - e0);
  for (int64_t i = tid + (int64_t)kTokens * nt; i < len; i += nt)
    mark(token(i) - e0);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kTokens; ++k)
    if (tid + k * nt < len && tid + k * nt >= prompt) count((int64_t)held[k] - e0);
  for (int64_t i = tid + (int64_t)kTokens * nt; i < len; i += nt)
    if (i >= prompt) count(token(i) - e0);
  __syncthreads();
}

// ALIGNED: every row of logits starts on 16 bytes.
template <typename T, int MODE, bool ALIGNED>
__global__ void __launch_bounds__(logit_threads<MODE>(), 2) logits_kernel(const LogitsParams p) {
  constexpr int kLogitWarps = logit_threads<MODE>() / 32;
  extern __shared__ __align__(16) uint32_t table[];  // bitmap and counters of a window
  __shared__ float warp_f[kLogitWarps], warp_b[kLogitWarps];
  __shared__ Drawn warp_d[kLogitWarps];
  __shared__ int first[2];   // lowest index of the window's largest logit; of a NaN
  __shared__ float reached;  // a score some element of the window reaches, in units of log 2
  __shared__ Choice mine;
  const m3_logits_args &a = p.a;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.slices, rank = blockIdx.x % p.slices;
  const char *logits = static_cast<const char *>(a.logits) + (int64_t)row * a.ld * sizeof(T);
  // places of the row: logit e is place e + shift; from here on, row pointers are place 0's
  const int shift = ALIGNED || MODE == kDraw ? 0 : (int)((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
  const int end = a.V + shift;
  logits -= shift * (int)sizeof(T);
  const bool vec_in = ALIGNED || (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
  const int64_t begin = (int64_t)rank * p.slice;
  const int lo = (int)min(begin, (int64_t)end), hi = (int)min(begin + p.slice, (int64_t)end);
  if (MODE != kProcess && tid == 0) first[0] = first[1] = INT_MAX;
  auto clear = [&] {
    for (int i = tid; i < p.window / 32; i += nt) table[i] = 0u;
  };
  if (p.history) clear();  // while the preceding kernel runs

  pdl_wait();
  pdl_trigger();
  char *out = nullptr;
  bool vec_out = false;
  if (MODE == kProcess) {
    const int size = a.out_dtype == M3_BF16 ? 2 : 4;
    out = static_cast<char *>(a.out) + ((int64_t)row * a.out_ld - shift) * size;
    vec_out = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  }
  const int32_t *allowed = a.allowed ? a.allowed + (int64_t)row * a.allowed_stride : nullptr;
  Row r = {};
  int len = 0, prompt = 0, held[kTokens];
  if (p.history) {
    // the tokens first, whatever the length turns out to be
    const int64_t at = (int64_t)row * a.tokens_stride;
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      const int i = tid + k * nt;
      const int64_t t = i < a.T ? load_int(a.tokens, at + i, a.tokens_i64) : -1;
      held[k] = t >= 0 && t < a.V ? (int)t : INT_MIN;
    }
    r.rep = a.repetition ? a.repetition[row] : a.repetition_value;
    r.pres = a.presence ? a.presence[row] : a.presence_value;
    r.freq = a.frequency ? a.frequency[row] : a.frequency_value;
    const int64_t n = a.lengths ? load_int(a.lengths, row, a.lengths_i64) : a.T;
    const int64_t m = a.prompt_lengths ? load_int(a.prompt_lengths, row, a.prompt_i64) : 0;
    len = (int)min(max(n, (int64_t)0), (int64_t)a.T);
    prompt = (int)min(max(m, (int64_t)0), (int64_t)len);
    if (len > 0) r.seen = table, r.counts = table + p.window / 32;
  }
  r.bias = a.bias ? a.bias + (int64_t)row * a.bias_stride - shift : nullptr;
  r.wide = p.wide, r.vec_bias = (reinterpret_cast<uintptr_t>(r.bias) & 15) == 0;
  float temp = 1.f;
  bool drawn = false;
  RowNoise noise = {};
  if (MODE == kDraw) {
    const float t = a.temperature ? a.temperature[row] : a.temperature_value;
    drawn = t > 0.f;
    if (drawn) temp = t;
    const uint64_t seed = (uint64_t)a.seeds[row], pos = a.positions ? (uint64_t)a.positions[row] : 0;
    noise.k0 = (uint32_t)seed, noise.k1 = (uint32_t)(seed >> 32);
    noise.c1 = (uint32_t)pos, noise.c2 = (uint32_t)(pos >> 32);
  }
  // exponents are taken to base 2; kept finite and above 0, so that -infinity stays it
  const float scale = fmaxf(fminf(kLog2e / temp, FLT_MAX), FLT_MIN);
  auto bound = [&](float v, uint32_t w) { return fmaf(v, scale, -noise_log2(w)); };
  __syncthreads();  // `first` stands, the bitmap is clear

  // A run and the mask's words it lies in, as they are in memory: nothing is
  // computed from them here, so that the loads wait for none before them.
  struct Held {
    Run<T> run;
    uint32_t m0, m1;
  };
  auto fetch = [&](Held &h, int q, int n) {
    if (n <= 0) return;
    h.run.load(logits + (int64_t)q * sizeof(T), ALIGNED || MODE == kDraw ? 0 : shift - q, n, vec_in);
    if (allowed) {
      const int e = q - shift;
      h.m0 = (uint32_t)allowed[max(e, 0) >> 5];
      if (shift) h.m1 = (uint32_t)allowed[min(e + kVec - 1, a.V - 1) >> 5];
    }
  };
  // the first element of the run at place q that is the row's
  auto from = [&](int q) { return ALIGNED || MODE == kDraw ? 0 : shift - q; };
  // the mask's bits of the run at place q
  auto bits = [&](const Held &h, int q) -> uint32_t {
    if (!allowed) return 0xffu;
    const int e = q - shift;  // before the row's first logit in its first run
    return (e < 0 ? h.m0 << -e : shift ? __funnelshift_r(h.m0, h.m1, e & 31) : h.m0 >> (e & 31)) & 0xffu;
  };
  // z, the run at place q (window offset o), adjusted
  auto adjust = [&](float (&z)[kVec], uint32_t ok, int q, int o, int n) {
    r.penalize(z, o, r.hits(o));
    r.finish(z, q, from(q), n, ok);
  };
  auto look_at = [&](float (&z)[kVec], int w0, int wn, int o) {
    Held h;
    fetch(h, w0 + o, wn - o);
    h.run.get(z);
    adjust(z, bits(h, w0 + o), w0 + o, o, wn - o);
  };

  const int step = nt * kVec;
  float top = -CUDART_INF_F, sum = 0.f;  // the CTA's largest logit of the windows done; this thread's sum relative to it
  Drawn best = {0.0, 0.f, INT_MAX};      // this thread's best drawn element
  int id = INT_MAX, nan_id = INT_MAX;
  for (int w0 = lo; w0 < hi; w0 += p.window) {
    const int wn = min(p.window, hi - w0);
    Held next[kRuns];
#pragma unroll
    for (int u = 0; u < kRuns; ++u) fetch(next[u], w0 + tid * kVec + u * step, wn - tid * kVec - u * step);
    if (r.seen) {
      if (w0 > lo) {
        __syncthreads();  // the table has been read
        clear();
        __syncthreads();
      }
      mark_history(p, row, len, prompt, w0 - shift, wn, held, table, table + p.window / 32);
    }
    float high = -CUDART_INF_F, mass = 0.f;  // this thread's largest of the window, the sum relative to it
    int high_at = 0;                         // the run it is in
    if (MODE == kDraw && tid == 0) reached = -CUDART_INF_F;
    float most = -CUDART_INF_F, second = -CUDART_INF_F;  // highest bounds of its runs
    int most_at = -1;
    // of bounds past fp32's range too the last run is kept
    auto raise = [&](float b, int o) {
      if (b >= most)
        second = most, most = b, most_at = o;
      else
        second = fmaxf(second, b);
    };
    for (int o0 = tid * kVec; o0 < wn; o0 += kRuns * step) {
#pragma unroll
      for (int u = 0; u < kRuns; ++u) {
        const int o = o0 + u * step, n = wn - o;
        if (n <= 0) continue;
        float z[kVec];
        next[u].run.get(z);
        const uint32_t ok = bits(next[u], w0 + o);
        fetch(next[u], w0 + o + kRuns * step, n - kRuns * step);
        adjust(z, ok, w0 + o, o, n);
        if (MODE == kProcess) {
          store_run(z, out, a.out_dtype == M3_BF16, w0 + o, from(w0 + o), n, vec_out);
          continue;
        }
        float m = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < kVec; ++i) m = fmaxf(m, z[i]);
        if (m > high) mass = rebase(mass, high, m, scale), high = m, high_at = o;
        // nothing but NaN and -infinity so far: relative to 0, where a NaN shows
        const float ref = high == -CUDART_INF_F ? 0.f : high;
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kVec; ++i) part[i & 1] += exp2_approx((z[i] - ref) * scale);
        mass += part[0] + part[1];
        if (MODE == kDraw && drawn && m > -CUDART_INF_F) {  // a run that the mask leaves empty draws nothing
          float b = -CUDART_INF_F;
#pragma unroll
          for (int h = 0; h < kVec / 4; ++h) {
            const uint4 w = noise.block(((uint32_t)(w0 + o) >> 2) + h);
#pragma unroll
            for (int i = 0; i < 4; ++i) b = fmaxf(b, bound(z[4 * h + i], pick(w, i)));
          }
          raise(b, o);
        }
      }
    }
    if (MODE == kProcess) continue;

    // the CTA's largest of the window, its index, and the first NaN
    const float warp_high = warp_max(high), warp_most = MODE == kDraw ? warp_max(most) : 0.f;
    if (lane == 0) warp_f[warp] = warp_high, warp_b[warp] = warp_most;
    const int bad = __syncthreads_or(mass != mass);
    float cta = warp_f[0];
    for (int w = 1; w < nt >> 5; ++w) cta = fmaxf(cta, warp_f[w]);
    const bool look = cta > top && (!drawn || cta == CUDART_INF_F);
    if (look && high == cta) {
      float z[kVec];
      look_at(z, w0, wn, high_at);
      int at = INT_MAX;
#pragma unroll
      for (int i = kVec - 1; i >= 0; --i)
        if (z[i] == cta) at = w0 + high_at + i - shift;
      atomicMin(&first[0], at);
    }
    if (bad) {
      for (int o = tid * kVec; o < wn; o += step) {
        float z[kVec];
        look_at(z, w0, wn, o);
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          if (z[i] != z[i]) atomicMin(&first[1], w0 + o + i - shift);
      }
    }
    if (MODE == kDraw && drawn && cta > -CUDART_INF_F) {
      // scores the run's elements whose bound is not below `from`
      auto score = [&](int o, float from) {
        float z[kVec];
        look_at(z, w0, wn, o);
#pragma unroll 1
        for (int h = 0; h < kVec / 4; ++h) {
          const uint32_t e = (uint32_t)(w0 + o + 4 * h);
          const uint4 w = noise.block(e >> 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = h ? z[4 + i] : z[i];
            if (v > -CUDART_INF_F && !(bound(v, pick(w, i)) < from)) {
              const Drawn c = {draw_noise(pick(w, i)), v, (int)e + i};
              if (draw_beats(c, best, temp)) best = c;
            }
          }
        }
      };
      float cta_most = warp_b[0];
      for (int w = 1; w < nt >> 5; ++w) cta_most = fmaxf(cta_most, warp_b[w]);
      if (most_at >= 0 && most == cta_most) {
        // bounds and scores past fp32's range prune nothing: infinities compare as not below
        float z[kVec], low = -CUDART_INF_F;
        look_at(z, w0, wn, most_at);
#pragma unroll
        for (int h = 0; h < kVec / 4; ++h) {
          const uint4 w = noise.block(((uint32_t)(w0 + most_at) >> 2) + h);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (bound(z[4 * h + i], pick(w, i)) == most) {
              // e for v rounded up to the next of the 23 bits; at most 23
              const float v = __uint_as_float(pick(w, i) >> 9 | 0x3f800000u) - 1.f + 0x1p-23f;
              const float e = v < 1.f ? -log1pf(-v) : 23.f;
              low = fmaf(z[4 * h + i], scale, -log2_approx(e));
            }
        }
        reached = low;
      }
      __syncthreads();
      const float limit = reached - slack(reached);
      if (most_at >= 0 && !(most < limit)) score(most_at, limit);
      if (!(second < limit))
        for (int o = tid * kVec; o < wn; o += step)
          if (o != most_at) score(o, limit);
    }
    __syncthreads();
    if (look) id = first[0];
    nan_id = first[1];
    const float now = fmaxf(top, cta);
    sum = rebase(sum, top, now, scale) + rebase(mass, high, now, scale);
    top = now;
    if (w0 + p.window < hi) {
      __syncthreads();
      if (tid == 0) first[0] = INT_MAX;
      __syncthreads();
    }
  }
  if (MODE == kProcess) return;

  sum = group_sum<32>(sum);
  if (MODE == kDraw && drawn) best = warp_best(best, temp);
  if (lane == 0) {
    warp_f[warp] = sum;
    if (MODE == kDraw) warp_d[warp] = best;
  }
  __syncthreads();
  if (warp == 0) {
    const int nw = nt >> 5;
    sum = group_sum<32>(lane < nw ? warp_f[lane] : 0.f);
    Drawn c = {0.0, top, id};
    if (MODE == kDraw && drawn && top < CUDART_INF_F)
      c = warp_best(lane < nw ? warp_d[lane] : Drawn{0.0, 0.f, INT_MAX}, temp);
    if (p.slices > 1 && lane == 0) {
      const uint64_t bits = (uint64_t)__double_as_longlong(c.g);
      mine.top = top, mine.sum = sum, mine.noise_hi = (uint32_t)(bits >> 32), mine.noise_lo = (uint32_t)bits;
      mine.z = c.z, mine.id = c.id, mine.nan_id = nan_id;
    }
    best = c;
  }
  if (p.slices > 1) {
    logits_cluster_sync();  // every CTA's choice stands
    if (rank == 0 && warp == 0) {
      const bool in = lane < p.slices;
      const uint32_t at = logits_peer(&mine, in ? (uint32_t)lane : 0u);
      const float t = in ? __uint_as_float(peer_load(at + offsetof(Choice, top))) : -CUDART_INF_F;
      const float s = in ? __uint_as_float(peer_load(at + offsetof(Choice, sum))) : 0.f;
      const uint64_t bits = (uint64_t)peer_load(at + offsetof(Choice, noise_hi)) << 32 |
                            peer_load(at + offsetof(Choice, noise_lo));
      Drawn c = {__longlong_as_double((long long)bits), __uint_as_float(peer_load(at + offsetof(Choice, z))),
                 in ? (int)peer_load(at + offsetof(Choice, id)) : INT_MAX};
      nan_id = __reduce_min_sync(kFullMask, in ? (int)peer_load(at + offsetof(Choice, nan_id)) : INT_MAX);
      top = warp_max(t);
      sum = group_sum<32>(rebase(s, t, top, scale));
      // of two infinite logits neither beats the other by the difference: the lowest index
      if (top == CUDART_INF_F) {
        c.id = __reduce_min_sync(kFullMask, t == top ? c.id : INT_MAX);
        c.z = top;
        best = c;
      } else {
        best = warp_best(c, temp);
      }
    }
  }
  if (rank == 0 && tid == 0) {
    // NaN with an infinite logit, as the formula gives
    float lp = (best.z - top) / temp - logf(sum);
    int chosen = best.id;
    if (nan_id != INT_MAX)
      chosen = nan_id, lp = CUDART_NAN_F;
    else if (top == -CUDART_INF_F)
      chosen = 0, lp = -CUDART_INF_F;
    a.ids[row] = chosen;
    a.logprobs[row] = lp;
  }
  if (p.slices > 1) logits_cluster_sync();  // no CTA leaves while its choice is read
}

template <typename T, int MODE, bool ALIGNED>
cudaError_t launch_logits_t(const m3_logits_args &a, cudaStream_t stream) {
  LogitsParams p = {};
  p.a = a;
  p.history = a.tokens && a.T > 0 &&
              (a.repetition || a.presence || a.frequency || a.repetition_value != 1.f || a.presence_value != 0.f ||
               a.frequency_value != 0.f);
  p.wide = a.T > kCountMax;
  // CTAs of a row: what fills two CTAs an SM, at least one run a thread each;
  // those that have to meet are a cluster, a power of two up to 8
  constexpr int kLogitThreads = logit_threads<MODE>();
  const int fill = 2 * sm_count_current() / a.B;
  const int runs = (int)(((int64_t)a.V + kLogitThreads * kVec - 1) / (kLogitThreads * kVec));
  int want = max(1, min(fill, runs));
  if (MODE != kProcess) {
    p.slices = 1;
    while (p.slices < 8 && p.slices * 2 <= want) p.slices *= 2;
  } else {
    p.slices = want;
  }
  const int places = a.V + (ALIGNED || MODE == kDraw ? 0 : kVec - 1);  // wherever the rows start
  p.slice = ((places + p.slices - 1) / p.slices + 31) / 32 * 32;
  p.window = p.history ? min(p.slice, p.wide ? kWindow / 2 : kWindow) : p.slice;
  const int64_t grid = (int64_t)a.B * p.slices;
  if (grid > 0x7fffffff) return cudaErrorInvalidValue;
  const int threads = min(kLogitThreads, ((p.slice + kVec - 1) / kVec + 31) / 32 * 32);
  auto kern = logits_kernel<T, MODE, ALIGNED>;
  const size_t smem = p.history ? (size_t)p.window / 8 + (size_t)p.window * (p.wide ? 4 : 2) : 0;
  static LaunchCache cache;
  if (cudaError_t e = ensure_smem_optin(cache, kern, kWindow / 8 + kWindow * 2); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.slices;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = MODE != kProcess && p.slices > 1 ? 2 : 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p); e != cudaSuccess) return e;
  return cudaGetLastError();
}

template <typename T, int MODE>
cudaError_t launch_logits_a(const m3_logits_args &a, cudaStream_t stream) {
  const bool aligned = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (a.B == 1 || a.ld * sizeof(T) % 16 == 0);
  return aligned ? launch_logits_t<T, MODE, true>(a, stream) : launch_logits_t<T, MODE, false>(a, stream);
}

template <int MODE>
cudaError_t launch_logits(const m3_logits_args &a, cudaStream_t stream) {
  return a.dtype == M3_BF16 ? launch_logits_a<__nv_bfloat16, MODE>(a, stream) : launch_logits_a<float, MODE>(a, stream);
}

}  // namespace

cudaError_t launch_process_logits(const m3_logits_args &a, cudaStream_t stream) {
  return launch_logits<kProcess>(a, stream);
}

cudaError_t launch_next_tokens(const m3_logits_args &a, cudaStream_t stream) {
  return a.sample ? launch_logits<kDraw>(a, stream) : launch_logits<kGreedy>(a, stream);
}

}  // namespace m3
