// Logit adjustments and the choice of the next token.
//
// A row of V logits is read once: by a cluster of up to 8 CTAs that take a
// slice each, 32 elements a thread, in registers from the load to the store
// or the choice.  What bounds it is the read (and write) of the logits for
// many rows, and the chain launch - load - combine for few.
//
//   * The history of a row is read once too: the cluster's CTAs share it out,
//     and add every token into a counter of the CTA that holds its logit,
//     through distributed shared memory (integers: the order does not
//     matter).  A logit whose counter is 0, nearly every one, costs a share
//     of a 16-byte load and a test.
//   * Penalties, bias and mask are applied in fp32 operation by operation (no
//     contraction), so the adjusted logit is that of the written formula.
//   * Largest logit and sum of exponentials: per thread, CTA and cluster, the
//     sum relative to the CTA's largest logit, joined in rank order.
//   * A draw takes the largest z / T - log(-log u), that is the smallest
//     e / p with e = -log u and p = exp(z / T - largest).  Only few elements
//     can win, so all get a lower bound (e >= v = 1 - u, from the generator's
//     upper 23 bits, times 1 / p), a thread's smallest gives an upper bound
//     of the winner, and the elements below that (one or two a CTA) are
//     compared in 64 bits.
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

constexpr int kVec = 8;                       // consecutive elements of a thread
constexpr int kVecs = 4;                      // such runs a thread holds
constexpr int kPer = kVec * kVecs;
constexpr int kLogitThreads = 256;
constexpr int kSliceMax = kLogitThreads * kPer;  // logits of a CTA at a time
constexpr int kLogitWarps = kLogitThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;

enum { kProcess = 0, kChoose = 1 };

struct LogitsParams {
  m3_logits_args a;
  int slices;       // CTAs of a row: a cluster where they have to meet
  int slice;        // logits of a CTA in a round, a multiple of 32
  int rounds;
  int history;      // counters are needed
  int vec_in, vec_out, vec_bias;  // rows start on 16 bytes
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
__device__ __forceinline__ void peer_add(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void peer_or(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
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
      const uint64_t a = (uint64_t)c.x * kM0, b = (uint64_t)c.z * kM1;
      c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ (k0 + r * kW0), (uint32_t)b,
                     (uint32_t)(a >> 32) ^ c.w ^ (k1 + r * kW1), (uint32_t)a);
    }
    return c;
  }
  __device__ __forceinline__ uint32_t word(uint32_t i) const {
    const uint4 c = block(i >> 2);
    const uint32_t w = i & 3;
    return w == 0 ? c.x : w == 1 ? c.y : w == 2 ? c.z : c.w;
  }
};

// Truncation of (w + 1/2) 2^-32 to 23 bits: a lower bound, short by less than 2^-23.
__device__ __forceinline__ float noise_low(uint32_t w) { return __uint_as_float(w >> 9 | 0x3f800000u) - 1.f; }

__device__ __noinline__ double draw_noise(uint32_t w) { return -log(-log1p(-((double)w + 0.5) * 0x1p-32)); }

// Whether logit z with noise g beats `bz` with `bg` (token `bid`): by the
// difference of the two, in 64 bits, so that large logits do not swallow the
// noise.
__device__ __forceinline__ bool draw_beats(float z, double g, int id, float bz, double bg, int bid, float temperature) {
  if (bid == INT_MAX) return id != INT_MAX;
  if (id == INT_MAX) return false;
  const double d = ((double)z - (double)bz) / (double)temperature + (g - bg);
  return d > 0.0 || (d == 0.0 && id < bid);
}

struct Choice {  // of a CTA; 32-bit words for the peers
  float top, sum;       // largest logit and the sum of exponentials relative to it
  uint32_t noise_hi, noise_lo;  // of the best element, as a double
  int id;               // or INT_MAX
  float z;              // its adjusted logit
  int nan_id;           // first NaN, or INT_MAX
};

template <typename T>
__device__ __forceinline__ void load_run(float (&z)[kVec], const void *row, int e, int n, int vec) {
  const T *p = static_cast<const T *>(row) + e;
  if (vec && n == kVec) {
    if (sizeof(T) == 2) {
      const uint4 q = *reinterpret_cast<const uint4 *>(p);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        z[2 * i] = __uint_as_float(w[i] << 16);
        z[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
      const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
      z[0] = a.x, z[1] = a.y, z[2] = a.z, z[3] = a.w, z[4] = b.x, z[5] = b.y, z[6] = b.z, z[7] = b.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) z[i] = i < n ? (float)p[i] : -CUDART_INF_F;
}

__device__ __forceinline__ void store_run(const float (&z)[kVec], void *row, int bf16, int e, int n, int vec) {
  if (bf16) {
    __nv_bfloat16 *p = static_cast<__nv_bfloat16 *>(row) + e;
    if (vec && n == kVec) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(z[2 * i], z[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&v);
      }
      *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (i < n) p[i] = __float2bfloat16_rn(z[i]);
    }
  } else {
    float *p = static_cast<float *>(row) + e;
    if (vec && n == kVec) {
      reinterpret_cast<float4 *>(p)[0] = make_float4(z[0], z[1], z[2], z[3]);
      reinterpret_cast<float4 *>(p)[1] = make_float4(z[4], z[5], z[6], z[7]);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (i < n) p[i] = z[i];
    }
  }
}

// The CTA's smallest or largest v (NaN ignored), to every thread.
template <bool MAX>
__device__ __forceinline__ float cta_extreme(float v, float *scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float w = __shfl_xor_sync(kFullMask, v, o);
    v = MAX ? fmaxf(v, w) : fminf(v, w);
  }
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
  for (int w = 1; w < (int)blockDim.x >> 5; ++w) v = MAX ? fmaxf(v, scratch[w]) : fminf(v, scratch[w]);
  __syncthreads();  // the scratch may be written again
  return v;
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const LogitsParams p) {
  extern __shared__ __align__(16) uint32_t counters[];  // p.slice of them, with a history
  __shared__ float scratch[kLogitWarps];
  __shared__ int first[2];  // lowest index of the CTA's largest logit; of a NaN
  __shared__ double warp_noise[kLogitWarps];
  __shared__ int warp_id[kLogitWarps];
  __shared__ float warp_z[kLogitWarps];
  __shared__ Choice mine;
  const m3_logits_args &a = p.a;
  const int tid = threadIdx.x, nt = blockDim.x;
  const int row = blockIdx.x / p.slices, rank = blockIdx.x % p.slices;

  pdl_wait();
  pdl_trigger();
  const char *logits = static_cast<const char *>(a.logits) + (int64_t)row * a.ld * sizeof(T);
  const int32_t *allowed = a.allowed ? a.allowed + (int64_t)row * a.allowed_stride : nullptr;
  const float *bias = a.bias ? a.bias + (int64_t)row * a.bias_stride : nullptr;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  int len = 0, prompt = 0;
  if (p.history) {
    rep = a.repetition ? a.repetition[row] : a.repetition_value;
    pres = a.presence ? a.presence[row] : a.presence_value;
    freq = a.frequency ? a.frequency[row] : a.frequency_value;
    const int64_t n = a.lengths ? load_int(a.lengths, row, a.lengths_i64) : a.T;
    const int64_t m = a.prompt_lengths ? load_int(a.prompt_lengths, row, a.prompt_i64) : 0;
    len = (int)min(max(n, (int64_t)0), (int64_t)a.T);
    prompt = (int)min(max(m, (int64_t)0), (int64_t)len);
  }
  float temp = 1.f;
  bool drawn = false;
  RowNoise noise = {};
  if (MODE == kChoose && a.sample) {
    const float t = a.temperature ? a.temperature[row] : a.temperature_value;
    drawn = t > 0.f;
    if (drawn) temp = t;
    const uint64_t seed = (uint64_t)a.seeds[row], pos = a.positions ? (uint64_t)a.positions[row] : 0;
    noise.k0 = (uint32_t)seed, noise.k1 = (uint32_t)(seed >> 32);
    noise.c1 = (uint32_t)pos, noise.c2 = (uint32_t)(pos >> 32);
  }
  const float scale = fminf(kLog2e / temp, FLT_MAX);  // exponents are taken to base 2
  float top = -CUDART_INF_F, sum = 0.f;  // the CTA's largest logit so far, this thread's sum relative to it
  double best_g = 0.0;                   // this thread's best drawn element
  float best_z = 0.f;
  int best_id = INT_MAX, top_id = INT_MAX, nan_id = INT_MAX;

  const int window = p.slices * p.slice;
  for (int round = 0; round < p.rounds; ++round) {
    const int w0 = round * window, base = w0 + rank * p.slice;
    if (round > 0) __syncthreads();  // the counters have been read
    float z[kVecs][kVec];
    uint32_t ok[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int o = (u * nt + tid) * kVec, e = base + o;
      const int n = o < p.slice ? min(a.V - e, kVec) : 0;
      if (n > 0) {
        load_run<T>(z[u], logits, e, n, p.vec_in);
        ok[u] = allowed ? (uint32_t)allowed[e >> 5] >> (e & 31) : 0xffu;
      } else {
        ok[u] = 0u;
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[u][i] = -CUDART_INF_F;
      }
    }
    if (p.history) {
      for (int i = tid * 4; i < p.slice; i += nt * 4) *reinterpret_cast<uint4 *>(counters + i) = make_uint4(0, 0, 0, 0);
      logits_cluster_sync();  // every counter is 0
      const int inside = min(a.V - w0, window);
      for (int i = rank * nt + tid; i < len; i += p.slices * nt) {
        const int64_t id = load_int(a.tokens, (int64_t)row * a.tokens_stride + i, a.tokens_i64) - w0;
        if (id < 0 || id >= inside) continue;
        const uint32_t owner = (uint32_t)id / (uint32_t)p.slice;
        const uint32_t at = logits_peer(counters + ((uint32_t)id - owner * p.slice), owner);
        if (i >= prompt)
          peer_add(at, 1u);
        else
          peer_or(at, 0x80000000u);
      }
      logits_cluster_sync();  // every token is counted
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int o = (u * nt + tid) * kVec, e = base + o;
      const int n = o < p.slice ? min(a.V - e, kVec) : 0;
      if (n <= 0) continue;
      if (p.history) {
        const uint4 c0 = *reinterpret_cast<const uint4 *>(counters + o);
        const uint4 c1 = *reinterpret_cast<const uint4 *>(counters + o + 4);
        if (c0.x | c0.y | c0.z | c0.w | c1.x | c1.y | c1.z | c1.w) {
          const uint32_t c[kVec] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            if (c[i] == 0u) continue;
            float v = z[u][i];
            v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            const uint32_t count = c[i] & 0x7fffffffu;
            if (count) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)count)), pres);
            z[u][i] = v;
          }
        }
      }
      if (bias) {
        if (p.vec_bias && n == kVec) {
          const float4 b0 = reinterpret_cast<const float4 *>(bias + e)[0];
          const float4 b1 = reinterpret_cast<const float4 *>(bias + e)[1];
          z[u][0] += b0.x, z[u][1] += b0.y, z[u][2] += b0.z, z[u][3] += b0.w;
          z[u][4] += b1.x, z[u][5] += b1.y, z[u][6] += b1.z, z[u][7] += b1.w;
        } else {
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (i < n) z[u][i] += bias[e + i];
        }
      }
      if (allowed) {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
          if (!(ok[u] >> i & 1u)) z[u][i] = -CUDART_INF_F;
      }
      if (MODE == kProcess)
        store_run(z[u], static_cast<char *>(a.out) + (int64_t)row * a.out_ld * (a.out_dtype == M3_BF16 ? 2 : 4),
                  a.out_dtype == M3_BF16, e, n, p.vec_out);
    }
    if (MODE == kProcess) continue;

    float high = -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
#pragma unroll
      for (int i = 0; i < kVec; ++i) high = fmaxf(high, z[u][i]);
    if (tid < 2) first[tid] = INT_MAX;
    const float cta_high = cta_extreme<true>(high, scratch);
    const bool raised = cta_high > top;
    if (raised) {
      sum = sum * exp2_approx((top - cta_high) * scale);  // 0 for the first round
      if (top == -CUDART_INF_F) sum = 0.f;
      top = cta_high;
    }
    // a round of NaN and -infinity only: relative to 0, where -infinity gives 0 and NaN shows
    const float ref = top == -CUDART_INF_F ? 0.f : top;
    float part = 0.f, low = CUDART_INF_F, low_q = CUDART_INF_F;
    if (drawn) {
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const uint32_t e = (uint32_t)(base + (u * nt + tid) * kVec);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 w = noise.block((e >> 2) + h);
          const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = (z[u][4 * h + i] - ref) * scale;
            part += exp2_approx(x);
            const float q = exp2_approx(-x), l = noise_low(ws[i]) * q;
            if (l < low) low = l, low_q = q;
          }
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
#pragma unroll
        for (int i = 0; i < kVec; ++i) part += exp2_approx((z[u][i] - ref) * scale);
    }
    sum += part;
    // rare: the first NaN; always cheap: the first element that is the largest
    if (part != part || (raised && high == cta_high)) {
      int at = INT_MAX, bad = INT_MAX;
#pragma unroll
      for (int u = kVecs - 1; u >= 0; --u)
#pragma unroll
        for (int i = kVec - 1; i >= 0; --i) {
          const int e = base + (u * nt + tid) * kVec + i;
          if (z[u][i] == cta_high) at = e;
          if (z[u][i] != z[u][i]) bad = e;
        }
      if (raised && at != INT_MAX) atomicMin(&first[0], at);
      if (bad != INT_MAX) atomicMin(&first[1], bad);
    }
    if (drawn) {
      // an upper bound of e / p of this thread's lowest element, the CTA's
      // smallest of them, and room for the rounding of 1 / p
      const float v_high = low / low_q + 0x1p-22f;
      const float bound = low_q == CUDART_INF_F ? CUDART_INF_F : (v_high < 1.f ? -log1pf(-v_high) : 23.f) * low_q;
      const float limit = cta_extreme<false>(bound, scratch) * 1.001f;
      if (low <= limit && limit < CUDART_INF_F) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u)
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const int e = base + (u * nt + tid) * kVec + i;
            const float q = exp2_approx(-((z[u][i] - ref) * scale));
            if (!(q < CUDART_INF_F)) continue;
            const uint32_t w = noise.word((uint32_t)e);
            if (noise_low(w) * q <= limit) {
              const double g = draw_noise(w);
              if (draw_beats(z[u][i], g, e, best_z, best_g, best_id, temp)) best_g = g, best_id = e, best_z = z[u][i];
            }
          }
      }
    } else {
      __syncthreads();
    }
    __syncthreads();
    if (raised) top_id = first[0];
    nan_id = min(nan_id, first[1]);
    __syncthreads();  // `first` may be reset
  }
  if (MODE == kProcess) return;

  // the CTA's sum, in a fixed order, and its best drawn element
  sum = group_sum<32>(sum);
  if (drawn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double g = __shfl_xor_sync(kFullMask, best_g, o);
      const int id = __shfl_xor_sync(kFullMask, best_id, o);
      const float bz = __shfl_xor_sync(kFullMask, best_z, o);
      if (draw_beats(bz, g, id, best_z, best_g, best_id, temp)) best_g = g, best_id = id, best_z = bz;
    }
  }
  if ((tid & 31) == 0) {
    scratch[tid >> 5] = sum;
    warp_noise[tid >> 5] = best_g, warp_id[tid >> 5] = best_id, warp_z[tid >> 5] = best_z;
  }
  __syncthreads();
  if (tid == 0) {
    float s = scratch[0];
    for (int w = 1; w < nt >> 5; ++w) s += scratch[w];
    double g = 0.0;
    float chosen = top;
    int id = top_id;
    if (drawn && top < CUDART_INF_F) {
      g = warp_noise[0], id = warp_id[0], chosen = warp_z[0];
      for (int w = 1; w < nt >> 5; ++w)
        if (draw_beats(warp_z[w], warp_noise[w], warp_id[w], chosen, g, id, temp))
          g = warp_noise[w], id = warp_id[w], chosen = warp_z[w];
    }
    const uint64_t bits = (uint64_t)__double_as_longlong(g);
    mine.top = top, mine.sum = s, mine.id = id, mine.nan_id = nan_id, mine.z = chosen;
    mine.noise_hi = (uint32_t)(bits >> 32), mine.noise_lo = (uint32_t)bits;
  }
  logits_cluster_sync();  // every CTA's choice stands
  if (rank == 0 && tid == 0) {
    float all_top = -CUDART_INF_F, all_sum = 0.f, chosen = 0.f;
    double g = 0.0;
    int id = INT_MAX, bad = INT_MAX;
    for (int r = 0; r < p.slices; ++r) {
      const uint32_t at = logits_peer(&mine, (uint32_t)r);
      const float t = __uint_as_float(peer_load(at + offsetof(Choice, top)));
      const float s = __uint_as_float(peer_load(at + offsetof(Choice, sum)));
      const int i = (int)peer_load(at + offsetof(Choice, id));
      const float z = __uint_as_float(peer_load(at + offsetof(Choice, z)));
      const uint64_t bits = (uint64_t)peer_load(at + offsetof(Choice, noise_hi)) << 32 |
                            peer_load(at + offsetof(Choice, noise_lo));
      const double rg = __longlong_as_double((long long)bits);
      bad = min(bad, (int)peer_load(at + offsetof(Choice, nan_id)));
      if (t > all_top) {
        all_sum = all_top == -CUDART_INF_F ? s : all_sum * exp2f((all_top - t) * scale) + s;
        all_top = t;
      } else if (t > -CUDART_INF_F) {
        all_sum += s * exp2f((t - all_top) * scale);
      }
      // of two infinite logits the difference is NaN: the lower rank's stays
      if (draw_beats(z, rg, i, chosen, g, id, temp)) g = rg, id = i, chosen = z;
    }
    float lp;
    if (bad != INT_MAX) {
      id = bad, lp = CUDART_NAN_F;
    } else if (all_top == -CUDART_INF_F) {
      id = 0, lp = -CUDART_INF_F;
    } else {
      lp = (chosen - all_top) / temp - logf(all_sum);  // NaN with an infinite logit, as the formula gives
    }
    a.ids[row] = id;
    a.logprobs[row] = lp;
  }
  logits_cluster_sync();  // no CTA leaves while its choice is read
}

bool rows_on_16(const void *p, int64_t ld, int B, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (B == 1 || ld * size % 16 == 0);
}

template <typename T, int MODE>
cudaError_t launch_logits_t(const m3_logits_args &a, cudaStream_t stream) {
  LogitsParams p = {};
  p.a = a;
  p.history = a.tokens && a.T > 0 &&
              (a.repetition || a.presence || a.frequency || a.repetition_value != 1.f || a.presence_value != 0.f ||
               a.frequency_value != 0.f);
  p.vec_in = rows_on_16(a.logits, a.ld, a.B, sizeof(T));
  p.vec_out = a.out && rows_on_16(a.out, a.out_ld, a.B, a.out_dtype == M3_BF16 ? 2 : 4);
  p.vec_bias = a.bias && rows_on_16(a.bias, a.bias_stride, a.B, 4);
  const bool cluster = MODE == kChoose || p.history;
  if (cluster) {
    p.slices = 8;
    p.rounds = (int)(((int64_t)a.V + p.slices * kSliceMax - 1) / (p.slices * kSliceMax));
    const int parts = p.slices * p.rounds;
    p.slice = ((a.V + parts - 1) / parts + 31) / 32 * 32;
  } else {  // CTAs that need not meet: enough of them for one row
    p.slice = 2048;
    p.slices = (a.V + p.slice - 1) / p.slice;
    p.rounds = 1;
  }
  const int64_t grid = (int64_t)a.B * p.slices;
  if (grid > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)((p.slice + kPer - 1) / kPer + 31) / 32 * 32);
  cfg.dynamicSmemBytes = p.history ? (size_t)p.slice * 4 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.slices;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, logits_kernel<T, MODE>, p); e != cudaSuccess) return e;
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_process_logits(const m3_logits_args &a, cudaStream_t stream) {
  return a.dtype == M3_BF16 ? launch_logits_t<__nv_bfloat16, kProcess>(a, stream)
                            : launch_logits_t<float, kProcess>(a, stream);
}

cudaError_t launch_next_tokens(const m3_logits_args &a, cudaStream_t stream) {
  return a.dtype == M3_BF16 ? launch_logits_t<__nv_bfloat16, kChoose>(a, stream)
                            : launch_logits_t<float, kChoose>(a, stream);
}

}  // namespace m3
