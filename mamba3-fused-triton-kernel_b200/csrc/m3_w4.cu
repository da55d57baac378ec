// Products with 4-bit weights: y[m, n] = sum_k x[m, k] (q[n, k] - z[n, G]) s[n, G].
//
// For the batches a token step has, the call is a stream of the codes (half
// a byte a weight); everything else has to fit under it.
//
//   * q - z is an integer of at most 5 bits, exact in bf16, and 128 + q is
//     the bf16 whose mantissa ends in q: a pair of codes becomes a bf16 pair
//     with one mask-and-or and one packed subtraction of 128 + z.
//   * mma.sync.m16n8k16 (bf16 in, fp32 sums) takes the 16 weight rows as its
//     M and 8 batch rows as its N, so one batch row costs no more than eight.
//     Products of a bf16 x are exact; an fp32 x is cut into three bf16 terms
//     of 8 significant bits each (24 together, all of x) and takes three MMAs.
//   * The scale is applied to the fp32 sum of a group, not to the weight:
//     nothing is rounded below fp32 before the output.
//   * The order of k is free.  A block of 16 rows by 128 columns is 1 KB in
//     which lane (g, t) of a warp reads 16 bytes of row g and of row g + 8
//     (words 4 t + j, j = 0..3): two contiguous 512-byte loads.  Word j of a
//     row's four lanes is the columns 32 j + 8 t .. + 7, a 32-column run: two
//     MMAs, and the finest group.  The batch operand of both is the 8
//     consecutive elements of x at the same columns.
#include "m3_w4.cuh"

namespace m3 {

namespace {

__device__ __forceinline__ void w4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of codes, read once: past L1.  Volatile, so that it stays behind
// the wait for the preceding kernel.
__device__ __forceinline__ uint4 w4_codes(const char *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// 16 bytes global -> shared, or 16 zero bytes
__device__ __forceinline__ void w4_copy16(void *dst, const void *src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(real ? 16 : 0)
               : "memory");
}

// Where a lane's next blocks are: the codes of NT row blocks (one tile each),
// and the scales and zeros of its two rows (g and g + 8) of each.  32-bit byte
// offsets: the launcher takes no weight past them.
template <int NT, int GPT, bool ZEROS>
struct W4At {
  uint32_t c[NT], s[NT][2], z[NT][2];
  __device__ __forceinline__ void set(const W4Params &p, int rb, int kt, int lane) {
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      const int block = min(rb * NT + a, p.blocks - 1);  // past the last: reaches no output
      c[a] = ((uint32_t)block * p.tiles + kt) * 1024u + lane * 16u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t n = min(block * 16 + h * 8 + (lane >> 2), p.N - 1);
        s[a][h] = (n * (uint32_t)p.s_ld + kt * GPT) << (p.s_bf16 ? 1 : 2);
        if (ZEROS) z[a][h] = n * (uint32_t)p.z_ld + kt * GPT;
      }
    }
  }
  __device__ __forceinline__ void advance(const W4Params &p, int tiles) {
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      c[a] += tiles * 1024u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[a][h] += (uint32_t)(tiles * GPT) << (p.s_bf16 ? 1 : 2);
        if (ZEROS) z[a][h] += tiles * GPT;
      }
    }
  }
};

// The blocks' codes, scales and zeros of a lane as they lie in memory:
// nothing is computed from them before they are used, so that a load waits
// for none before it.
template <int NT, int GPT, bool ZEROS>
struct W4Stage {
  uint4 c[NT][2];
  uint32_t s[NT][2][GPT], z[NT][2][GPT];
  __device__ __forceinline__ void load(const W4Params &p, const W4At<NT, GPT, ZEROS> &at, int kt) {
    const char *codes = reinterpret_cast<const char *>(p.codes);
#pragma unroll
    for (int a = 0; a < NT; ++a) {
      c[a][0] = w4_codes(codes + at.c[a]);
      c[a][1] = w4_codes(codes + at.c[a] + 512);
    }
#pragma unroll
    for (int j = 0; j < GPT; ++j)
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool in = GPT == 1 || kt * GPT + j < p.groups;  // a group wholly past K has a sum of 0
          const char *sp = static_cast<const char *>(p.scales) + at.s[a][h];
          s[a][h][j] = !in ? 0u
                           : p.s_bf16 ? (uint32_t) reinterpret_cast<const uint16_t *>(sp)[j]
                                      : reinterpret_cast<const uint32_t *>(sp)[j];
          if (ZEROS) z[a][h][j] = in ? p.zeros[at.z[a][h] + j] : 0u;
        }
  }
  __device__ __forceinline__ float scale(const W4Params &p, int a, int h, int j) const {
    return __uint_as_float(p.s_bf16 ? s[a][h][j] << 16 : s[a][h][j]);
  }
  __device__ __forceinline__ uint32_t bias(int a, int h, int j) const {  // (128 + z, 128 + z)
    return ZEROS ? 0x43004300u + z[a][h][j] * 0x10001u : 0x43084308u;
  }
};

// tot += the products of NT row blocks with MT 8-row batch tiles; get(o, j, b)
// gives the terms of x for run j of the tile and batch tile b, which the row
// blocks share.  A run's two MMAs go to sums of their own where one tile
// would leave the chain of dependent MMAs bare.
template <int MT, int NT, int GPT, bool ZEROS, int TERMS, typename Get>
__device__ __forceinline__ void w4_block(const W4Params &p, float (&tot)[MT][NT][4],
                                         const W4Stage<NT, GPT, ZEROS> &st, Get get) {
  constexpr int PER = 4 / GPT;  // 32-column runs of a group
  constexpr int CHAINS = MT * NT == 1 ? 2 : 1;
  float d[MT][NT][CHAINS][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int gj = j / PER;
    if (j % PER == 0) {
#pragma unroll
      for (int b = 0; b < MT; ++b)
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
          for (int c = 0; c < CHAINS; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[b][a][c][e] = 0.f;
    }
    uint32_t w[NT][2][4];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t zz = st.bias(a, h, gj);
        const uint4 c = st.c[a][h];
        const uint32_t word = j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[a][h][i] = w4_pair(word, i, zz, p.mask, p.magic);
      }
#pragma unroll
    for (int b = 0; b < MT; ++b) {
      uint4 o[TERMS];
      get(o, j, b);
#pragma unroll
      for (int q = TERMS - 1; q >= 0; --q) {  // small terms first
#pragma unroll
        for (int a = 0; a < NT; ++a) w4_mma(d[b][a][0], w[a][0][0], w[a][1][0], w[a][0][1], w[a][1][1], o[q].x, o[q].y);
#pragma unroll
        for (int a = 0; a < NT; ++a)
          w4_mma(d[b][a][CHAINS - 1], w[a][0][2], w[a][1][2], w[a][0][3], w[a][1][3], o[q].z, o[q].w);
      }
    }
    if (j % PER == PER - 1) {
#pragma unroll
      for (int a = 0; a < NT; ++a) {
        const float s[2] = {st.scale(p, a, 0, gj), st.scale(p, a, 1, gj)};
#pragma unroll
        for (int b = 0; b < MT; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            tot[b][a][e] = fmaf(CHAINS == 2 ? d[b][a][0][e] + d[b][a][CHAINS - 1][e] : d[b][a][0][e], s[e >> 1],
                                tot[b][a][e]);
      }
    }
  }
}

constexpr int kW4SmemBudget = 227 * 1024;  // x and the partial sums: all an SM gives a CTA

// The shape of a CTA by its batch tiles MT and the row blocks NT of a warp.
// One tile: as many warps as the SM takes, which the chain unpack - MMA -
// scale of a block needs.  Two: two row blocks a warp, which share the batch
// operand's loads from shared memory, where that still leaves a row block to
// every SM (50,280 x 2,560, 16 rows: 26.6 against 32.0 us with one; 2,048 x
// 4,096 has 128 row blocks: 7.1 against 6.0 us).  Four: one row block and 16
// warps (64 rows of 9,440 x 2,048: 13.9 against 16.5 us with two and 12).
// Finer groups hold more scales in flight: fewer warps, one block.
template <int MT, int NT, int GPT>
struct W4Shape {
  static constexpr int kWarps = MT == 1 ? (GPT == 1 ? 32 : GPT == 2 ? 24 : 16) : 16;
  static constexpr int kDepth = 2;                         // blocks a warp has in flight: 32 KB an SM or more
  static constexpr int kLd = NT * 16 + 1;                  // partial sums of a batch row, padded against conflicts
  static constexpr int kRed = MT * 8 * kLd;                // partial sums of a warp
  static constexpr int kBufs = MT == 4 ? 1 : 2;            // of them: a second one saves a barrier, x wants the room
};

// x as the MMAs take it: [tile][run j][batch tile][term][lane] pieces of 16 bytes
template <typename S, int MT, int TERMS>
int64_t w4_stream_smem(int tiles, int wk, int wn) {
  return (int64_t)tiles * 4 * MT * TERMS * 512 + (int64_t)S::kBufs * wk * wn * S::kRed * 4;
}

// The decode batches' kernel: persistent CTAs that hold all of x in shared
// memory, in fragment order, and stream blocks of codes through registers,
// a few ahead.  A CTA's p.wk x p.wn warps are p.wn groups; a group takes NT
// row blocks in turn, its warps the tiles kt = wk, wk + p.wk, ... of them, and
// their sums are added in warp order through shared memory, behind a barrier
// of the group.
template <typename XT, int MT, int NT, int GPT, bool ZEROS>
__global__ void __launch_bounds__(W4Shape<MT, NT, GPT>::kWarps * 32, 1) w4_stream_kernel(const W4Params p) {
  using X = W4X<XT>;
  using S = W4Shape<MT, NT, GPT>;
  constexpr int TERMS = X::kTerms, RED = S::kRed, DEPTH = S::kDepth, ROWS = NT * 16, LD = S::kLd;
  extern __shared__ __align__(16) uint4 w4_smem[];
  const int pieces = p.tiles * 4 * MT * 32;
  float *red = reinterpret_cast<float *>(w4_smem + (int64_t)pieces * TERMS);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wk = warp % p.wk, wn = warp / p.wk;
  const int m0 = (int)(blockIdx.x % p.mtiles) * MT * 8, rows = min(p.M - m0, MT * 8);
  const int rb0 = (int)(blockIdx.x / p.mtiles) * p.wn + wn, rstep = (int)(gridDim.x / p.mtiles) * p.wn;
  const int rbs = (p.blocks + NT - 1) / NT;
  const int steps = wk < p.tiles ? (p.tiles - wk + p.wk - 1) / p.wk : 0;  // of this warp in a row block

  // the first blocks into L2 while the preceding kernel runs
  if (rb0 < rbs && wk == 0 && lane < NT && rb0 * NT + lane < p.blocks) {
    const uint32_t bytes = (uint32_t)min(p.tiles, DEPTH * p.wk) * 1024u;
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.codes + (int64_t)(rb0 * NT + lane) * p.tiles * 64),
                 "r"(bytes)
                 : "memory");
  }
  pdl_wait();  // x is the preceding kernel's output, and the weight may be too
  pdl_trigger();

  int lrb = rb0, lk = wk;  // the next blocks to load
  W4At<NT, GPT, ZEROS> at;
  if (steps > 0) at.set(p, min(lrb, rbs - 1), lk, lane);
  auto load = [&](W4Stage<NT, GPT, ZEROS> &st) {
    if (lrb >= rbs) return;
    st.load(p, at, lk);
    lk += p.wk;
    if (lk < p.tiles) {
      at.advance(p, p.wk);
    } else {
      lk = wk, lrb += rstep;
      if (lrb < rbs) at.set(p, lrb, lk, lane);
    }
  };
  W4Stage<NT, GPT, ZEROS> st[DEPTH];
  if (steps > 0) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) load(st[u]);
  }

  // x into shared memory: a bf16 piece is copied as it is, all copies in
  // flight; fp32 and odd pieces go through registers, a few at a time
  auto stage = [&](int i) {  // row and column of piece i
    const int l = i & 31, b = (i >> 5) % MT, kj = (i >> 5) / MT;
    return make_int2(b * 8 + (l >> 2), kj * 32 + 8 * (l & 3));
  };
  if (TERMS == 1 && p.x_vec) {
    for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
      const int2 at = stage(i);
      const bool real = at.x < rows && at.y + 8 <= p.K;
      if (at.x < rows && at.y < p.K && !real) {
        X xv;
        uint4 o[TERMS];
        xv.load(p.x, (int64_t)(m0 + at.x) * p.ldx, at.y, p.K, false);
        xv.terms(o);
        w4_smem[i] = o[0];
      } else {
        const XT *src = static_cast<const XT *>(p.x) + (real ? (int64_t)(m0 + at.x) * p.ldx + at.y : 0);
        w4_copy16(w4_smem + i, src, real);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    constexpr int AHEAD = TERMS == 1 ? 4 : 2;
    for (int i0 = threadIdx.x; i0 < pieces; i0 += AHEAD * blockDim.x) {
      X xv[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = i0 + u * blockDim.x;
        const int2 at = stage(i);
        if (i < pieces && at.x < rows)
          xv[u].load(p.x, (int64_t)(m0 + at.x) * p.ldx, at.y, p.K, p.x_vec);
        else
          xv[u].zero();
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int i = i0 + u * blockDim.x;
        uint4 o[TERMS];
        xv[u].terms(o);
        if (i < pieces) {
#pragma unroll
          for (int q = 0; q < TERMS; ++q) w4_smem[((i >> 5) * TERMS + q) * 32 + (i & 31)] = o[q];
        }
      }
    }
  }
  __syncthreads();

  float tot[MT][NT][4];
  // the row blocks are done: their sums, added over the group's warps
  auto finish = [&](int rb, int parity) {
    // element e of a tile: weight row g + 8 (e / 2), batch row 2 t + e % 2
    float *group = red + ((S::kBufs == 2 ? parity * p.wn : 0) + wn) * p.wk * RED;
    float *mine = group + wk * RED;
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mine[(b * 8 + 2 * (lane & 3) + (e & 1)) * LD + a * 16 + (e >> 1) * 8 + (lane >> 2)] = tot[b][a][e];
    if (p.wk > 1)
      asm volatile("bar.sync %0, %1;" ::"r"(wn), "r"(p.wk * 32) : "memory");
    else
      __syncwarp();
    for (int i = wk * 32 + lane; i < rows * ROWS; i += p.wk * 32) {
      const int r = i % ROWS, m = i / ROWS, n = rb * ROWS + r;
      float s = group[m * LD + r];
      for (int k = 1; k < p.wk; ++k) s += group[k * RED + m * LD + r];
      if (n < p.N) w4_store(p, m0 + m, n, s);
    }
    if (S::kBufs == 1) {  // the sums have been read
      if (p.wk > 1)
        asm volatile("bar.sync %0, %1;" ::"r"(wn), "r"(p.wk * 32) : "memory");
      else
        __syncwarp();
    }
  };
  auto clear = [&] {
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) tot[b][a][e] = 0.f;
  };
  const int xstep = 4 * MT * TERMS * 32;  // pieces of a tile
  int rb = rb0, left = steps, parity = 0;
  const uint4 *xs = w4_smem + (int64_t)wk * xstep + lane;
  clear();
  if (steps == 0) {  // more warps than tiles: zeros to the sums
    for (; rb < rbs; rb += rstep, parity ^= 1) finish(rb, parity);
    return;
  }
  while (rb < rbs) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) {
      if (rb < rbs) {
        w4_block<MT, NT, GPT, ZEROS, TERMS>(p, tot, st[u], [&](uint4 (&o)[TERMS], int j, int b) {
#pragma unroll
          for (int q = 0; q < TERMS; ++q) o[q] = xs[((j * MT + b) * TERMS + q) * 32];
        });
        load(st[u]);
        xs += p.wk * xstep;
        if (--left == 0) {
          finish(rb, parity);
          clear();
          parity ^= 1, left = steps, rb += rstep, xs = w4_smem + (int64_t)wk * xstep + lane;
        }
      }
    }
  }
}

// Any batch and any K (a weight of less than 4 GB): the same blocks, x read
// where it is.  A CTA is 8 warps, 2 along K by 4 row blocks that share x
// through L1.
template <typename XT, int MT, int GPT, bool ZEROS>
__global__ void __launch_bounds__(256) w4_direct_kernel(const W4Params p, int mtiles) {
  using X = W4X<XT>;
  constexpr int WK = 2, WN = 4, COLS = MT * 8, LD = 17;
  __shared__ float red[WN][WK][COLS * LD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wk = warp % WK, wn = warp / WK;
  const int m0 = (int)(blockIdx.x % mtiles) * COLS;
  const int rb = min((int)(blockIdx.x / mtiles) * WN + wn, p.blocks - 1);  // past the last: computed, not stored
  float tot[MT][1][4];
#pragma unroll
  for (int b = 0; b < MT; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) tot[b][0][e] = 0.f;
  pdl_wait();
  pdl_trigger();
  W4Stage<1, GPT, ZEROS> cur, nxt;
  W4At<1, GPT, ZEROS> at;
  at.set(p, rb, wk, lane);
  if (wk < p.tiles) cur.load(p, at, wk);
  for (int kt = wk; kt < p.tiles; kt += WK) {
    at.advance(p, WK);
    if (kt + WK < p.tiles) nxt.load(p, at, kt + WK);
    w4_block<MT, 1, GPT, ZEROS, X::kTerms>(p, tot, cur, [&](uint4 (&o)[X::kTerms], int j, int b) {
      const int m = m0 + b * 8 + g;
      X xv;
      if (m < p.M)
        xv.load(p.x, (int64_t)m * p.ldx, kt * M3_W4_TILE + 32 * j + 8 * t, p.K, p.x_vec);
      else
        xv.zero();
      xv.terms(o);
    });
    cur = nxt;
  }
#pragma unroll
  for (int b = 0; b < MT; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[wn][wk][(b * 8 + 2 * t + (e & 1)) * LD + (e >> 1) * 8 + g] = tot[b][0][e];
  __syncthreads();
  for (int i = threadIdx.x; i < COLS * WN * 16; i += 256) {
    const int r = i & 15, w = (i >> 4) % WN, c = i / (WN * 16);
    const int m = m0 + c, n = ((int)(blockIdx.x / mtiles) * WN + w) * 16 + r;
    if (m < p.M && n < p.N) w4_store(p, m, n, red[w][0][c * LD + r] + red[w][1][c * LD + r]);
  }
}

template <typename XT, int MT, int GPT, bool ZEROS>
cudaError_t launch_w4_direct(const W4Params &p, cudaStream_t stream) {
  const int mtiles = (p.M + MT * 8 - 1) / (MT * 8);
  const int64_t grid = (int64_t)((p.blocks + 3) / 4) * mtiles;
  if (grid > 0x7fffffff) return cudaErrorInvalidValue;
  return launch_pdl(w4_direct_kernel<XT, MT, GPT, ZEROS>, dim3((unsigned)grid), dim3(256), 0, stream, p, mtiles);
}

// Warps along K: the split with the fewest steps of the busiest warp (fewest
// warps a row block on ties: less to add up), then as many row blocks per CTA
// as keep every SM busy.
template <typename XT, int MT, int NT, int GPT, bool ZEROS>
cudaError_t launch_w4_stream(W4Params p, cudaStream_t stream, bool *taken) {
  using S = W4Shape<MT, NT, GPT>;
  constexpr int TERMS = W4X<XT>::kTerms, WARPS = S::kWarps;
  p.mtiles = (p.M + MT * 8 - 1) / (MT * 8);
  const int sms = max(1, sm_count_current() / p.mtiles);  // of a batch tile
  const int rbs = (p.blocks + NT - 1) / NT;
  int64_t best = INT64_MAX;
  for (int wk = (WARPS + 15) / 16; wk <= WARPS; wk *= 2) {  // at most 16 groups: a barrier each
    const int64_t streams = (int64_t)sms * (WARPS / wk);
    const int64_t steps = (rbs + streams - 1) / streams * ((p.tiles + wk - 1) / wk);
    if (steps < best) best = steps, p.wk = wk;
  }
  p.wn = min(WARPS / p.wk, (rbs + sms - 1) / sms);
  const int64_t smem = w4_stream_smem<S, MT, TERMS>(p.tiles, p.wk, p.wn);
  *taken = smem <= kW4SmemBudget;
  if (!*taken) return cudaSuccess;
  auto kern = w4_stream_kernel<XT, MT, NT, GPT, ZEROS>;
  static LaunchCache cache;
  if (cudaError_t e = ensure_smem_optin(cache, kern, kW4SmemBudget); e != cudaSuccess) return e;
  const int64_t grid = (int64_t)min(sms, (rbs + p.wn - 1) / p.wn) * p.mtiles;
  if (grid > 0x7fffffff) return cudaErrorInvalidValue;
  return launch_pdl(kern, dim3((unsigned)grid), dim3(p.wk * p.wn * 32), (size_t)smem, stream, p);
}

template <typename XT, int GPT, bool ZEROS>
cudaError_t launch_w4_x(const W4Params &p, cudaStream_t stream) {
  bool taken = false;
  cudaError_t e = cudaSuccess;
  // the largest batch tile whose x fits in shared memory, whatever M: fp32 rows
  // of 2,048 x 4,096, where that is 8, here / in the direct kernel, us: 64 rows
  // 18 / 112, 256 rows 55 / 183, 4,096 rows 795 / 2,091
  if (p.M > 16) e = launch_w4_stream<XT, 4, 1, GPT, ZEROS>(p, stream, &taken);
  if (!taken && e == cudaSuccess && p.M > 8) {
    if constexpr (GPT != 4)
      if (p.blocks >= 2 * sm_count_current()) e = launch_w4_stream<XT, 2, 2, GPT, ZEROS>(p, stream, &taken);
    if (!taken && e == cudaSuccess) e = launch_w4_stream<XT, 2, 1, GPT, ZEROS>(p, stream, &taken);
  }
  if (!taken && e == cudaSuccess) e = launch_w4_stream<XT, 1, 1, GPT, ZEROS>(p, stream, &taken);
  if (taken || e != cudaSuccess) return e;
  return p.M <= 8 ? launch_w4_direct<XT, 1, GPT, ZEROS>(p, stream) : launch_w4_direct<XT, 4, GPT, ZEROS>(p, stream);
}

template <typename XT, int GPT>
cudaError_t launch_w4_z(const W4Params &p, cudaStream_t stream) {
  return p.zeros ? launch_w4_x<XT, GPT, true>(p, stream) : launch_w4_x<XT, GPT, false>(p, stream);
}

template <typename XT>
cudaError_t launch_w4_g(const W4Params &p, int group, cudaStream_t stream) {
  return group == 128 ? launch_w4_z<XT, 1>(p, stream)
                      : group == 64 ? launch_w4_z<XT, 2>(p, stream) : launch_w4_z<XT, 4>(p, stream);
}

}  // namespace

cudaError_t launch_linear_w4(const m3_w4_args &a, cudaStream_t stream) {
  W4Params p = {};
  p.M = a.M, p.N = a.N, p.K = a.K;
  p.tiles = (int)(((int64_t)a.K + M3_W4_TILE - 1) / M3_W4_TILE);
  p.blocks = (int)(((int64_t)a.N + M3_W4_ROWS - 1) / M3_W4_ROWS);
  p.x = a.x, p.ldx = a.ldx;
  const int es = a.x_dtype == M3_BF16 ? 2 : 4;
  p.x_vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ldx * es % 16 == 0;
  p.codes = reinterpret_cast<const uint4 *>(a.codes);
  p.mask = 0x000F000Fu, p.magic = 0x43004300u;
  p.scales = a.scales, p.s_ld = a.scale_stride, p.s_bf16 = a.s_dtype == M3_BF16;
  p.groups = (int)(((int64_t)a.K + a.group - 1) / a.group);
  p.zeros = a.zeros, p.z_ld = a.zero_stride;
  p.y = a.y, p.ldy = a.ldy, p.y_bf16 = a.y_dtype == M3_BF16;
  // Many rows of a bf16 x go to the tensor memory path once there are some 30
  // blocks and 64 batch rows of work for an SM: us there / with the kernels
  // here, G 128, 50,280 x 2,560, 64 rows 31 / 72, 256 rows 78 / 204; 9,440 x
  // 2,048, 64 rows 11.2 / 13.9; 4,096 x 2,048 (27.7 blocks an SM), 64 rows
  // 8.8 / 8.8; 4,224 x 1,024 (14.3), 64 rows 7.3 / 5.7, 128 rows 8.8 / 8.4.  17
  // to 32 rows take more work, and groups of 128, whose sums are read back
  // least often: 32 rows of 50,280 x 2,560 31 / 42, of 9,440 x 2,048 11.0 / 9.3;
  // with groups of 64 48 / 44.  Finer groups at 64 rows, G 64 and G 32: 50,280 x
  // 2,560 48 / 77 and 74 / 93, 20,000 x 1,024 (67.6) 15.3 / 23.3 and 22.3 / 26.1,
  // 9,440 x 2,048 (63.8) 12.9 / 14.7 and 17.1 / 17.6, 4,096 x 2,048 9.4 / 9.3 and
  // 11.9 / 10.8: for groups of 32 the two cross at some 60 blocks an SM, and
  // between 30 and that the rule loses up to a sixth.
  const int64_t work = (int64_t)p.blocks * p.tiles * ((a.M + 63) / 64);
  if (a.x_dtype == M3_BF16 && ((a.M > 32 && work >= 30ll * sm_count_current()) ||
                               (a.M > 16 && a.group == 128 && work >= 150ll * sm_count_current()))) {
    bool taken = false;
    if (cudaError_t e = launch_w4_tc(p, a.group, stream, &taken); taken || e != cudaSuccess) return e;
  }
  return a.x_dtype == M3_BF16 ? launch_w4_g<__nv_bfloat16>(p, a.group, stream)
                              : launch_w4_g<float>(p, a.group, stream);
}

}  // namespace m3
