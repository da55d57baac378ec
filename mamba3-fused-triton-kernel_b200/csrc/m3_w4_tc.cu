// Products with 4-bit weights for many batch rows (bf16 x), on tcgen05 with
// the weight as the MMA's A from TMEM.
//
// D[128 weight rows, NB batch rows] of one group of columns = (q - z) times
// x, exact products and fp32 sums; the group's scale is applied when D is
// read back, so nothing is rounded below fp32 before the output.  x comes by
// TMA as the MMA takes it.  The weight has to be unpacked; unpacked into TMEM
// it never crosses shared memory.  A warp's TMEM lanes are its rows, so a
// thread unpacks one row: 64 bytes of codes are the 64 32-bit columns of a
// 128-column tile, in order.
//
//   readers      8 or 16 warps: D (TMEM lanes 32 (w % 4) .. + 31: the
//                thread's weight row, a share of the batch rows each), times
//                the row's scale into registers, stored at the end
//   unpackers    the other 16 or 8 of the first 24 warps, in sets of four
//                that take the tiles in turn: warp w of a set the rows of
//                lanes 32 (w % 4) .., and their scales into shared memory
//   warp 24      one lane: copies of codes into a ring of tiles
//   warp 25      one lane: copies of x likewise
//   warps 26-27  one lane each: the MMAs of every other group; the first
//                allocates TMEM
//
// What bounds it is the hand-overs and the issue of MMAs and commits, about
// 90 and 300 cycles each, hence two warps for them and few commits: a tile's
// MMAs take 512 cycles (NB 128), the kernel 1,150.  Steps, 1,024 rows of 9,440
// x 2,048: one MMA warp, three commits a tile, 8 readers of 64 columns 89 us;
// two, one barrier for a tile's places, 16 readers 62; scales through shared
// memory, D read 16 columns at a time, which spills nothing 57; stores with
// their addresses hoisted 47; elect.sync for the one lane 44 (tensor pipe
// active 42 % of the time).  Groups of 32 read D four times as often: 99 us.
// 64 rows of 50,280 x 2,560: 31 us (72 with the stream kernel); 256 rows of
// 9,440 x 2,048: 14 (75).  NB is 64 up to 64 rows (46 us with 128), with 16
// unpackers for groups of 128 and 16 readers for finer ones (73 us for groups
// of 32, 76 the other way).
//
// CTAs are persistent over items of 128 weight rows by NB batch rows.  Where
// there are too few of them and K is long, the CTAs of a cluster split K and
// their sums are added in rank order through distributed shared memory, which
// takes as long as about six tiles (128 rows of 4,224 x 1,024, 8 tiles: 8.3
// with one, 8.8 us with four).  Clusters of 8 took longer than of 4 (128 rows
// of 2,048 x 4,096: 21 against 12 us).  Every mbarrier wait is bounded; no copy
// uses cluster multicast.
#include <cuda.h>

#include "m3_async.cuh"
#include "m3_tmap.cuh"
#include "m3_w4.cuh"

namespace m3 {

namespace {

constexpr int kTcRows = 128;        // weight rows of an item
constexpr int kTcCodes = 8 * 1024;  // codes of a tile
constexpr int kTcRing = 4;          // tiles of x, and of unpacked codes (64 TMEM columns each)
constexpr int kTcCodeRing = 8;      // tiles of codes
constexpr int kTcMmas = 2;          // warps that issue MMAs
constexpr int kTcCopyCodes = 24, kTcCopyX = kTcCopyCodes + 1, kTcMma = kTcCopyX + 1;
constexpr int kTcThreads = (kTcMma + kTcMmas) * 32;
constexpr int kTmemCols = 512;

// Shared memory: x, codes, scales (128 of each of a tile's GPT groups),
// barriers, and up to 1,024 bytes of alignment.  NB: batch rows of an item.
template <int NB, int GPT>
struct TcSmem {
  static constexpr int kD = 256 / NB;  // accumulators, NB TMEM columns each
  static constexpr int kScaleRing = 4 * kD;  // tiles of scales: more than the ring and the accumulators together
  static constexpr int kX = NB * 256;  // of a tile: two 64-column halves
  static constexpr int kCodes = kTcRing * kX, kScales = kCodes + kTcCodeRing * kTcCodes;
  static constexpr int kBars = kScales + kScaleRing * GPT * kTcRows * 4;
  static constexpr int kBytes = kBars + 512 + 1024;
  static_assert(64 * kTcRing + NB * kD <= kTmemCols, "TMEM columns");
  static_assert((3 * kTcRing + 2 * kTcCodeRing + 2 * kD) * 8 + 8 <= 512, "barriers");
  static_assert(kTcRows * NB * 4 <= kCodes, "the sums of a split K take the place of x");
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// One thread of the warp, which the compiler knows to be one: it then issues
// tcgen05 instructions from uniform registers without a loop over threads.
__device__ __forceinline__ bool tc_elect() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void tc_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// A from TMEM, B from shared memory
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// K-major operand in the 128-byte swizzle: 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t tc_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tc_load_x(uint32_t dst, const CUtensorMap *map, int k, int m, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(k), "r"(m), "r"(bar)
      : "memory");
}
// 8 row blocks of one tile of the codes
__device__ __forceinline__ void tc_load_codes(uint32_t dst, const CUtensorMap *map, int kt, int rb, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(kt), "r"(rb), "r"(bar)
      : "memory");
}
// 16 columns of this thread's TMEM lane; with the wait in one statement, so
// that no use of them is moved before it
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float tc_peer_f32(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// mbar_wait that lets the warp sleep for up to 10 us a poll: with this many
// warps waiting, polls would take half of the issue slots.  Bounded likewise.
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < 1 << 18; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(10000)
        : "memory");
    if (ok) return true;
  }
  atomicOr(&g_device_error, M3_DEVERR_TIMEOUT);
  return false;
}

// A ring position: slot and the parity of its phase.
template <int S>
struct TcPos {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == S) s = 0, ph ^= 1u;
  }
};

// cs: CTAs that split K; items: (128 weight rows, NB batch rows) pairs
template <int NB, int GPT>
__global__ void __launch_bounds__(kTcThreads, 1)
    w4_tc_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tcodes, const W4Params p,
                 int cs, int items) {
  using L = TcSmem<NB, GPT>;
  constexpr int READERS = NB == 64 && GPT == 1 ? 8 : 16, SETS = (kTcCopyCodes - READERS) / 4;
  extern __shared__ unsigned char tc_raw[];
  unsigned char *smem =
      reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~(uintptr_t)1023);
  float *red = reinterpret_cast<float *>(smem);
  auto xs = [&](int i) { return smem + i * L::kX; };  // 1024-byte aligned
  auto codes = [&](int i) { return smem + L::kCodes + i * kTcCodes; };
  auto scales = [&](int i, int g) { return reinterpret_cast<float *>(smem + L::kScales) + (i * GPT + g) * kTcRows; };
  uint64_t *x_full = reinterpret_cast<uint64_t *>(smem + L::kBars), *a_full = x_full + kTcRing,
           *done = a_full + kTcRing, *c_full = done + kTcRing, *c_empty = c_full + kTcCodeRing,
           *d_full = c_empty + kTcCodeRing, *d_empty = d_full + L::kD;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(d_empty + L::kD);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)blockIdx.x % cs, item0 = (int)blockIdx.x / cs, istep = (int)gridDim.x / cs;
  const int kper = (p.tiles + cs - 1) / cs;
  const int k0 = min(rank * kper, p.tiles), k1 = min(k0 + kper, p.tiles);

  if (tid == 0) {
    // done: a tile's MMAs, which leave the places of its x and its unpacked codes free
    for (int i = 0; i < kTcRing; ++i)
      mbar_init(smem_addr(&x_full[i]), 1), mbar_init(smem_addr(&a_full[i]), 4),
          mbar_init(smem_addr(&done[i]), GPT == 1 ? 1 : kTcMmas);
    for (int i = 0; i < kTcCodeRing; ++i) mbar_init(smem_addr(&c_full[i]), 1), mbar_init(smem_addr(&c_empty[i]), 4);
    for (int i = 0; i < L::kD; ++i) mbar_init(smem_addr(&d_full[i]), 1), mbar_init(smem_addr(&d_empty[i]), READERS);
    mbar_init_fence();
  }
  if (warp == kTcMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_d = tmem + 64 * kTcRing;

  pdl_wait();  // x is the preceding kernel's output, and the weight may be too
  pdl_trigger();

  if (warp < READERS) {
    // read D, scale, sum: batch rows c0 .. + COLS of the item
    constexpr int COLS = NB * 4 / READERS;
    const int c0 = warp / 4 * COLS, lrow = tid % 128;
    TcPos<L::kD> d;
    bool live = true;
    int tile = 0;
    for (int item = item0; item < items; item += istep) {
      const int m0 = item % p.mtiles * NB, n = item / p.mtiles * kTcRows + lrow;
      float acc[COLS];
#pragma unroll
      for (int m = 0; m < COLS; ++m) acc[m] = 0.f;
      for (int g = 0; g < (k1 - k0) * GPT; ++g) {
        if (live) live = tc_wait(smem_addr(&d_full[d.s]), d.ph);
        const float s = scales(tile & (L::kScaleRing - 1), GPT == 1 ? 0 : g & (GPT - 1))[lrow];
        if (GPT == 1 || (g & (GPT - 1)) == GPT - 1) ++tile;
        __syncwarp();
        tc_after();
        const uint32_t at = tmem_d + (uint32_t)(d.s * NB + c0) + ((uint32_t)(32 * (warp & 3)) << 16);
#pragma unroll
        for (int c = 0; c < COLS; c += 16) {
          uint32_t v[16];
          tc_ld16(at + c, v);
          if (c + 16 == COLS) {
            tc_before();
            __syncwarp();
            if (lane == 0) tc_arrive(smem_addr(&d_empty[d.s]));
          }
#pragma unroll
          for (int m = 0; m < 16; ++m) acc[c + m] = fmaf(__uint_as_float(v[m]), s, acc[c + m]);
        }
        d.next();
      }
      if (cs == 1) {
        const int rows = n < p.N ? p.M - m0 - c0 : 0;
        const int64_t at = (int64_t)(m0 + c0) * p.ldy + n;
        if (p.y_bf16) {
          __nv_bfloat16 *y = static_cast<__nv_bfloat16 *>(p.y) + at;
#pragma unroll
          for (int m = 0; m < COLS; ++m, y += p.ldy)
            if (m < rows) *y = __float2bfloat16_rn(acc[m]);
        } else {
          float *y = static_cast<float *>(p.y) + at;
#pragma unroll
          for (int m = 0; m < COLS; ++m, y += p.ldy)
            if (m < rows) *y = acc[m];
        }
      } else {
        // the one item is done: all MMAs have read the ring, no copy is under way
#pragma unroll
        for (int m = 0; m < COLS; ++m) red[(c0 + m) * kTcRows + lrow] = acc[m];
      }
    }
  } else if (warp < kTcCopyCodes) {
    // unpack: this warp's rows of every SETS-th tile, and their scales
    const int quarter = warp & 3, set = (warp - READERS) >> 2, lrow = quarter * 32 + lane;
    const int per = k1 - k0, total = item0 < items ? (items - item0 + istep - 1) / istep * per : 0;
    uint32_t zraw[GPT], sraw[GPT];  // zeros and scales of this warp's next tile, as they lie in memory
    int next = set, item = item0, kt = k0 + set;
    // a tile's loads are asked for before the tile before it is unpacked, also
    // from one item to the next
    auto fetch = [&] {
      if (next >= total) return;
      while (kt >= k1) kt -= per, item += istep;
      const int64_t n = min(item / p.mtiles * kTcRows + lrow, p.N - 1);
      const int64_t srow = n * p.s_ld;
      const uint8_t *zrow = p.zeros ? p.zeros + n * p.z_ld : nullptr;
#pragma unroll
      for (int j = 0; j < GPT; ++j) {
        const int g = kt * GPT + j;
        zraw[j] = 8u, sraw[j] = 0u;  // of a group wholly past K, whose sum is 0
        if (g < p.groups) {
          if (zrow) zraw[j] = zrow[g];
          sraw[j] = p.s_bf16 ? (uint32_t) static_cast<const uint16_t *>(p.scales)[srow + g]
                             : static_cast<const uint32_t *>(p.scales)[srow + g];
        }
      }
      next += SETS, kt += SETS;
    };
    bool live = true;
    fetch();
    for (int i = set; i < total; i += SETS) {
      const int c = i % kTcCodeRing, a = i % kTcRing;
      uint32_t zz[GPT];  // (128 + z, 128 + z)
      float sc[GPT];
#pragma unroll
      for (int j = 0; j < GPT; ++j) {
        zz[j] = 0x43004300u + zraw[j] * 0x10001u;
        sc[j] = __uint_as_float(p.s_bf16 ? sraw[j] << 16 : sraw[j]);
      }
      fetch();
      if (live) live = tc_wait(smem_addr(&c_full[c]), i / kTcCodeRing & 1);
      const uint4 *src = reinterpret_cast<const uint4 *>(codes(c)) + lrow * 4;
      uint4 q[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) q[t] = src[t];
      if (live) live = tc_wait(smem_addr(&done[a]), (i / kTcRing & 1) ^ 1);
      // tile i - 4 is done, so its accumulator's tile before, i - 4 - kD or a
      // later one, has been read, and the scales of all up to that
#pragma unroll
      for (int j = 0; j < GPT; ++j) scales(i & (L::kScaleRing - 1), j)[lrow] = sc[j];
      __syncwarp();
      tc_after();
      const uint32_t at = tmem + (uint32_t)(a * 64) + ((uint32_t)(32 * quarter) << 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // columns 32 j ..: words 4 t + j
        uint32_t r[16];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t w = j == 0 ? q[t].x : j == 1 ? q[t].y : j == 2 ? q[t].z : q[t].w;
#pragma unroll
          for (int e = 0; e < 4; ++e) r[4 * t + e] = w4_pair(w, e, zz[j * GPT / 4], p.mask, p.magic);
        }
        tc_st16(at + 16 * j, r);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_before();
      __syncwarp();
      if (lane == 0) {
        tc_arrive(smem_addr(&a_full[a]));
        tc_arrive(smem_addr(&c_empty[c]));  // here, where the codes have been used: an arrival may overtake a load
      }
    }
  } else if (warp == kTcCopyCodes) {
    if (tc_elect()) {
      TcPos<kTcCodeRing> c;
      int issued = 0;
      bool live = true;
      for (int item = item0; item < items && live; item += istep) {
        const int rb = item / p.mtiles * (kTcRows / M3_W4_ROWS);
        for (int kt = k0; kt < k1 && live; ++kt, c.next()) {
          live = tc_wait(smem_addr(&c_empty[c.s]), c.ph ^ 1u);
          if (!live) break;
          const uint32_t bar = smem_addr(&c_full[c.s]);
          mbar_arrive_expect_tx(bar, kTcCodes);
          tc_load_codes(smem_addr(codes(c.s)), &tcodes, kt, rb, bar);  // rows past the weight's: zeros
          ++issued;
        }
      }
      // the copies in flight land before this thread leaves
      for (int j = max(0, issued - kTcCodeRing); j < issued; ++j)
        tc_wait(smem_addr(&c_full[j % kTcCodeRing]), (uint32_t)((j / kTcCodeRing) & 1));
    }
    __syncwarp();
  } else if (warp == kTcCopyX) {
    if (tc_elect()) {
      TcPos<kTcRing> c;
      int issued = 0;
      bool live = true;
      for (int item = item0; item < items && live; item += istep) {
        const int m0 = item % p.mtiles * NB;
        for (int kt = k0; kt < k1 && live; ++kt, c.next()) {
          live = tc_wait(smem_addr(&done[c.s]), c.ph ^ 1u);
          if (!live) break;
          const uint32_t bar = smem_addr(&x_full[c.s]);
          mbar_arrive_expect_tx(bar, L::kX);
          for (int h = 0; h < 2; ++h)  // rows and columns past x's: zeros
            tc_load_x(smem_addr(xs(c.s) + h * (L::kX / 2)), &tx, kt * M3_W4_TILE + h * 64, m0, bar);
          ++issued;
        }
      }
      for (int j = max(0, issued - kTcRing); j < issued; ++j)
        tc_wait(smem_addr(&x_full[j % kTcRing]), (uint32_t)((j / kTcRing) & 1));
    }
    __syncwarp();
  } else {
    if (tc_elect()) {
      // fp32 accumulator, bf16 A and B, both K-major, N / 8 and M / 16
      const uint32_t idesc =
          (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NB >> 3) << 17) | ((uint32_t)(kTcRows >> 4) << 24);
      // every other group, the accumulators in turn
      const int me = warp - kTcMma;
      TcPos<kTcRing> c, last;
      TcPos<L::kD / kTcMmas> d;
      bool live = true, any = false;
      int i = 0;
      for (int item = item0; item < items && live; item += istep) {
        for (int kt = k0; kt < k1 && live; ++kt, ++i, c.next()) {
          if (GPT == 1 && (i & 1) != me) continue;
          live = tc_wait(smem_addr(&x_full[c.s]), c.ph) && tc_wait(smem_addr(&a_full[c.s]), c.ph);
          if (!live) break;
          const uint32_t ta = tmem + (uint32_t)(c.s * 64), sb = smem_addr(xs(c.s));
          for (int g = GPT == 1 ? 0 : me; g < GPT; g += kTcMmas, d.next()) {
            const int at = me + kTcMmas * d.s;
            if (live) live = tc_wait(smem_addr(&d_empty[at]), d.ph ^ 1u);
            tc_after();
#pragma unroll
            for (int j = 0; j < 8 / GPT; ++j) {
              const int step = g * (8 / GPT) + j;  // 16 columns
              tc_mma(tmem_d + (uint32_t)(at * NB), ta + 8 * step,
                     tc_desc(sb + (step >> 2) * (L::kX / 2) + (step & 3) * 32), idesc, j != 0);
            }
            tc_commit(smem_addr(&d_full[at]));
          }
          tc_commit(smem_addr(&done[c.s]));
          last = c, any = true;
        }
      }
      // the MMAs issued end, and the commits' arrivals land, before this thread
      // leaves and the tensor memory is freed, also behind a wait that ran out
      if (any) tc_wait(smem_addr(&done[last.s]), last.ph);
    }
    __syncwarp();
  }

  if (cs > 1) {
    // one item a cluster: its CTAs' sums, a share of the rows each
    tc_cluster_sync();
    const int m0 = item0 % p.mtiles * NB, n0 = item0 / p.mtiles * kTcRows;
    const int share = (NB * kTcRows + cs - 1) / cs, i1 = min((rank + 1) * share, NB * kTcRows);
    for (int i = rank * share + tid; i < i1; i += kTcThreads) {
      const int m = m0 + i / kTcRows, n = n0 + i % kTcRows;
      if (m >= p.M || n >= p.N) continue;
      float s = 0.f;
      for (int r = 0; r < cs; ++r) s += tc_peer_f32(smem_addr(red + i), (uint32_t)r);
      w4_store(p, m, n, s);
    }
    tc_cluster_sync();  // no CTA leaves while its sums are read
  }
  tc_before();
  __syncthreads();
  if (warp == kTcMma) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// The codes' blocks: (blocks, tiles, 256 words), boxes of 8 blocks of a tile.
bool make_codes_map(CUtensorMap *map, const W4Params &p) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[3] = {256, (cuuint64_t)p.tiles, (cuuint64_t)p.blocks};
  cuuint64_t strides[2] = {1024, (cuuint64_t)p.tiles * 1024};
  cuuint32_t box[3] = {256, 1, kTcRows / M3_W4_ROWS}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<uint4 *>(p.codes), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NB, int GPT>
cudaError_t launch_tc_t(W4Params p, cudaStream_t stream, bool *taken) {
  p.mtiles = (p.M + NB - 1) / NB;
  const int64_t all = (int64_t)((p.N + kTcRows - 1) / kTcRows) * p.mtiles;
  CUtensorMap tx, tcodes;
  if (all > 0x3fffffff || !make_map(&tx, p.x, p.M, p.K, p.ldx, NB) || !make_codes_map(&tcodes, p))
    return cudaSuccess;
  *taken = true;
  const int items = (int)all, sms = sm_count_current();
  int cs = 1;
  while (p.tiles >= 12 && cs < 4 && items * cs * 2 <= sms) cs *= 2;
  const int grid = cs > 1 ? items * cs : min(items, sms);
  auto kern = w4_tc_kernel<NB, GPT>;
  static LaunchCache cache;
  if (cudaError_t e = ensure_smem_optin(cache, kern, TcSmem<NB, GPT>::kBytes); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = TcSmem<NB, GPT>::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cs;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cs > 1 ? 2 : 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tx, tcodes, p, cs, items); e != cudaSuccess) return e;
  return cudaGetLastError();
}

template <int NB>
cudaError_t launch_tc_g(const W4Params &p, int group, cudaStream_t stream, bool *taken) {
  return group == 128 ? launch_tc_t<NB, 1>(p, stream, taken)
                      : group == 64 ? launch_tc_t<NB, 2>(p, stream, taken) : launch_tc_t<NB, 4>(p, stream, taken);
}

}  // namespace

int w4_device_error(bool reset) { return device_error_of_this_unit(reset); }

cudaError_t launch_w4_tc(const W4Params &p, int group, cudaStream_t stream, bool *taken) {
  *taken = false;
  // what TMA asks of x; rows that overlap stay with the other kernels
  if (!p.x_vec || p.ldx < p.K || p.K < M3_W4_TILE) return cudaSuccess;
  return p.M <= 64 ? launch_tc_g<64>(p, group, stream, taken) : launch_tc_g<128>(p, group, stream, taken);
}

}  // namespace m3
