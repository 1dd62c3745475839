// The layers of gk_terms.cuh on dense-band graphs, on the tensor cores: gk_banded.cuh's tiles (128 nodes of one head, the band in
// blocks of 64 through two slots of shared memory) with a bias in the scores, and with two maps of scores.
//
// Heads of v have 64 features.  With two maps of 32 features a tile's q and k are the same 64 columns: either map's scores are the
// product over its half of them, so that the loads are those of one head of 64, and only the products, the element-wise stage and
// the staging tiles double.
//
// The bias is looked up: 4 bytes of bucket per edge, read once per head along 128 rows, are more than a tile's k and v, and no two
// rows begin at the same alignment.  A pass before (band_ids_kernel) lays them out as a byte per element of the tiles, in the
// order the threads of a tile read them, 255 where an element takes no part or lies outside the band; the head's column of the
// table waits in shared memory with -inf at 255, so that the masks and the band's edge need no tests.
//
// dT sums the score gradients by bucket: the destination side stores them with 16 bits of mantissa, in two planes (as bfloat16, to
// which they are rounded for the product with k, a sum of gradients of either sign was 2.4e-3 off float64, of which the stored dT's own
// rounding is 1.7e-3) in the tiles' order, and band_bucket_sum_kernel adds them up, a private table per thread.
//
// A product takes whole blocks: 0 * NaN from a row that takes no part, or that lies next to the band, reaches every row of the
// tile.  A tile that ends with a value that is not finite says so in `dirty`, and band_again_kernel does it again edge by edge.
#pragma once
#include "gk_terms_band.cuh"

namespace gk {
namespace banded {

constexpr unsigned kNoPart = 255;                 // id of an element that takes no part

struct TermsTile {
  const __nv_bfloat16 *table, *lam;          // (buckets, H * maps), (H)
  const unsigned char* ids;                  // band_ids_kernel's
  int pitch;                                 // columns of the band per tile, a multiple of 64
  int buckets;
  const int32_t *node_lo, *node_deg;         // of the owning side
  int* dirty;                                // (H, tiles): 0, kTileAgain or kTileLost
  long long n_own, n_other;
  int H;
  float scale;
  // forward
  __nv_bfloat16* o;
  float *sums, *lse;                         // (n, H, maps, 64) unrounded, may be null; (n, H, maps)
  // backward
  float2* stat;                              // (n_dst, H, maps): (lse in base-2 units, dO . o)
  unsigned short* g;                         // (H, maps, tiles, pitch / 32, 128, 32): upper halves of the score gradients
  unsigned char* g_low;                      // and the next 8 bits
  __nv_bfloat16 *out0, *out1;                // dq | dk, dv
};

// first and last column that a warp's 32 rows of a tile reach: INT_MAX and -1 where none has a neighbour
__device__ __forceinline__ void band_reduce(int lo, int deg, int part, bool writes, int* s_min, int* s_top) {
  int wmin = lo, wtop = deg > 0 ? lo + deg - 1 : -1;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    wmin = min(wmin, __shfl_xor_sync(kFull, wmin, o));
    wtop = max(wtop, __shfl_xor_sync(kFull, wtop, o));
  }
  if (writes) { s_min[part] = wmin; s_top[part] = wtop; }
}

// ids[tile][column / kC][row][column % kC], kC columns per thread of the tile's kernel.  eid: the transposed CSR's edge ids, or null.
struct BandIds {
  const int32_t *node_lo, *node_deg, *node_first, *tile_lo, *eid;
  long long n;
  int pitch, per;        // per: kC
  unsigned char* ids;
};
// A warp per row (`row` of tile `tile`), four columns per lane at a time.  Bound by its instructions (a select per element) and by the
// chain node - position - (edge id -) bucket, which every warp goes through once; with one column per lane and step, 443 instructions
// per row and the tile's first neighbour found by every block, 4.2M edges took 13 us; so they take 6.7.
__device__ __forceinline__ void band_ids_row(const BandIds& a, long long tile, int row, const int32_t* __restrict__ bucket, int buckets) {
  const int lane = threadIdx.x & 31, shift = a.per == 32 ? 5 : 4;
  const long long r = tile * kTileM + row;
  int deg = 0, lo = 0, first = 0;
  const int kmin = __ldg(a.tile_lo + tile);
  if (r < a.n) {
    deg = __ldg(a.node_deg + r);
    lo = __ldg(a.node_lo + r);
    first = __ldg(a.node_first + r);
  }
  unsigned char* out = a.ids + (size_t)tile * a.pitch * kTileM + (row << shift);
  const int skip = deg > 0 ? lo - kmin : 0;              // columns before the row's first
  const int32_t* src = a.eid ? a.eid : bucket;
  constexpr int kSteps = kSpan / 128;
  int b[kSteps][4];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int k = i * 128 + lane * 4 - skip;
    const int32_t* at = src + ((long long)first + k);    // read where the column is one of the row's alone
#pragma unroll
    for (int q = 0; q < 4; ++q) b[i][q] = (unsigned)(k + q) < (unsigned)deg ? __ldg(at + q) : -1;
  }
  if (a.eid) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (b[i][q] >= 0) b[i][q] = __ldg(bucket + b[i][q]);
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int c = i * 128 + lane * 4;
    unsigned w = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) w |= ((unsigned)b[i][q] < (unsigned)buckets ? (unsigned)b[i][q] : kNoPart) << (8 * q);
    if (c < a.pitch) *reinterpret_cast<unsigned*>(out + ((size_t)(c >> shift) << (shift + 7)) + (c & ((1 << shift) - 1))) = w;
  }
}
static __global__ void __launch_bounds__(256)
band_ids_kernel(const __grid_constant__ BandIds a, const int32_t* __restrict__ bucket, int buckets) {
  band_ids_row(a, blockIdx.x, blockIdx.y * 8 + (threadIdx.x >> 5), bucket, buckets);
}

// 16 consecutive columns of N regions of this thread's tensor-memory lane in flight together, one wait for all.  The wait names
// every destination register, so that no use of the values can be scheduled ahead of it.
__device__ __forceinline__ void tmem_ask16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_keep16(uint32_t (&r)[16]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[N][16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) tmem_keep16(r[i]);
}

// 16 values as bfloat16 into a row of a staging tile, its columns `chunk0 * 8` and up
__device__ __forceinline__ void stage16(unsigned char* row_at, int row, int chunk0, const uint32_t (&packed)[8]) {
#pragma unroll
  for (int q = 0; q < 2; ++q)
    *reinterpret_cast<uint4*>(row_at + (((chunk0 + q) ^ (row & 7)) * 16)) =
        make_uint4(packed[4 * q], packed[4 * q + 1], packed[4 * q + 2], packed[4 * q + 3]);
}
__device__ __forceinline__ void store16(__nv_bfloat16* dst, const float (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack_bf16(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
    *reinterpret_cast<uint4*>(dst + q * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// 16 floats, whole sectors: the lanes of a warp write rows far apart
__device__ __forceinline__ void store_sums16(float* dst, const float (&v)[16]) {
#pragma unroll
  for (int j = 0; j < 16; j += 8)
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + j), "f"(v[j]), "f"(v[j + 1]), "f"(v[j + 2]),
                 "f"(v[j + 3]), "f"(v[j + 4]), "f"(v[j + 5]), "f"(v[j + 6]), "f"(v[j + 7])
                 : "memory");
}
__device__ __forceinline__ bool not_finite(const float (&v)[16]) {
  float t = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) t = fmaf(v[j], 0.f, t);   // NaN as soon as one is not finite
  return t != t;
}
template <bool kBucket>
__device__ __forceinline__ void fill_table(float* s_table, const TermsTile& p, int maps, int head, int tid) {
  if constexpr (kBucket) {
    for (int i = tid; i < maps * 256; i += kThreads) {
      const int m = i >> 8, b = i & 255;
      float t = -INFINITY;
      if (b < p.buckets) t = __bfloat162float(p.table[(long long)b * p.H * maps + head * maps + m]);
      s_table[i] = t <= (float)kMaskedBias ? -INFINITY : t * (float)kLog2e;
    }
  }
}
// a score in base-2 units; a position that takes no part has none, whatever the product says
template <bool kBucket>
__device__ __forceinline__ float score_of(float s, float sl2, const float* table, unsigned id, bool inside) {
  if constexpr (kBucket) {
    const float b = table[id];
    return b == -INFINITY ? b : fmaf(s, sl2, b);
  } else {
    return inside ? s * sl2 : -INFINITY;
  }
}
__device__ __forceinline__ unsigned id_at(const uint4& w, int j) {
  const unsigned x = j < 4 ? w.x : j < 8 ? w.y : j < 12 ? w.z : w.w;
  return (x >> (8 * (j & 3))) & 255u;
}

// Two maps: the output is the difference of two sums, and probabilities rounded to bfloat16 would be the larger part of its error
// (0.0025 against 0.0017 of the rounded output alone), so that a second product adds what the rounding left off, rounded again: 16 bits
// of mantissa.  The room for it comes from k, which needs no second slot: block b + 1 is asked for at the same moment either way,
// when the scores of b are there.  One map keeps one product: three tiles share an SM.
template <int kMaps>
struct FwdLayout {
  static constexpr bool kRest = kMaps == 2;                               // probabilities in two parts
  static constexpr int kOffV = kOffK + kBandBytes;                        // of slot 0
  static constexpr int kStepK = kRest ? 0 : 2 * kBandBytes, kStepV = kRest ? kBandBytes : 2 * kBandBytes;   // from slot 0 to slot 1
  static constexpr int kOffP = kOffK + (kRest ? 3 : 4) * kBandBytes;      // a staging tile per map and part
  static constexpr int kOffBar = kOffP + (kRest ? 2 : 1) * kMaps * kBlockBytes;
  static constexpr int kOffRed = kOffBar + 128;                           // maxima, and at the end sums, of the two column groups
  static constexpr int kOffTable = kOffRed + kMaps * kColGroups * kTileM * 4;
  static constexpr int kBytes = kOffTable + kMaps * 256 * 4 + 1024;
  static constexpr int kTmem = kMaps * 128;                               // scores of every map, output of every map
  static constexpr int kCtas = kMaps == 1 ? 3 : 2;
};

// One block per (tile, head), as attention_forward_kernel, and bound like it by the chain load - product - element-wise stage - product
// behind block-wide barriers: 2 x 8192 nodes, 256 neighbours, 8 heads, a bias 61 us (issue slots 48 %, tensor pipe 11 %, three blocks
// per SM), two maps 110 us.
template <int kMaps, bool kBucket>
__global__ void __launch_bounds__(kThreads, FwdLayout<kMaps>::kCtas)
terms_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TermsTile p) {
  using L = FwdLayout<kMaps>;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  const uint32_t s_base = smem_u32(smem);
  const uint32_t bar_load = s_base + L::kOffBar, bar_s = bar_load + 8, bar_full = bar_load + 64;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffBar + 32);
  int* s_min = reinterpret_cast<int*>(smem + L::kOffBar + 40);
  int* s_top = reinterpret_cast<int*>(smem + L::kOffBar + 96);
  float* s_row = reinterpret_cast<float*>(smem + L::kOffRed);      // [map][column group][row]
  float* s_table = reinterpret_cast<float*>(smem + L::kOffTable);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quarter = warp & 3, cg = warp >> 2, row = quarter * 32 + lane;
  const int head = blockIdx.y;
  const long long r0 = (long long)blockIdx.x * kTileM, r = r0 + row;
  int lo = INT_MAX, deg = 0;
  if (r < p.n_own) {
    deg = p.node_deg[r];
    if (deg > 0) lo = p.node_lo[r];
  }
  band_reduce(lo, deg, quarter, lane == 0 && cg == 0, s_min, s_top);
  fill_table<kBucket>(s_table, p, kMaps, head, tid);
  if (tid == 0) {
    mbar_init(bar_load, 1);
    mbar_init(bar_s, 1);
#pragma unroll
    for (int b = 0; b < kSlots; ++b) mbar_init(bar_full + 8 * b, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::kTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int kmin = min(min(s_min[0], s_min[1]), min(s_min[2], s_min[3]));
  bool bad = false;

  if (kmin != INT_MAX) {
    const int ktop = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
    int nb = (ktop - kmin) / kKeys + 1;
    nb = nb < p.pitch / kKeys ? nb : p.pitch / kKeys;
    auto issue_band = [&](int b) {   // one thread
      const uint32_t bar = bar_full + 8 * (b & 1);
      mbar_expect_tx(bar, (uint32_t)(2 * kBandBytes));
      tma_load_3d(s_base + kOffK + (b & 1) * L::kStepK, &map_k, bar, 0, head, kmin + b * kKeys);
      tma_load_3d(s_base + L::kOffV + (b & 1) * L::kStepV, &map_v, bar, 0, head, kmin + b * kKeys);
    };
    constexpr int kSteps = kD / kMaps / 16;   // of 16 features, per map
    auto issue_scores = [&](int b) {   // one thread
      constexpr uint32_t idesc = umma_idesc(kTileM, kKeys, false);
      const uint32_t at = s_base + kOffK + (b & 1) * L::kStepK;
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk)
        umma_f16(tmem + (kk / kSteps) * kKeys, umma_desc(s_base + kOffQ + kk * 32, 16, 1024), umma_desc(at + kk * 32, 16, 1024), idesc,
                 kk % kSteps > 0);
    };
    if (tid == 0) {
      mbar_expect_tx(bar_load, (uint32_t)kBlockBytes);
      tma_load_3d(s_base + kOffQ, &map_q, bar_load, 0, head, (int)r0);
      tma_load_3d(s_base + kOffQ + kBandBytes, &map_q, bar_load, 0, head, (int)r0 + kKeys);
      issue_band(0);
      if (!L::kRest && nb > 1) issue_band(1);
    }
    int issued = L::kRest || nb < kSlots ? 1 : kSlots;
    bool ok = __syncthreads_and(mbar_wait(bar_load, 0) && mbar_wait(bar_full, 0));

    const int jlo = deg > 0 ? lo - kmin : 1, jhi = deg > 0 ? lo - kmin + deg - 1 : 0;   // this row's columns of the band
    int wlo = deg > 0 ? jlo : INT_MAX, whi = deg > 0 ? jhi : -1;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      wlo = min(wlo, __shfl_xor_sync(kFull, wlo, o));
      whi = max(whi, __shfl_xor_sync(kFull, whi, o));
    }
    const uint32_t row_taddr = tmem + ((uint32_t)(quarter * 32) << 16);
    const float sl2 = p.scale * (float)kLog2e;
    unsigned char* prow = smem + L::kOffP + row * kRowBytes;
    const unsigned char* id_row = kBucket ? p.ids + (size_t)blockIdx.x * p.pitch * kTileM + row * 32 : nullptr;
    float mx[kMaps], l[kMaps];   // a map's reference maximum, in both of the row's threads; this thread's part of the sum
#pragma unroll
    for (int m = 0; m < kMaps; ++m) { mx[m] = -INFINITY; l[m] = 0.f; }

    if (ok && tid == 0) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      issue_scores(0);
      umma_commit(bar_s);
    }
    // per block one wait, as in attention_forward_kernel
    for (int b = 0; b < nb; ++b) {
      const int col0 = b * kKeys + cg * 32;
      uint4 id[2];
      if constexpr (kBucket) {
        const uint4* src = reinterpret_cast<const uint4*>(id_row + (size_t)(2 * b + cg) * 32 * kTileM);
        id[0] = __ldg(src);
        id[1] = __ldg(src + 1);
      }
      ok = __syncthreads_and(ok && mbar_wait(bar_s, b & 1));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (ok && (b > 0 || L::kRest) && b + 1 < nb) {   // block b - 1's slot is free, and where k has one alone, b's too
        if (tid == 0) issue_band(b + 1);
        issued = b + 2;
      }
      const bool live = ok && col0 <= whi && col0 + 31 >= wlo;   // warp-uniform
      float x[kMaps][32];
#pragma unroll
      for (int m = 0; m < kMaps; ++m) {
        float top = -INFINITY;
        if (live) {
          tmem_ld32(row_taddr + m * kKeys + cg * 32, x[m]);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            x[m][j] = score_of<kBucket>(x[m][j], sl2, s_table + m * 256, kBucket ? id_at(id[j >> 4], j & 15) : 0u,
                                        col0 + j >= jlo && col0 + j <= jhi);
            top = fmaxf(top, x[m][j]);
          }
        }
        s_row[(m * kColGroups + cg) * kTileM + row] = top;
      }
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");   // the two warps of these rows
#pragma unroll
      for (int m = 0; m < kMaps; ++m) {
        const float top = fmaxf(s_row[(m * kColGroups) * kTileM + row], s_row[(m * kColGroups + 1) * kTileM + row]);
        // A reference that lags behind the maximum by up to 2^8 serves as well: the rounding is relative.
        const bool grows = top > mx[m] + 8.f || (mx[m] == -INFINITY && top > -INFINITY);
        const float corr = !grows ? 1.f : mx[m] == -INFINITY ? 0.f : exp2_fast(mx[m] - top);
        if (grows) {
          mx[m] = top;
          l[m] *= corr;
        }
        if (b > 0 && __any_sync(kFull, grows)) {
          float o[32];
          tmem_ld32(row_taddr + (kMaps + m) * kKeys + cg * 32, o);
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] *= corr;
          tmem_st32(row_taddr + (kMaps + m) * kKeys + cg * 32, o);
        }
        const float ref = mx[m] == -INFINITY ? 0.f : mx[m];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t packed[8], rest[8];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            float p0 = 0.f, p1 = 0.f;
            if (live) {
              p0 = exp2_fast(x[m][16 * half + j] - ref);
              p1 = exp2_fast(x[m][16 * half + j + 1] - ref);
              l[m] += p0 + p1;
            }
            packed[j / 2] = pack_bf16(p0, p1);
            if constexpr (L::kRest)
              rest[j / 2] = pack_bf16(p0 - __uint_as_float(packed[j / 2] << 16), p1 - __uint_as_float(packed[j / 2] & 0xffff0000u));
          }
          stage16(prow + m * kBlockBytes, row, cg * 4 + 2 * half, packed);
          if constexpr (L::kRest) stage16(prow + (kMaps + m) * kBlockBytes, row, cg * 4 + 2 * half, rest);
        }
      }
      // the probabilities were written through the generic proxy; the tensor core reads through the async proxy
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      ok = __syncthreads_and(ok && (b + 1 >= nb || mbar_wait(bar_full + 8 * ((b + 1) & 1), ((b + 1) >> 1) & 1)));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (ok && tid == 0) {
        constexpr uint32_t idesc = umma_idesc(kTileM, kD, true);
        const uint32_t at = s_base + L::kOffV + (b & 1) * L::kStepV;
#pragma unroll
        for (int part = 0; part < (L::kRest ? 2 : 1); ++part)
#pragma unroll
          for (int m = 0; m < kMaps; ++m)
#pragma unroll
            for (int ks = 0; ks < kKeys / 16; ++ks)
              umma_f16(tmem + (kMaps + m) * kKeys, umma_desc(s_base + L::kOffP + (part * kMaps + m) * kBlockBytes + ks * 32, 16, 1024),
                       umma_desc(at + ks * 16 * kRowBytes, 16, 1024), idesc, (part | b | ks) != 0);
        if (b + 1 < nb) issue_scores(b + 1);
        umma_commit(bar_s);
      }
    }
#pragma unroll
    for (int m = 0; m < kMaps; ++m) s_row[(m * kColGroups + cg) * kTileM + row] = l[m];
    ok = __syncthreads_and(ok && mbar_wait(bar_s, nb & 1));   // the last block's output product
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float inv[kMaps];
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      l[m] = s_row[(m * kColGroups) * kTileM + row] + s_row[(m * kColGroups + 1) * kTileM + row];
      inv[m] = l[m] == 0.f ? 0.f : 1.f / l[m];
    }
    const float lam = kMaps == 2 ? __bfloat162float(p.lam[head]) : 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {   // this thread's 32 of the row's 64 output features
      const int f0 = cg * 32 + half * 16;
      float out[16];
#pragma unroll
      for (int m = 0; m < kMaps; ++m) {
        float o[16];
        if (ok) tmem_ld16(row_taddr + (kMaps + m) * kKeys + f0, o);   // warp-wide, whether or not the lane's row exists
        bad = bad || (r < p.n_own && ok && not_finite(o));
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          o[j] = !ok ? NAN : l[m] == 0.f ? 0.f : o[j] * inv[m];
          out[j] = m == 0 ? o[j] : fmaf(-lam, o[j], out[j]);
        }
        if (p.sums && r < p.n_own) {
          store_sums16(p.sums + (((long long)r * p.H + head) * kMaps + m) * kD + f0, o);
        }
      }
      if (r < p.n_own) store16(p.o + ((long long)r * p.H + head) * kD + f0, out);
    }
    if (r < p.n_own && cg == 0)
#pragma unroll
      for (int m = 0; m < kMaps; ++m)
        p.lse[((long long)r * p.H + head) * kMaps + m] = !ok ? NAN : (mx[m] + log2f(l[m])) * (float)kLn2;   // -inf where nothing took part
    if (!ok) {   // a wait ran out: loads asked for are given (bounded) time to land before the shared memory is handed back
      mbar_wait(bar_load, 0);
      for (int b = issued > kSlots ? issued - kSlots : 0; b < issued; ++b) mbar_wait(bar_full + 8 * (b & 1), (b >> 1) & 1);
    }
  } else if (r < p.n_own && cg == 0) {   // no node of the tile has a neighbour
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < kD / 8; ++q) {
      *reinterpret_cast<uint4*>(p.o + ((long long)r * p.H + head) * kD + q * 8) = zero;
    }
    if (p.sums)
      for (int q = 0; q < kMaps * kD / 4; ++q) *reinterpret_cast<uint4*>(p.sums + ((long long)r * p.H + head) * kMaps * kD + q * 4) = zero;
#pragma unroll
    for (int m = 0; m < kMaps; ++m) p.lse[((long long)r * p.H + head) * kMaps + m] = -INFINITY;
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  bad = __syncthreads_or(bad);
  if (tid == 0) p.dirty[(size_t)head * gridDim.x + blockIdx.x] = bad ? kTileAgain : 0;
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmem) : "memory");
}

// ---------------------------------------------------------------------------------------------------------
// Backward, a kernel per side as attention_backward_kernel.  The source side of two maps takes blocks of 32 queries: scores and dP of
// 64 would leave no room in half of the tensor memory for dk and dv, and two tiles share an SM.
// ---------------------------------------------------------------------------------------------------------
template <bool kSrc, int kMaps>
struct BwdLayout {
  static constexpr int kB = kSrc && kMaps == 2 ? 32 : 64;             // columns of a block
  static constexpr int kC = kB / 2;                                   // of a thread
  static constexpr int kSlot = 2 * kB * kRowBytes;
  static constexpr int kStages = kSrc ? 1 + kMaps : kMaps;            // weights (source side), then g of every map
  static constexpr int kTmem = 256;
  static constexpr int kOffA = 0, kOffB = kBlockBytes, kOffC = 2 * kBlockBytes;   // owned tiles, slots of the band
  static constexpr int kOffStage = kOffC + kSlots * kSlot;
  static constexpr int kOffBar = kOffStage + kStages * kBlockBytes;
  static constexpr int kOffStat = kOffBar + 128;
  static constexpr int kStatBytes = kSrc ? kSpan * kMaps * 8 : 0;
  static constexpr int kOffTable = kOffStat + kStatBytes;
  static constexpr int kBytes = kOffTable + kMaps * 256 * 4 + 1024;
  // tensor memory: scores of every map, dP, then dq | dk, dv
  static constexpr int kColP = kMaps * kB, kColG0 = (kMaps + 1) * kB, kColG1 = kColG0 + kD;
  static_assert(kColG0 + (kSrc ? 2 : 1) * kD <= kTmem, "half of the tensor memory");
};

template <bool kSrc, int kMaps, bool kBucket>
__device__ __forceinline__ void terms_backward_tile(const CUtensorMap& map_a, const CUtensorMap& map_b, const CUtensorMap& map_c,
                                                    const CUtensorMap& map_d, const TermsTile& p, unsigned tiles) {
  using L = BwdLayout<kSrc, kMaps>;
  constexpr int kB = L::kB, kC = L::kC;
  extern __shared__ unsigned char raw_smem[];
  unsigned char* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  const uint32_t s_base = smem_u32(smem);
  const uint32_t bar_load = s_base + L::kOffBar, bar_s = bar_load + 8, bar_g = bar_load + 16, bar_full = bar_load + 64;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffBar + 32);
  int* s_min = reinterpret_cast<int*>(smem + L::kOffBar + 40);
  int* s_top = reinterpret_cast<int*>(smem + L::kOffBar + 96);
  float2* s_stat = reinterpret_cast<float2*>(smem + L::kOffStat);   // source side: [query][map]
  float* s_table = reinterpret_cast<float*>(smem + L::kOffTable);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quarter = warp & 3, cg = warp >> 2, row = quarter * 32 + lane;
  const int head = blockIdx.y;
  const long long r0 = (long long)blockIdx.x * kTileM, r = r0 + row;
  int lo = INT_MAX, deg = 0;
  if (r < p.n_own) {
    deg = p.node_deg[r];
    if (deg > 0) lo = p.node_lo[r];
  }
  band_reduce(lo, deg, quarter, lane == 0 && cg == 0, s_min, s_top);
  fill_table<kBucket>(s_table, p, kMaps, head, tid);
  if (tid == 0) {
    mbar_init(bar_load, 1);
    mbar_init(bar_s, 1);
    mbar_init(bar_g, 1);
#pragma unroll
    for (int b = 0; b < kSlots; ++b) mbar_init(bar_full + 8 * b, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::kTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int bmin = min(min(s_min[0], s_min[1]), min(s_min[2], s_min[3]));
  bool ok = true, bad = false;
  const long long cell = ((long long)r * p.H + head) * kMaps;   // of this row's statistics

  if (bmin != INT_MAX) {
    const int btop = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
    int nb = (btop - bmin) / kB + 1;
    nb = nb < p.pitch / kB ? nb : p.pitch / kB;
    auto issue_band = [&](int b) {   // one thread
      const uint32_t bar = bar_full + 8 * (b & 1), at = s_base + L::kOffC + (b & 1) * L::kSlot;
      mbar_expect_tx(bar, (uint32_t)L::kSlot);
      tma_load_3d(at, &map_c, bar, 0, head, bmin + b * kB);
      tma_load_3d(at + L::kSlot / 2, &map_d, bar, 0, head, bmin + b * kB);
    };
    if (tid == 0) {
      mbar_expect_tx(bar_load, (uint32_t)(kBlockBytes * 2));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        tma_load_3d(s_base + L::kOffA + half * kBandBytes, &map_a, bar_load, 0, head, (int)r0 + half * kKeys);
        tma_load_3d(s_base + L::kOffB + half * kBandBytes, &map_b, bar_load, 0, head, (int)r0 + half * kKeys);
      }
      issue_band(0);
      if (nb > 1) issue_band(1);
    }
    int issued = nb < kSlots ? nb : kSlots;
    // the rows' statistics while the tiles travel; column j of the source side's scores is query bmin + j
    float lse2[kMaps], delta[kMaps];
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
      const float2 st = !kSrc && r < p.n_own ? p.stat[cell + m] : make_float2(INFINITY, 0.f);
      lse2[m] = st.x;
      delta[m] = st.y;
    }
    if constexpr (kSrc) {
      for (int i = tid; i < nb * kB * kMaps; i += kThreads) {
        const long long qn = (long long)bmin + i / kMaps;
        s_stat[i] = qn < p.n_other ? p.stat[(qn * p.H + head) * kMaps + i % kMaps] : make_float2(INFINITY, 0.f);
      }
    }
    ok = __syncthreads_and(mbar_wait(bar_load, 0) && mbar_wait(bar_full, 0));

    const int jlo = deg > 0 ? lo - bmin : 1, jhi = deg > 0 ? lo - bmin + deg - 1 : 0;
    int wlo = deg > 0 ? jlo : INT_MAX, whi = deg > 0 ? jhi : -1;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      wlo = min(wlo, __shfl_xor_sync(kFull, wlo, o));
      whi = max(whi, __shfl_xor_sync(kFull, whi, o));
    }
    const uint32_t row_taddr = tmem + ((uint32_t)(quarter * 32) << 16);
    const float sl2 = p.scale * (float)kLog2e;
    const float lam = kMaps == 2 ? __bfloat162float(p.lam[head]) : 0.f;
    unsigned char* stage = smem + L::kOffStage + row * kRowBytes;
    const size_t tile_at = (size_t)blockIdx.x * p.pitch * kTileM;
    const unsigned char* id_row = kBucket ? p.ids + tile_at + row * kC : nullptr;

    constexpr int kSteps = kD / kMaps / 16;
    auto issue_scores = [&](int b) {   // one thread: owned operands x the band's block
      constexpr uint32_t idesc = umma_idesc(kTileM, kB, false);
      const uint32_t at = s_base + L::kOffC + (b & 1) * L::kSlot;
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk)
        umma_f16(tmem + (kk / kSteps) * kB, umma_desc(s_base + L::kOffA + kk * 32, 16, 1024), umma_desc(at + kk * 32, 16, 1024), idesc,
                 kk % kSteps > 0);
#pragma unroll
      for (int kk = 0; kk < kD / 16; ++kk)   // dP
        umma_f16(tmem + L::kColP, umma_desc(s_base + L::kOffB + kk * 32, 16, 1024), umma_desc(at + L::kSlot / 2 + kk * 32, 16, 1024), idesc,
                 kk > 0);
    };
    if (ok && tid == 0) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      issue_scores(0);
      umma_commit(bar_s);
    }
    // per block one wait, as in attention_backward_kernel
    for (int b = 0; b < nb; ++b) {
      const int col0 = b * kB + cg * kC;
      uint4 id[kC / 16];
      if constexpr (kBucket) {
        const uint4* src = reinterpret_cast<const uint4*>(id_row + (size_t)(2 * b + cg) * kC * kTileM);
#pragma unroll
        for (int q = 0; q < kC / 16; ++q) id[q] = __ldg(src + q);
      }
      ok = __syncthreads_and(ok && mbar_wait(bar_s, b & 1));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (ok && b > 0 && b + 1 < nb) {   // block b - 1's slot is free: its gradient products were before block b's scores
        if (tid == 0) issue_band(b + 1);
        issued = b + 2;
      }
      const bool live = ok && col0 <= whi && col0 + kC - 1 >= wlo;   // warp-uniform
#pragma unroll
      for (int half = 0; half < kC / 16; ++half) {
        uint32_t pw[8], pg[kMaps][8];
        [[maybe_unused]] uint32_t up[kMaps][8], low[kMaps][4];
        if (live) {
          uint32_t raw[kMaps + 1][16];
#pragma unroll
          for (int m = 0; m < kMaps; ++m) tmem_ask16(row_taddr + m * kB + cg * kC + half * 16, raw[m]);
          tmem_ask16(row_taddr + L::kColP + cg * kC + half * 16, raw[kMaps]);
          tmem_wait16(raw);
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            float w[2], g[kMaps][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = col0 + half * 16 + j + e;
              const unsigned ident = kBucket ? id_at(id[half], j + e) : 0u;
              w[e] = 0.f;
#pragma unroll
              for (int m = 0; m < kMaps; ++m) {
                const float2 st = kSrc ? s_stat[col * kMaps + m] : make_float2(lse2[m], delta[m]);
                const float b = kBucket ? s_table[m * 256 + ident] : 0.f;
                const bool part = kBucket ? b != -INFINITY : col >= jlo && col <= jhi;   // not by the score: st.x may be NaN
                const float pr = part ? exp2_fast(fmaf(__uint_as_float(raw[m][j + e]), sl2, b) - st.x) * (m == 0 ? 1.f : -lam) : 0.f;
                w[e] += pr;
                const float gr = pr * (__uint_as_float(raw[kMaps][j + e]) - st.y);
                g[m][e] = pr == 0.f ? 0.f : gr;   // dP of a position that takes no part may be anything
              }
            }
            if constexpr (kSrc) pw[j / 2] = pack_bf16(w[0], w[1]);
#pragma unroll
            for (int m = 0; m < kMaps; ++m) pg[m][j / 2] = pack_bf16(g[m][0], g[m][1]);
            if constexpr (kBucket && !kSrc) {   // bits 31-16 and 15-8 of both, the latter four elements to a word
#pragma unroll
              for (int m = 0; m < kMaps; ++m) {
                const uint32_t x = __float_as_uint(g[m][0]), y = __float_as_uint(g[m][1]);
                up[m][j / 2] = __byte_perm(x, y, 0x7632);
                const uint32_t two = __byte_perm(x, y, 0x0051);
                if (j & 2) low[m][j / 4] |= two << 16;
                else low[m][j / 4] = two & 0xffffu;
              }
            }
          }
          if constexpr (kBucket && !kSrc) {
#pragma unroll
            for (int m = 0; m < kMaps; ++m) {
              const size_t to = (size_t)(head * kMaps + m) * tiles * p.pitch * kTileM + tile_at + (size_t)(2 * b + cg) * kC * kTileM + row * kC + half * 16;
              uint4* at = reinterpret_cast<uint4*>(p.g + to);
              at[0] = make_uint4(up[m][0], up[m][1], up[m][2], up[m][3]);
              at[1] = make_uint4(up[m][4], up[m][5], up[m][6], up[m][7]);
              *reinterpret_cast<uint4*>(p.g_low + to) = make_uint4(low[m][0], low[m][1], low[m][2], low[m][3]);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            pw[j] = 0u;
#pragma unroll
            for (int m = 0; m < kMaps; ++m) pg[m][j] = 0u;
          }
        }
        const int chunk = cg * (kC / 8) + 2 * half;
        if constexpr (kSrc) stage16(stage, row, chunk, pw);
#pragma unroll
        for (int m = 0; m < kMaps; ++m) stage16(stage + ((kSrc ? 1 : 0) + m) * kBlockBytes, row, chunk, pg[m]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      // the staging tiles are written by all, and the next block of the band has landed
      ok = __syncthreads_and(ok && (b + 1 >= nb || mbar_wait(bar_full + 8 * ((b + 1) & 1), ((b + 1) >> 1) & 1)));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (ok && tid == 0) {
        const uint32_t at = s_base + L::kOffC + (b & 1) * L::kSlot;
#pragma unroll
        for (int ks = 0; ks < kB / 16; ++ks) {
          const uint32_t rows = ks * 16 * kRowBytes;
          if constexpr (kSrc)   // dv += W^T dO_b
            umma_f16(tmem + L::kColG1, umma_desc(s_base + L::kOffStage + ks * 32, 16, 1024), umma_desc(at + L::kSlot / 2 + rows, 16, 1024),
                     umma_idesc(kTileM, kD, true), (b | ks) != 0);
#pragma unroll
          for (int m = 0; m < kMaps; ++m)   // dq += g k_b | dk += g^T q_b: a map's features are its part of the 64 columns
            umma_f16(tmem + L::kColG0 + m * (kD / kMaps),
                     umma_desc(s_base + L::kOffStage + ((kSrc ? 1 : 0) + m) * kBlockBytes + ks * 32, 16, 1024),
                     umma_desc(at + rows + m * (kRowBytes / kMaps), 16, 1024), umma_idesc(kTileM, kD / kMaps, true), (b | ks) != 0);
        }
        if (b + 1 < nb) {
          issue_scores(b + 1);
          umma_commit(bar_s);
        } else {
          umma_commit(bar_g);
        }
      }
    }
    ok = __syncthreads_and(ok && mbar_wait(bar_g, 0));   // the last block's gradient products
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");

#pragma unroll
    for (int half = 0; half < 2; ++half) {   // gradients of the owned rows: this thread's 32 of the 64 features
      const int f0 = cg * 32 + half * 16;
      const long long at = ((long long)r * p.H + head) * kD + f0;
#pragma unroll
      for (int w = 0; w < (kSrc ? 2 : 1); ++w) {
        float v[16];
        if (ok) tmem_ld16(row_taddr + (w == 0 ? L::kColG0 : L::kColG1) + f0, v);
        bad = bad || (r < p.n_own && ok && not_finite(v));
        if (r < p.n_own) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = !ok ? NAN : deg == 0 ? 0.f : w == 0 ? v[j] * p.scale : v[j];
          store16((w == 0 ? p.out0 : p.out1) + at, v);
        }
      }
    }
    if (!ok) {   // a wait ran out: loads asked for are given (bounded) time to land before the shared memory is handed back
      mbar_wait(bar_load, 0);
      for (int b = issued > kSlots ? issued - kSlots : 0; b < issued; ++b) mbar_wait(bar_full + 8 * (b & 1), (b >> 1) & 1);
    }
  } else if (r < p.n_own && cg == 0) {  // no owned node of the tile has a neighbour: zero gradients
    const long long at = ((long long)r * p.H + head) * kD;
#pragma unroll
    for (int q = 0; q < kD / 8; ++q) {
      *reinterpret_cast<uint4*>(p.out0 + at + q * 8) = make_uint4(0, 0, 0, 0);
      if constexpr (kSrc) *reinterpret_cast<uint4*>(p.out1 + at + q * 8) = make_uint4(0, 0, 0, 0);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  bad = __syncthreads_or(bad);
  if (tid == 0) p.dirty[(size_t)head * tiles + blockIdx.x] = !ok ? kTileLost : bad ? kTileAgain : 0;
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmem) : "memory");
}

// Both sides in one launch, the destination's tiles first: 1024 tiles two to an SM are 3.5 rounds of the chip, which take the time of
// four; twice as many are seven (2 x 8192 nodes, 8 heads: 78 + 82 us apart, 142 together with 24-bit score gradients; two maps without
// a bias 175).
template <int kMaps, bool kBucket>
__global__ void __launch_bounds__(kThreads, 2)
terms_backward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                      const __grid_constant__ CUtensorMap band_q, const __grid_constant__ CUtensorMap band_g,
                      const __grid_constant__ TermsTile dst, const __grid_constant__ TermsTile src, const unsigned tiles_dst,
                      const unsigned tiles_src) {
  if (blockIdx.z == 0) {
    if (blockIdx.x < tiles_dst) terms_backward_tile<false, kMaps, kBucket>(map_q, map_g, map_k, map_v, dst, tiles_dst);
  } else {
    if (blockIdx.x < tiles_src) terms_backward_tile<true, kMaps, kBucket>(map_k, map_v, band_q, band_g, src, tiles_src);
  }
}

// What the tiles need before they begin, in one launch: the ids of both orientations (blockIdx.z 0 and 1, with kBucket alone), and (lse in
// base-2 units, dO . o) of every node and map, with dO . o2 for dlam, eight lanes per node and head.  A row of which nothing took part
// has no probabilities, whatever dO holds.
template <int kMaps, bool kBucket>
__global__ void __launch_bounds__(256)
band_prepare_kernel(const __grid_constant__ BandIds a0, const __grid_constant__ BandIds a1, const int32_t* __restrict__ bucket, int buckets,
                    const float* __restrict__ sums, const __nv_bfloat16* __restrict__ d_o, const float* __restrict__ lse, long long cells,
                    float2* __restrict__ stat, float* __restrict__ t2) {
  if constexpr (kBucket) {
    if (blockIdx.z < 2) {
      const BandIds& a = blockIdx.z ? a1 : a0;
      if ((long long)blockIdx.x * kTileM < a.n) band_ids_row(a, blockIdx.x, blockIdx.y * 8 + (threadIdx.x >> 5), bucket, buckets);
      return;
    }
  }
  const int part = threadIdx.x & 7;
  const long long stride = (long long)gridDim.x * gridDim.y * 32;
  for (long long i0 = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * 32; i0 < cells; i0 += stride) {
    const long long i = i0 + (threadIdx.x >> 3);
    const bool in = i < cells;
    float d[kMaps];
#pragma unroll
    for (int m = 0; m < kMaps; ++m) d[m] = 0.f;
    if (in) {
      const uint4 gv = __ldg(reinterpret_cast<const uint4*>(d_o + i * kD) + part);
      const __nv_bfloat162* g2 = reinterpret_cast<const __nv_bfloat162*>(&gv);
#pragma unroll
      for (int m = 0; m < kMaps; ++m) {
        const float4* at = reinterpret_cast<const float4*>(sums + (i * kMaps + m) * kD) + 2 * part;
        const float4 x = __ldg(at), y = __ldg(at + 1);
        const float of[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 gf = __bfloat1622float2(g2[e]);
          d[m] += of[2 * e] * gf.x + of[2 * e + 1] * gf.y;
        }
      }
    }
#pragma unroll
    for (int m = 0; m < kMaps; ++m) {
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) d[m] += __shfl_xor_sync(kFull, d[m], o);
      if (in && part == 0) {
        const float l = lse[i * kMaps + m];
        const bool none = l == -INFINITY;
        if (none) d[m] = 0.f;
        stat[i * kMaps + m] = make_float2(none ? INFINITY : l * (float)kLog2e, d[m]);
        if (m == 1) t2[i] = d[m];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// tiles done again, edge by edge: kSide 0 forward, 1 destination side (dq), 2 source side (dk, dv)
// ---------------------------------------------------------------------------------------------------------
struct AgainArgs {
  TermsTile t;
  const __nv_bfloat16 *q, *k, *v, *d_o;
  const int32_t *node_first, *eid, *bucket;
  int tiles;
};
// A warp per dirty tile and head; a lane has two of the 64 features, with two maps the first 16 lanes map 0's.
template <int kSide, int kMaps, bool kBucket>
__global__ void __launch_bounds__(256) band_again_kernel(const __grid_constant__ AgainArgs a) {
  const int lane = threadIdx.x & 31, mine = kMaps == 2 ? lane >> 4 : 0;
  const TermsTile& t = a.t;
  const int warps = gridDim.x * 8, total = a.tiles * t.H;
  const float sl2 = t.scale * (float)kLog2e;
  const auto two = [&](const __nv_bfloat16* x, long long n, int head) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(x + (n * t.H + head) * kD + 2 * lane));
  };
  const auto put = [&](__nv_bfloat16* x, long long at, float u, float v) {
    *reinterpret_cast<__nv_bfloat162*>(x + at * kD + 2 * lane) = __floats2bfloat162_rn(u, v);
  };
  for (int f = blockIdx.x * 8 + (threadIdx.x >> 5); f < total; f += warps) {
    if (t.dirty[f] != kTileAgain) continue;
    const int head = f / a.tiles;
    const long long r0 = (long long)(f - head * a.tiles) * kTileM;
    const float lam = kMaps == 2 ? __bfloat162float(t.lam[head]) : 0.f;
    for (int i = 0; i < kTileM && r0 + i < t.n_own; ++i) {
      const long long r = r0 + i, at = r * t.H + head;
      const int deg = t.node_deg[r], lo = deg ? t.node_lo[r] : 0, first = deg ? a.node_first[r] : 0;
      float2 x = two(kSide == 2 ? a.k : a.q, r, head);
      x.x *= sl2; x.y *= sl2;
      const float2 y = kSide == 0 ? make_float2(0.f, 0.f) : two(kSide == 2 ? a.v : a.d_o, r, head);
      float mx[kMaps], l[kMaps], acc[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int m = 0; m < kMaps; ++m) { mx[m] = -INFINITY; l[m] = 0.f; }
      for (int j = 0; j < deg; ++j) {
        float bias[kMaps];
        bool any = false;
#pragma unroll
        for (int m = 0; m < kMaps; ++m) {
          bias[m] = 0.f;
          if constexpr (kBucket) {
            const unsigned b = (unsigned)a.bucket[a.eid ? a.eid[first + j] : first + j];
            bias[m] = b < (unsigned)t.buckets ? __bfloat162float(t.table[(long long)b * t.H * kMaps + head * kMaps + m]) : -INFINITY;
            bias[m] = bias[m] <= (float)kMaskedBias ? -INFINITY : bias[m] * (float)kLog2e;
          }
          any = any || bias[m] > -INFINITY || bias[m] != bias[m];
        }
        if (!any) continue;
        const long long c = (long long)lo + j;
        const float2 z = two(kSide == 2 ? a.q : a.k, c, head);
        float s = x.x * z.x + x.y * z.y, dp = 0.f;
#pragma unroll
        for (int o = 1; o < (kMaps == 2 ? 16 : 32); o <<= 1) s += __shfl_xor_sync(kFull, s, o);
        const float2 u = two(kSide == 2 ? a.d_o : a.v, c, head);
        if constexpr (kSide != 0) {
          dp = y.x * u.x + y.y * u.y;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) dp += __shfl_xor_sync(kFull, dp, o);
        }
        float w = 0.f, own = 0.f;
#pragma unroll
        for (int m = 0; m < kMaps; ++m) {
          const float sm = bias[m] == -INFINITY ? bias[m] : (kMaps == 2 ? __shfl_sync(kFull, s, m * 16) : s) + bias[m];
          if constexpr (kSide == 0) {
            const float mn = fmaxf(mx[m], sm), ref = mn == -INFINITY ? 0.f : mn;
            const float corr = mx[m] == mn ? 1.f : exp2_fast(mx[m] - mn), pr = sm == -INFINITY ? 0.f : exp2_fast(sm - ref);
            mx[m] = mn;
            l[m] = l[m] * corr + pr;
            acc[m][0] *= corr; acc[m][1] *= corr;
            if (pr != 0.f) { acc[m][0] = fmaf(pr, u.x, acc[m][0]); acc[m][1] = fmaf(pr, u.y, acc[m][1]); }
          } else {
            const float2 st = t.stat[((kSide == 2 ? c : r) * t.H + head) * kMaps + m];
            const float pr = bias[m] == -INFINITY ? 0.f : exp2_fast(sm - st.x) * (m == 0 ? 1.f : -lam);
            const float g = pr == 0.f ? 0.f : pr * (dp - st.y);
            w += pr;
            if (m == mine) own = g;
          }
        }
        if constexpr (kSide != 0) {
          if (own != 0.f) { acc[0][0] = fmaf(own, z.x, acc[0][0]); acc[0][1] = fmaf(own, z.y, acc[0][1]); }
          if (kSide == 2 && w != 0.f) { acc[1][0] = fmaf(w, u.x, acc[1][0]); acc[1][1] = fmaf(w, u.y, acc[1][1]); }
        }
      }
      if constexpr (kSide == 0) {
        float o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int m = 0; m < kMaps; ++m) {
          const float inv = l[m] == 0.f ? 0.f : 1.f / l[m], e0 = acc[m][0] * inv, e1 = acc[m][1] * inv, cm = m == 0 ? 1.f : -lam;
          if (t.sums) *reinterpret_cast<float2*>(t.sums + (at * kMaps + m) * kD + 2 * lane) = make_float2(e0, e1);
          o0 = fmaf(cm, e0, o0);
          o1 = fmaf(cm, e1, o1);
          if (lane == 0) t.lse[at * kMaps + m] = (mx[m] + log2f(l[m])) * (float)kLn2;
        }
        put(t.o, at, o0, o1);
      } else {
        put(t.out0, at, acc[0][0] * t.scale, acc[0][1] * t.scale);
        if constexpr (kSide == 2) put(t.out1, at, acc[1][0], acc[1][1]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------------------
inline BandIds band_ids_of(const graphop_plan_t* plan, const int32_t* eid, long long n, int per, unsigned char* ids) {
  return BandIds{plan->node_lo, plan->node_deg, plan->node_first, plan->tile_lo, eid, n, band_pitch(plan), per, ids};
}
template <int kSide, int kMaps, bool kBucket>
inline int run_band_again(const AgainArgs& a, cudaStream_t st) {
  const int warps = a.tiles * a.t.H;
  band_again_kernel<kSide, kMaps, kBucket><<<warps < 148 * 8 ? (warps + 7) / 8 : 148, 256, 0, st>>>(a);
  GK_LAUNCHED("band_again");
  return GRAPHOP_OK;
}

template <int kMaps, bool kBucket>
inline int terms_forward(const graphop_plan_t* plan, const TermsCall<__nv_bfloat16>& c, __nv_bfloat16* o, void* sums, void* lse,
                         Arena& ar, cudaStream_t st) {
  using L = FwdLayout<kMaps>;
  const int pitch = band_pitch(plan);
  const long long tiles = band_tiles_of(c.n_dst);
  const BandRoom room = band_room_forward(ar, plan, c.n_dst, c.H, c.buckets);
  TermsTile t{};
  t.ids = room.ids;
  t.dirty = room.dirty;
  if (ar.overflow) return GRAPHOP_ERR_UNSUPPORTED;
  CUtensorMap mq, mk, mv;
  if (!make_map(&mq, c.q, c.n_dst, c.H) || !make_map(&mk, c.k, c.n_src, c.H) || !make_map(&mv, c.v, c.n_src, c.H))
    return GRAPHOP_ERR_UNSUPPORTED;
  static std::atomic<bool> configured[64];
  GK_TRY(allow_smem(terms_forward_kernel<kMaps, kBucket>, L::kBytes, configured));
  if (kBucket) {
    band_ids_kernel<<<dim3((unsigned)tiles, kTileM / 8), 256, 0, st>>>(
        band_ids_of(plan, nullptr, c.n_dst, 32, room.ids), c.bucket, c.buckets);
    GK_LAUNCHED("band_ids");
  }
  t.table = c.table; t.lam = c.lam; t.pitch = pitch; t.buckets = c.buckets; t.node_lo = plan->node_lo; t.node_deg = plan->node_deg;
  t.n_own = c.n_dst; t.n_other = c.n_src; t.H = c.H; t.scale = (float)c.scale; t.o = o; t.sums = (float*)sums; t.lse = (float*)lse;
  terms_forward_kernel<kMaps, kBucket><<<dim3((unsigned)tiles, (unsigned)c.H), kThreads, L::kBytes, st>>>(mq, mk, mv, t);
  GK_LAUNCHED(kMaps == 2 ? "attention_diff_fwd_banded" : "attention_bucket_fwd_banded");
  const AgainArgs a{t, c.q, c.k, c.v, nullptr, plan->node_first, nullptr, c.bucket, (int)tiles};
  return run_band_again<0, kMaps, kBucket>(a, st);
}

template <int kMaps, bool kBucket>
inline int terms_backward(const graphop_plan_t* plan_r, const graphop_plan_t* plan_t, const TermsCall<__nv_bfloat16>& c,
                          const void* sums, const void* lse, const __nv_bfloat16* dout, __nv_bfloat16* dq, __nv_bfloat16* dk,
                          __nv_bfloat16* dv, __nv_bfloat16* d_table, __nv_bfloat16* d_lam, Arena& ar, cudaStream_t st) {
  using LD = BwdLayout<false, kMaps>;
  using LS = BwdLayout<true, kMaps>;
  const int pitch = band_pitch(plan_r), pitch_t = band_pitch(plan_t), columns = c.H * kMaps;
  const long long tiles = band_tiles_of(c.n_dst), tiles_t = band_tiles_of(c.n_src);
  const BandRoom room = band_room_backward(ar, plan_r, plan_t, c.n_dst, c.n_src, c.H, kMaps, c.buckets);
  if (room.bytes > ar.cap) return GRAPHOP_ERR_UNSUPPORTED;
  TermsTile t{};
  t.stat = room.stat; t.dirty = room.dirty; t.g = room.g; t.g_low = room.g_low;
  CUtensorMap mq, mk, mv, mg, mqs, mgs;
  if (!make_map(&mq, c.q, c.n_dst, c.H) || !make_map(&mk, c.k, c.n_src, c.H) || !make_map(&mv, c.v, c.n_src, c.H) ||
      !make_map(&mg, dout, c.n_dst, c.H) || !make_map_rows(&mqs, c.q, c.n_dst, c.H, LS::kB) ||
      !make_map_rows(&mgs, dout, c.n_dst, c.H, LS::kB))
    return GRAPHOP_ERR_UNSUPPORTED;
  constexpr int smem = LD::kBytes > LS::kBytes ? LD::kBytes : LS::kBytes;
  static std::atomic<bool> configured[64];
  GK_TRY(allow_smem(terms_backward_kernel<kMaps, kBucket>, smem, configured));
  const BandIds own = band_ids_of(plan_r, nullptr, c.n_dst, LD::kC, room.ids), other = band_ids_of(plan_t, plan_t->eid, c.n_src, LS::kC, room.ids_t);
  band_prepare_kernel<kMaps, kBucket><<<dim3((unsigned)(kBucket && tiles_t > tiles ? tiles_t : tiles), kTileM / 8, kBucket ? 3 : 1), 256, 0, st>>>(
      own, other, c.bucket, c.buckets, (const float*)sums, dout, (const float*)lse, c.n_dst * c.H, t.stat, room.t2);
  GK_LAUNCHED("band_prepare");
  t.table = c.table; t.lam = c.lam; t.ids = room.ids; t.pitch = pitch; t.buckets = c.buckets; t.node_lo = plan_r->node_lo;
  t.node_deg = plan_r->node_deg; t.n_own = c.n_dst; t.n_other = c.n_src; t.H = c.H; t.scale = (float)c.scale; t.out0 = dq;
  TermsTile u = t;
  u.ids = room.ids_t; u.pitch = pitch_t; u.node_lo = plan_t->node_lo; u.node_deg = plan_t->node_deg; u.dirty = room.dirty_t; u.n_own = c.n_src;
  u.n_other = c.n_dst; u.out0 = dk; u.out1 = dv;
  terms_backward_kernel<kMaps, kBucket><<<dim3((unsigned)(tiles > tiles_t ? tiles : tiles_t), (unsigned)c.H, 2), kThreads, smem, st>>>(
      mq, mk, mv, mg, mqs, mgs, t, u, (unsigned)tiles, (unsigned)tiles_t);
  GK_LAUNCHED(kMaps == 2 ? "attention_diff_bwd_banded" : "attention_bucket_bwd_banded");
  GK_TRY((run_band_again<1, kMaps, kBucket>(AgainArgs{t, c.q, c.k, c.v, dout, plan_r->node_first, nullptr, c.bucket, (int)tiles}, st)));
  GK_TRY((run_band_again<2, kMaps, kBucket>(AgainArgs{u, c.q, c.k, c.v, dout, plan_t->node_first, plan_t->eid, c.bucket, (int)tiles_t}, st)));
  if (kBucket) GK_TRY(run_band_bucket_sum(room, (int)tiles, c.buckets, c.H, kMaps, d_table, st));
  if (kMaps == 2) GK_TRY((run_bucket_sum<__nv_bfloat16>(ar, room.t2, c.n_dst, c.H, 1, c.H, nullptr, 1, nullptr, -1.0, d_lam, st)));
  return GRAPHOP_OK;
}

}  // namespace banded

// Where band_serves and the workspace is as large as graphop_terms_workspace_bytes_planned asks; GRAPHOP_ERR_UNSUPPORTED else: the caller
// then runs the walkers.
template <>
inline int banded_terms_forward<__nv_bfloat16>(const graphop_plan_t* plan, const TermsCall<__nv_bfloat16>& c, __nv_bfloat16* o,
                                               void* sums, void* lse, void* ws, size_t wsb, cudaStream_t st) {
  if (!banded::band_serves(plan, nullptr, c.n_dst, c.n_src, c.H, c.row_d(), c.buckets) || ((uintptr_t)sums & 31))   // store_sums16's alignment
    return GRAPHOP_ERR_UNSUPPORTED;
  Arena ar(ws, wsb);
  if (!c.diff) return banded::terms_forward<1, true>(plan, c, o, sums, lse, ar, st);
  if (c.buckets) return banded::terms_forward<2, true>(plan, c, o, sums, lse, ar, st);
  return banded::terms_forward<2, false>(plan, c, o, sums, lse, ar, st);
}
template <>
inline int banded_terms_backward<__nv_bfloat16>(const graphop_plan_t* plan_r, const graphop_plan_t* plan_t,
                                                const TermsCall<__nv_bfloat16>& c, const void* sums, const void* lse,
                                                const __nv_bfloat16* dout, __nv_bfloat16* dq, __nv_bfloat16* dk, __nv_bfloat16* dv,
                                                __nv_bfloat16* d_table, __nv_bfloat16* d_lam, void* ws, size_t wsb, cudaStream_t st) {
  if (!banded::band_serves(plan_r, plan_t, c.n_dst, c.n_src, c.H, c.row_d(), c.buckets)) return GRAPHOP_ERR_UNSUPPORTED;
  Arena ar(ws, wsb);
  if (!c.diff) return banded::terms_backward<1, true>(plan_r, plan_t, c, sums, lse, dout, dq, dk, dv, d_table, d_lam, ar, st);
  if (c.buckets) return banded::terms_backward<2, true>(plan_r, plan_t, c, sums, lse, dout, dq, dk, dv, d_table, d_lam, ar, st);
  return banded::terms_backward<2, false>(plan_r, plan_t, c, sums, lse, dout, dq, dk, dv, d_table, d_lam, ar, st);
}

}  // namespace gk
