// The adapters' products for prompts, on tcgen05 (included by awqb_lora.cu).
//
// On mma.sync the warps that issue the products also move the operands and were
// bound by their own instructions and shared-memory reads (4111 rows, K = 4096,
// rank 64, 28672 features: 25 us the first, 219 us the second product for 470 MB of base and
// out). Here the tensor core fetches its operands from shared memory, TMA brings
// them, and the warps only turn the accumulator and stream base and out.
//   first:  a CTA takes 128 places of one adapter x up to 128 columns over a part of
//           K. The rows of x are scattered: each lane of the producer warp gathers four
//           by their numbers per stage. Columns on the accumulator's lanes, so
//           that a warp writes 32 neighbouring columns of a place.
//   join:   a warp per place adds the parts in order and splits the sums in halves.
//   second: a CTA takes 128 places and a chunk of one slice's features, keeps the
//           places' halves in shared memory and walks the chunk in blocks of 128
//           features (both halves times the same block of B, two accumulators);
//           two groups of four warps take turns over 32 places at a time.
#pragma once
#include "awqb_ptx.cuh"

namespace awqb {
namespace {

constexpr int kWideRows = 128;          // places per CTA
constexpr int kWideFeat = 128;          // features per block of the second product
constexpr int kAtomBytes = 128 * 128;   // 128 rows of 64 k, 128-byte swizzle
constexpr int kFirstWideThreads = 192;  // four epilogue warps, producer, MMA issuer
constexpr int kFirstStages = 3;         // two CTAs per SM
constexpr int kSecondWideThreads = 320; // eight epilogue warps, producer, MMA issuer
constexpr uint32_t kErrLoraWait = 256u; // a bounded wait gave up

constexpr int first_wide_smem() { return 1024 + kFirstStages * 2 * kAtomBytes; }
// atoms: ceil(rank / 64). The halves of h, two blocks of B, two turning buffers.
constexpr int second_wide_smem(int atoms) { return 1024 + 4 * atoms * kAtomBytes + 2 * 32 * kWideFeat * 4; }

// Four rows (y0..y3) x 64 k by their numbers; the tensor map's box is one row high.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const void* tmap, int32_t x, int32_t y0, int32_t y1, int32_t y2,
                                            int32_t y3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(tmap), "r"(x), "r"(y0), "r"(y1), "r"(y2), "r"(y3), "r"(bar)
      : "memory");
}

// After a wait gave up: copies and products in flight get time to end.
__device__ __forceinline__ void linger() {
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 10000000ull) {
  }
}

template <typename T>
__global__ void __launch_bounds__(kFirstWideThreads, 2)
lora_first_wide_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_run, const __grid_constant__ CUtensorMap tm_a,
                       const __grid_constant__ Args g, int col_box) {
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  __shared__ uint64_t full[kFirstStages], empty[kFirstStages], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dep_wait();
  grid_dep_launch();
  const int col_tiles = (g.R + 127) / 128;
  const int part = blockIdx.x % g.parts, ct = blockIdx.x / g.parts % col_tiles;
  const Rows r = find_rows<kFirstWideThreads, kWideRows>(g, blockIdx.x / (g.parts * col_tiles), true);
  if (r.n <= 0) return;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kFirstStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(&acc_full), 1);
    failed = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_x);
    prefetch_tmap(&tm_a);
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(&tmem_slot), kWideRows);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int k_begin = part * g.k_part, k_end = min(g.K, k_begin + g.k_part);
  const int stages = (k_end - k_begin + 63) / 64;
  const int n = (r.n + 15) / 16 * 16;
  bool ok = true;
  if (warp == 4) {
    int row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int place = lane * 4 + i;
      const int tok = place < r.n ? g.order[r.p0 + place] : 0;
      row[i] = tok >= 0 && tok < g.M ? tok : 0;  // no such place: some row, its column is not used
    }
    const int groups = (n + 3) / 4;
    // a run of one request's tokens: neighbouring rows, one box
    const int row0 = __shfl_sync(0xffffffffu, row[0], 0);
    bool mine = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine = mine && (lane * 4 + i >= r.n || row[i] == row0 + lane * 4 + i);
    const bool run = __all_sync(0xffffffffu, mine);
    const uint64_t keep = policy_evict_last();
    for (int i = 0; i < stages && ok; ++i) {
      const int s = i % kFirstStages;
      ok = mbar_wait(smem_u32(&empty[s]), ((i / kFirstStages) & 1) ^ 1);
      if (!ok) break;
      const uint32_t base = smem_u32(ring + s * 2 * kAtomBytes), bar = smem_u32(&full[s]);
      const int k = k_begin + i * 64;
      if (elect_one()) {
        mbar_arrive_expect_tx(bar, (run ? kAtomBytes : groups * 512) + col_box * 128);
        if (run) tma_load_2d(base, &tm_run, k, row0, bar, keep);
        tma_load_2d(base + kAtomBytes, &tm_a, k, r.adapter * g.R + ct * 128, bar, keep);
      }
      __syncwarp();
      if (!run && lane < groups) tma_gather4(base + lane * 512, &tm_x, k, row[0], row[1], row[2], row[3], bar);
    }
  } else if (warp == 5) {
    const uint32_t idesc = make_idesc_f16(128, n, std::is_same<T, __nv_bfloat16>::value);
    for (int i = 0; i < stages && ok; ++i) {
      const int s = i % kFirstStages;
      ok = mbar_wait(smem_u32(&full[s]), (i / kFirstStages) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t x_desc = make_sw128_kmajor_desc(smem_u32(ring + s * 2 * kAtomBytes));
        const uint64_t a_desc = make_sw128_kmajor_desc(smem_u32(ring + s * 2 * kAtomBytes + kAtomBytes));
        // a part ends at a multiple of 64 k or at K, past which the copies read zeros
        for (int j = 0; j < 4; ++j) tc_mma_f16(tmem, a_desc + 2 * j, x_desc + 2 * j, idesc, i + j > 0);
        tc_commit(smem_u32(&empty[s]));
        if (i == stages - 1) tc_commit(smem_u32(&acc_full));
      }
      __syncwarp();
    }
  } else {
    ok = mbar_wait(smem_u32(&acc_full), 0);
    if (named_bar_and(1, 128, ok)) {
      tc_fence_after();
      const int col = ct * 128 + threadIdx.x;
      float* h = g.h + ((int64_t)part * g.M + r.p0) * g.R + col;
      for (int c = 0; c < r.n; c += 16) {
        uint32_t v[16];
        tmem_ld16(tmem + c + ((uint32_t)warp << 21), v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (col < g.R && c + j < r.n) h[(int64_t)(c + j) * g.R] = __uint_as_float(v[j]);
      }
    }
  }
  if (!ok && lane == 0) {
    failed = 1;
    atomicOr(g.err, kErrLoraWait);
  }
  __syncwarp();
  __syncthreads();
  if (failed) linger();
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, kWideRows);
  }
}

// halves[slice][hi, lo][place][rank], down[slice][place]: the power of two that a
// place's halves were divided by.
template <typename T>
__global__ void __launch_bounds__(256) lora_join_kernel(const __grid_constant__ Args g) {
  const int place = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  grid_dep_wait();
  grid_dep_launch();
  if (place >= g.M || place < g.offsets[0] || place >= g.offsets[g.L]) return;
  for (int s = 0; s < g.S; ++s) {
    float2 v[kMaxRank / 64] = {};
    const float* src = g.h + (int64_t)place * g.R + s * g.rank + lane * 2;
    for (int p0 = 0; p0 < g.parts; p0 += 4) {
      float2 u[4][kMaxRank / 64];
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < kMaxRank / 64; ++i)
          u[p][i] = p0 + p < g.parts && i * 64 + lane * 2 < g.rank
                        ? *reinterpret_cast<const float2*>(src + (int64_t)(p0 + p) * g.M * g.R + i * 64)
                        : make_float2(0.f, 0.f);
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < kMaxRank / 64; ++i) v[i].x += u[p][i].x, v[i].y += u[p][i].y;
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxRank / 64; ++i) top = fmaxf(top, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
    const int e = row_exponent<T>(top);
    const float down = ldexpf(1.f, -e);
    T* to = static_cast<T*>(g.halves) + ((int64_t)s * 2 * g.M + place) * g.rank + lane * 2;
#pragma unroll
    for (int i = 0; i < kMaxRank / 64; ++i) {
      if (i * 64 + lane * 2 >= g.rank) continue;
      T hi[2], lo[2];
      halves<T>(v[i].x * down, &hi[0], &lo[0]);
      halves<T>(v[i].y * down, &hi[1], &lo[1]);
      *reinterpret_cast<uint32_t*>(to + i * 64) = *reinterpret_cast<uint32_t*>(hi);
      *reinterpret_cast<uint32_t*>(to + (int64_t)g.M * g.rank + i * 64) = *reinterpret_cast<uint32_t*>(lo);
    }
    if (lane == 0) g.up[(int64_t)s * g.M + place] = ldexpf(1.f, e);
  }
}

template <typename T>
__global__ void __launch_bounds__(kSecondWideThreads, 2)
lora_second_wide_kernel(const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_h,
                        const __grid_constant__ Args g, int chunks, int chunk, int atoms) {
  extern __shared__ uint8_t raw[];
  uint8_t* h_smem = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  uint8_t* b_smem = h_smem + 2 * atoms * kAtomBytes;
  float* turns = reinterpret_cast<float*>(b_smem + 2 * atoms * kAtomBytes);  // [2][32][kWideFeat]
  __shared__ float row_scale[kWideRows];
  __shared__ int64_t row_in[kWideRows], row_out[kWideRows];  // where a place's row starts, or -1
  __shared__ uint64_t h_full, b_full[2], b_empty[2], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Rows r = find_rows<kSecondWideThreads, kWideRows>(g, blockIdx.x / chunks, g.out == g.base);
  if (r.n <= 0) {
    grid_dep_wait();
    return;
  }
  const Feats feats = find_feats(g, blockIdx.x % chunks, chunk);
  const int s = feats.slice, f_begin = feats.begin, f_end = feats.end;
  const int blocks = (f_end - f_begin + kWideFeat - 1) / kWideFeat;
  for (int i = threadIdx.x; i < kWideRows; i += kSecondWideThreads) {
    const int tok = i < r.n ? g.order[r.p0 + i] : -1;
    const bool in = tok >= 0 && tok < g.M;
    row_in[i] = in ? tok * g.ld_base : -1;
    row_out[i] = in ? tok * g.ld_out : -1;
  }
  if (r.adapter < 0) {  // rows without an adapter: out = base
    __syncthreads();
    grid_dep_wait();
    const int vecs = (f_end - f_begin) / 8;
    for (int i = threadIdx.x; i < r.n * vecs; i += kSecondWideThreads) {
      const int row = i / vecs, f = f_begin + i % vecs * 8;
      if (row_in[row] >= 0)
        *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + row_out[row] + f) =
            *reinterpret_cast<const uint4*>(static_cast<const T*>(g.base) + row_in[row] + f);
    }
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&h_full), 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&b_full[b]), 1);
      mbar_init(smem_u32(&b_empty[b]), 1);
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), 8);
    }
    failed = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_b);
    prefetch_tmap(&tm_h);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&tmem_slot), 2 * kWideRows);
    tmem_relinquish();
  }
  grid_dep_wait();
  const float scale = g.scales ? g.scales[r.adapter] : 1.f;
  for (int i = threadIdx.x; i < r.n; i += kSecondWideThreads) row_scale[i] = scale * g.up[(int64_t)s * g.M + r.p0 + i];
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  bool ok = true;
  if (warp == 8) {  // ------------------------------------------------- h, B
    const uint64_t keep = policy_evict_last();
    if (elect_one()) {
      mbar_arrive_expect_tx(smem_u32(&h_full), 2 * atoms * kAtomBytes);
      for (int half = 0; half < 2; ++half)
        for (int a = 0; a < atoms; ++a)
          tma_load_2d(smem_u32(h_smem + (half * atoms + a) * kAtomBytes), &tm_h, a * 64, (2 * s + half) * g.M + r.p0,
                      smem_u32(&h_full), keep);
    }
    __syncwarp();
    for (int fb = 0; fb < blocks && ok; ++fb) {
      const int b = fb & 1;
      ok = mbar_wait(smem_u32(&b_empty[b]), ((fb >> 1) & 1) ^ 1);
      if (ok && elect_one()) {
        mbar_arrive_expect_tx(smem_u32(&b_full[b]), atoms * kAtomBytes);
        for (int a = 0; a < atoms; ++a)
          tma_load_2d(smem_u32(b_smem + (b * atoms + a) * kAtomBytes), &tm_b, a * 64,
                      r.adapter * g.N + f_begin + fb * kWideFeat, smem_u32(&b_full[b]), keep);
      }
      __syncwarp();
    }
  } else if (warp == 9) {  // ------------------------------------------ products
    const uint32_t idesc = make_idesc_f16(kWideFeat, (r.n + 15) / 16 * 16, std::is_same<T, __nv_bfloat16>::value);
    const uint64_t h_desc = make_sw128_kmajor_desc(smem_u32(h_smem));
    const int steps = (g.rank + 15) / 16;
    ok = mbar_wait(smem_u32(&h_full), 0);
    for (int fb = 0; fb < blocks && ok; ++fb) {
      const int b = fb & 1;
      ok = mbar_wait(smem_u32(&acc_empty[b]), ((fb >> 1) & 1) ^ 1) && mbar_wait(smem_u32(&b_full[b]), (fb >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t b_desc = make_sw128_kmajor_desc(smem_u32(b_smem + b * atoms * kAtomBytes));
        for (int half = 0; half < 2; ++half)
          for (int k = 0; k < steps; ++k) {
            const uint32_t at = (k >> 2) * (kAtomBytes >> 4) + (k & 3) * 2;
            tc_mma_f16(tmem + b * kWideRows, b_desc + at, h_desc + half * atoms * (kAtomBytes >> 4) + at, idesc,
                       half + k > 0);
          }
        tc_commit(smem_u32(&b_empty[b]));
        tc_commit(smem_u32(&acc_full[b]));
      }
      __syncwarp();
    }
  } else {  // ---------------------------------------------------------- epilogue
    const int group = warp >> 2, tid = threadIdx.x & 127;
    const int fl = (tid & 15) * 8, tk = tid >> 4;
    // Feature c stands at c, its halves of eight swapped where bit 5 is set: the
    // 16-byte reads of eight lanes then hit all banks.
    const int put = tid ^ ((tid >> 3) & 4), get = fl + ((fl >> 3) & 4);
    float* turn = turns + group * 32 * kWideFeat;
    uint4 y[4];
    const auto load_base = [&](int f, int first, uint4 (&v)[4]) {  // places first + tk + 8 j
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t at = row_in[(first + tk + 8 * j) & (kWideRows - 1)];  // -1 past r.n
        if (at >= 0 && f < f_end) v[j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(g.base) + at + f);
      }
    };
    if (group * 32 < r.n) load_base(f_begin + fl, group * 32, y);
    for (int fb = 0; fb < blocks; ++fb) {
      const int b = fb & 1, f = f_begin + fb * kWideFeat + fl;
      ok = mbar_wait(smem_u32(&acc_full[b]), (fb >> 1) & 1);
      if (!named_bar_and(1 + group, 128, ok)) break;
      tc_fence_after();
      if (group * 32 >= r.n) {  // nothing for this group
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&acc_empty[b]));
        continue;
      }
      for (int first = group * 32; first < r.n; first += 64) {
        uint32_t v[2][16];
        const uint32_t at = tmem + b * kWideRows + first + ((uint32_t)(warp & 3) << 21);
        tmem_ld16(at, v[0]);
        tmem_ld16(at + 16, v[1]);
        tmem_ld_wait();
        const bool last = first + 64 >= r.n;
        if (last) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&acc_empty[b]));
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) turn[j * kWideFeat + put] = __uint_as_float(v[j / 16][j % 16]);
        uint4 y_next[4];
        load_base(last ? f + kWideFeat : f, last ? group * 32 : first + 64, y_next);
        named_bar_sync(1 + group, 128);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = first + tk + 8 * j;
          const int64_t to = row_out[i];
          if (to >= 0 && f < f_end) {
            const float w = row_scale[i];
            const float4 p0 = *reinterpret_cast<const float4*>(turn + (tk + 8 * j) * kWideFeat + get);
            const float4 p1 = *reinterpret_cast<const float4*>(turn + (tk + 8 * j) * kWideFeat + (get ^ 4));
            float o[8];
            unpack_vec<T>(y[j], o);
            o[0] += w * p0.x, o[1] += w * p0.y, o[2] += w * p0.z, o[3] += w * p0.w;
            o[4] += w * p1.x, o[5] += w * p1.y, o[6] += w * p1.z, o[7] += w * p1.w;
            *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + to + f) = pack_vec<T>(o);
          }
          y[j] = y_next[j];
        }
        named_bar_sync(1 + group, 128);
      }
    }
  }
  if (!ok && lane == 0) {
    failed = 1;
    atomicOr(g.err, kErrLoraWait);
  }
  __syncwarp();
  __syncthreads();
  if (failed) linger();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kWideRows);
  }
}

}  // namespace
}  // namespace awqb
