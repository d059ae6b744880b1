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
//           two groups of four warps turn 16 places at a time. base comes through
//           cp.async, three turns ahead: each thread reads what it copied itself. (In
//           registers one turn ahead fit, 121 us; two were slower, 185 us, since
//           waiting for the older loads also waited for the younger ones.)
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
constexpr int kTurn = 16;               // places that a group turns at a time
constexpr int kAhead = 3;               // turns whose base is on its way

// atoms: ceil(rank / 64). The halves of h, a block of B, for each group two turning
// buffers and the base of kAhead turns: two CTAs per SM up to rank 64.
constexpr int second_wide_smem(int atoms) {
  return 1024 + 3 * atoms * kAtomBytes + 2 * 2 * kTurn * kWideFeat * 4 + 2 * kAhead * kTurn * kWideFeat * 2;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

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
  float* turns = reinterpret_cast<float*>(b_smem + atoms * kAtomBytes);  // [group][2][kTurn][kWideFeat]
  uint8_t* bases = reinterpret_cast<uint8_t*>(turns + 4 * kTurn * kWideFeat);  // [group][kAhead][2][128] vectors
  __shared__ float row_scale[kWideRows];
  __shared__ int64_t row_in[kWideRows], row_out[kWideRows];  // where a place's row starts, or -1
  __shared__ uint64_t h_full, b_full, b_empty, acc_full[2], acc_empty[2];
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
    for (int row = warp; row < r.n; row += kSecondWideThreads / 32) {
      if (row_in[row] < 0) continue;
      const T* src = static_cast<const T*>(g.base) + row_in[row];
      T* dst = static_cast<T*>(g.out) + row_out[row];
      for (int f = f_begin + lane * 8; f < f_end; f += 4 * 256) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (f + j * 256 < f_end) v[j] = *reinterpret_cast<const uint4*>(src + f + j * 256);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (f + j * 256 < f_end) *reinterpret_cast<uint4*>(dst + f + j * 256) = v[j];
      }
    }
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&h_full), 1);
    mbar_init(smem_u32(&b_full), 1);
    mbar_init(smem_u32(&b_empty), 1);
    for (int b = 0; b < 2; ++b) {
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
      ok = mbar_wait(smem_u32(&b_empty), (fb & 1) ^ 1);
      if (ok && elect_one()) {
        mbar_arrive_expect_tx(smem_u32(&b_full), atoms * kAtomBytes);
        for (int a = 0; a < atoms; ++a)
          tma_load_2d(smem_u32(b_smem + a * kAtomBytes), &tm_b, a * 64, r.adapter * g.N + f_begin + fb * kWideFeat,
                      smem_u32(&b_full), keep);
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
      ok = mbar_wait(smem_u32(&acc_empty[b]), ((fb >> 1) & 1) ^ 1) && mbar_wait(smem_u32(&b_full), fb & 1);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t b_desc = make_sw128_kmajor_desc(smem_u32(b_smem));
        for (int half = 0; half < 2; ++half)
          for (int k = 0; k < steps; ++k) {
            const uint32_t at = (k >> 2) * (kAtomBytes >> 4) + (k & 3) * 2;
            tc_mma_f16(tmem + b * kWideRows, b_desc + at, h_desc + half * atoms * (kAtomBytes >> 4) + at, idesc,
                       half + k > 0);
          }
        tc_commit(smem_u32(&b_empty));
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
    float* turn = turns + group * 2 * kTurn * kWideFeat;
    const uint32_t mine = smem_u32(bases) + (group * kAhead * 2 * 128 + tid) * 16;
    // This group's turns: every second 16 places of every block.
    const int per_block = max(0, ((r.n + kTurn - 1) / kTurn - group + 1) / 2);
    const int all = blocks * per_block;
    int copy_block = 0, copy_turn = 0, copied = 0;  // the next turn to copy base for, and its number
    const auto copy_base = [&]() {
      if (copied < all) {
        const int f = f_begin + copy_block * kWideFeat + fl, first = (group + 2 * copy_turn) * kTurn + tk;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int64_t at = row_in[first + 8 * j];  // -1 past r.n
          if (at >= 0 && f < f_end)
            cp_async16(mine + (copied % kAhead * 2 + j) * 128 * 16, static_cast<const T*>(g.base) + at + f);
        }
        if (++copy_turn == per_block) copy_turn = 0, ++copy_block;
        ++copied;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < kAhead; ++i) copy_base();
    int q = 0;
    for (int fb = 0; fb < blocks && per_block > 0; ++fb) {
      const int b = fb & 1, f = f_begin + fb * kWideFeat + fl;
      ok = named_bar_and(1 + group, 128, mbar_wait(smem_u32(&acc_full[b]), (fb >> 1) & 1));
      if (!ok) break;
      tc_fence_after();
      for (int i = 0; i < per_block; ++i, ++q) {
        const int first = (group + 2 * i) * kTurn;
        uint32_t v[16];
        tmem_ld16(tmem + b * kWideRows + first + ((uint32_t)(warp & 3) << 21), v);
        tmem_ld_wait();
        if (i == per_block - 1) {  // the accumulator is read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&acc_empty[b]));
        }
        float* here = turn + (q & 1) * kTurn * kWideFeat;
#pragma unroll
        for (int j = 0; j < kTurn; ++j) here[j * kWideFeat + put] = __uint_as_float(v[j]);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        named_bar_sync(1 + group, 128);  // two buffers: the next turn's writes need no second one
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int64_t to = row_out[first + tk + 8 * j];
          if (to >= 0 && f < f_end) {
            const float w = row_scale[first + tk + 8 * j];
            const float4 p0 = *reinterpret_cast<const float4*>(here + (tk + 8 * j) * kWideFeat + get);
            const float4 p1 = *reinterpret_cast<const float4*>(here + (tk + 8 * j) * kWideFeat + (get ^ 4));
            uint4 y;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                         : "r"(mine + (q % kAhead * 2 + j) * 128 * 16)
                         : "memory");
            float o[8];
            unpack_vec<T>(y, o);
            o[0] += w * p0.x, o[1] += w * p0.y, o[2] += w * p0.z, o[3] += w * p0.w;
            o[4] += w * p1.x, o[5] += w * p1.y, o[6] += w * p1.z, o[7] += w * p1.w;
            *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + to + f) = pack_vec<T>(o);
          }
        }
        copy_base();
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (per_block == 0)  // no places for this group: it only lets the accumulators go
      for (int fb = 0; fb < blocks && ok; ++fb) {
        ok = mbar_wait(smem_u32(&acc_full[fb & 1]), (fb >> 1) & 1);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&acc_empty[fb & 1]));
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
