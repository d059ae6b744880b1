// The adapters' products for prompts, on tcgen05 (included by awqb_lora.cu).
//
// On mma.sync the warps that issue the products also move the operands and were
// bound by their own instructions and shared-memory reads (4111 rows, K = 4096,
// rank 64, 28672 features: 25 us the first, 219 us the second product for 470 MB of base and
// out). Here the tensor core fetches its operands from shared memory, TMA brings
// them, and the warps only turn the accumulator and stream base and out.
//   first:  a CTA takes 128 places of one adapter x up to 128 columns over a part of
//           K. A run of neighbouring rows of x (one request's tokens) comes by one TMA box
//           a stage; scattered rows by cp.async of the four warps that wait for
//           the accumulator. (Gathering copies, four rows each, took about 60 clocks
//           apiece: 22 us for 4111 rows, K = 4096, 128 columns.) Columns on the
//           accumulator's lanes, so that a warp writes 32 neighbouring columns of
//           a place.
//   join:   a warp per place and slice adds the parts in order and splits the sums in halves.
//   second: persistent CTAs take equal runs of units (128 places x 128 features) and
//           walk them in segments of one tile of places and one slice, whose halves of
//           h stay in shared memory. Places on the accumulator's lanes: a thread adds
//           its products to its place's row of base in shared memory, where its warp
//           copied 32 rows of 128 features (256 bytes each) one block ahead and from
//           where it writes them out the same way; no warp waits for another. Two
//           groups of four warps work on alternate blocks. (Features on the lanes, the
//           accumulator turned through shared memory in fp32 and base through the
//           threads: bound by their instructions, 115 us for 4111 rows, rank 64, 28672
//           features. Rows by bulk copies, one per row and block: 124 us, 16 clocks
//           for each copy.)
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
// A row of a block in shared memory: 16 bytes past a multiple of 128, so that the
// 16-byte accesses of eight rows hit all banks.
constexpr int kRowBytes = kWideFeat * 2 + 16;
constexpr int kTileBytes = kWideRows * kRowBytes;
// atoms: ceil(rank / 64). The halves of h, two blocks of B, and for each group two
// tiles of base, or one where the factors leave no room.
__host__ __device__ constexpr int base_tiles(int atoms) { return atoms == 1 ? 2 : 1; }
__host__ __device__ constexpr int second_wide_smem(int atoms) { return 1024 + 4 * atoms * kAtomBytes + 2 * base_tiles(atoms) * kTileBytes; }

__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in = true) {  // zeros if not in
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kFirstWideThreads, 2)
lora_first_wide_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_a,
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
  const Rows r = find_rows<kFirstWideThreads, kWideRows>(g, blockIdx.x / (g.parts * col_tiles), true, nullptr);
  if (r.n <= 0) return;
  const int row0 = g.order[r.p0];
  const bool run = __syncthreads_and((int)threadIdx.x >= r.n || g.order[r.p0 + threadIdx.x] == row0 + (int)threadIdx.x) &&
                   row0 >= 0 && row0 + r.n <= g.M;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kFirstStages; ++s) {
      mbar_init(smem_u32(&full[s]), run ? 1 : 1 + 128);
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
    const uint64_t keep = policy_evict_last();
    for (int i = 0; i < stages && ok; ++i) {
      const int s = i % kFirstStages;
      ok = mbar_wait(smem_u32(&empty[s]), ((i / kFirstStages) & 1) ^ 1);
      if (!ok) break;
      const uint32_t base = smem_u32(ring + s * 2 * kAtomBytes), bar = smem_u32(&full[s]);
      const int k = k_begin + i * 64;
      if (elect_one()) {
        mbar_arrive_expect_tx(bar, (run ? kAtomBytes : 0) + col_box * 128);
        if (run) tma_load_2d(base, &tm_x, k, row0, bar, keep);
        tma_load_2d(base + kAtomBytes, &tm_a, k, r.adapter * g.R + ct * 128, bar, keep);
      }
      __syncwarp();
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
    if (!run) {  // these warps copy x: 8 lanes a row, 16 bytes each
      const int chunk = threadIdx.x & 7, line = threadIdx.x >> 3;
      int row[8];  // rows line + 16 j; no such place: its column is not used
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int place = line + 16 * j;
        row[j] = place < r.n ? g.order[r.p0 + place] : -1;
        if (row[j] >= g.M) row[j] = -1;
      }
      const auto landed = [&](int i) {  // stage i's copies of this thread are complete
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(&full[i % kFirstStages]));
      };
      for (int i = 0; i < stages && ok; ++i) {
        const int s = i % kFirstStages, k = k_begin + i * 64 + chunk * 8;
        ok = mbar_wait(smem_u32(&empty[s]), ((i / kFirstStages) & 1) ^ 1);
        if (!ok) break;
        const uint32_t base = smem_u32(ring + s * 2 * kAtomBytes) + line * 128 + ((chunk ^ (line & 7)) << 4);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (row[j] >= 0)
            cp_async16(base + j * 16 * 128, static_cast<const T*>(g.x) + row[j] * g.ldx + (k < g.K ? k : 0), k < g.K);
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        if (i > 1) landed(i - 2);
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      if (ok && stages > 1) landed(stages - 2);
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (ok) landed(stages - 1);
    }
    ok = ok && mbar_wait(smem_u32(&acc_full), 0);
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

// halves[slice][hi, lo][place][rank], up[slice][place]: the power of two that a
// place's halves were divided by.
template <typename T>
__global__ void __launch_bounds__(256) lora_join_kernel(const __grid_constant__ Args g) {
  const int unit = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int place = unit / g.S, s = unit - place * g.S;
  grid_dep_wait();
  grid_dep_launch();
  if (place >= g.M || place < g.offsets[0] || place >= g.offsets[g.L]) return;
  constexpr int kPairs = kMaxRank / 64;
  const float* src = g.h + (int64_t)place * g.R + s * g.rank + lane * 2;
  float2 u[kMaxParts][kPairs], v[kPairs] = {};
#pragma unroll
  for (int p = 0; p < kMaxParts; ++p)
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      u[p][i] = p < g.parts && i * 64 + lane * 2 < g.rank
                    ? *reinterpret_cast<const float2*>(src + (int64_t)p * g.M * g.R + i * 64)
                    : make_float2(0.f, 0.f);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
#pragma unroll
    for (int p = 0; p < kMaxParts; ++p) v[i].x += u[p][i].x, v[i].y += u[p][i].y;
    top = fmaxf(top, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
  }
  const int e = row_exponent<T>(top);
  const float down = ldexpf(1.f, -e);
  T* to = static_cast<T*>(g.halves) + ((int64_t)s * 2 * g.M + place) * g.rank + lane * 2;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    if (i * 64 + lane * 2 >= g.rank) continue;
    T hi[2], lo[2];
    halves<T>(v[i].x * down, &hi[0], &lo[0]);
    halves<T>(v[i].y * down, &hi[1], &lo[1]);
    *reinterpret_cast<uint32_t*>(to + i * 64) = *reinterpret_cast<uint32_t*>(hi);
    *reinterpret_cast<uint32_t*>(to + (int64_t)g.M * g.rank + i * 64) = *reinterpret_cast<uint32_t*>(lo);
  }
  if (lane == 0) g.up[(int64_t)s * g.M + place] = ldexpf(1.f, e);
}

template <typename T>
__global__ void __launch_bounds__(kSecondWideThreads, 1)
lora_second_wide_kernel(const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_h,
                        const __grid_constant__ Args g, int blocks_per_tile, int atoms) {
  extern __shared__ uint8_t raw[];
  uint8_t* h_smem = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  uint8_t* b_smem = h_smem + 2 * atoms * kAtomBytes;
  uint8_t* tiles_smem = b_smem + 2 * atoms * kAtomBytes;  // [group][base_tiles][kTileBytes]
  __shared__ int64_t row_in[kWideRows], row_out[kWideRows];  // where a place's row starts, or -1
  __shared__ uint64_t h_full, b_full[2], b_empty[2], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bufs = base_tiles(atoms);
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&h_full), 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&b_full[b]), 1);
      mbar_init(smem_u32(&b_empty[b]), 1);
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), 4);
    }
    failed = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_b);
    prefetch_tmap(&tm_h);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&tmem_slot), 2 * kWideFeat);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const bool in_place = g.out == g.base;
  int tiles = 0;
  find_rows<kSecondWideThreads, kWideRows>(g, -1, in_place, &tiles);
  const int64_t units = (int64_t)tiles * blocks_per_tile;
  const int64_t u1 = units * (blockIdx.x + 1) / gridDim.x;
  int done = 0, segments = 0;  // blocks and segments of products so far: the barriers' phases
  bool ok = true;
  grid_dep_wait();
  for (int64_t u = units * blockIdx.x / gridDim.x; u < u1;) {
    const Rows r = find_rows<kSecondWideThreads, kWideRows>(g, (int)(u / blocks_per_tile), in_place, nullptr);
    const Feats feats = find_feats(g, (int)(u % blocks_per_tile), kWideFeat);
    const int s = feats.slice, f_begin = feats.begin;
    const int left = (g.slice_end[s] - f_begin + kWideFeat - 1) / kWideFeat;
    const int blocks = (int)min((int64_t)left, u1 - u);
    const int f_end = min(g.slice_end[s], f_begin + blocks * kWideFeat);
    u += blocks;
    if (r.adapter < 0) {  // rows without an adapter: out = base, a row per warp
      for (int row = warp; row < r.n; row += kSecondWideThreads / 32) {
        const int tok = g.order[r.p0 + row];
        if (tok < 0 || tok >= g.M) continue;
        const T* src = static_cast<const T*>(g.base) + tok * g.ld_base;
        T* dst = static_cast<T*>(g.out) + tok * g.ld_out;
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
      continue;
    }
    if (warp == 8) {  // ----------------------------------------------- h, B
      const uint64_t keep = policy_evict_last();
      if (elect_one()) {
        mbar_arrive_expect_tx(smem_u32(&h_full), 2 * atoms * kAtomBytes);
        for (int half = 0; half < 2; ++half)
          for (int a = 0; a < atoms; ++a)
            tma_load_2d(smem_u32(h_smem + (half * atoms + a) * kAtomBytes), &tm_h, a * 64, (2 * s + half) * g.M + r.p0,
                        smem_u32(&h_full), keep);
      }
      __syncwarp();
      for (int i = 0; i < blocks && ok; ++i) {
        const int b = (done + i) & 1;
        ok = mbar_wait(smem_u32(&b_empty[b]), (((done + i) >> 1) & 1) ^ 1);
        if (ok && elect_one()) {
          mbar_arrive_expect_tx(smem_u32(&b_full[b]), atoms * kAtomBytes);
          for (int a = 0; a < atoms; ++a)
            tma_load_2d(smem_u32(b_smem + (b * atoms + a) * kAtomBytes), &tm_b, a * 64,
                        r.adapter * g.N + f_begin + i * kWideFeat, smem_u32(&b_full[b]), keep);
        }
        __syncwarp();
      }
    } else if (warp == 9) {  // ---------------------------------------- products
      const uint32_t idesc = make_idesc_f16(kWideRows, kWideFeat, std::is_same<T, __nv_bfloat16>::value);
      const uint64_t h_desc = make_sw128_kmajor_desc(smem_u32(h_smem));
      const int steps = (g.rank + 15) / 16;
      ok = mbar_wait(smem_u32(&h_full), segments & 1);
      for (int i = 0; i < blocks && ok; ++i) {
        const int b = (done + i) & 1, phase = ((done + i) >> 1) & 1;
        ok = mbar_wait(smem_u32(&acc_empty[b]), phase ^ 1) && mbar_wait(smem_u32(&b_full[b]), phase);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t b_desc = make_sw128_kmajor_desc(smem_u32(b_smem + b * atoms * kAtomBytes));
          for (int half = 0; half < 2; ++half)
            for (int k = 0; k < steps; ++k) {
              const uint32_t at = (k >> 2) * (kAtomBytes >> 4) + (k & 3) * 2;
              tc_mma_f16(tmem + b * kWideFeat, h_desc + half * atoms * (kAtomBytes >> 4) + at, b_desc + at, idesc,
                         half + k > 0);
            }
          tc_commit(smem_u32(&b_empty[b]));
          tc_commit(smem_u32(&acc_full[b]));
        }
        __syncwarp();
      }
    } else {  // -------------------------------------------------------- epilogue
      const int group = warp >> 2, row = threadIdx.x & 127;
      int tok = row < r.n ? g.order[r.p0 + row] : -1;
      if (tok >= g.M) tok = -1;
      const float scale = tok >= 0 ? (g.scales ? g.scales[r.adapter] : 1.f) * g.up[(int64_t)s * g.M + r.p0 + row] : 0.f;
      if (group == 0) {
        row_in[row] = tok >= 0 ? tok * g.ld_base : -1;
        row_out[row] = tok >= 0 ? tok * g.ld_out : -1;
      }
      named_bar_sync(1, 256);
      // the warp's rows of a block: lane l moves vector l % 16 of rows l / 16 + 2 j
      const int row0 = (warp & 3) * 32 + (lane >> 4), rows = min(32, r.n - (warp & 3) * 32), fl = (lane & 15) * 8;
      const uint32_t tile = smem_u32(tiles_smem) + (group * bufs * 4 + (warp & 3)) * 32 * kRowBytes;
      const uint32_t mine = tile + (row & 31) * kRowBytes, moved = tile + (lane >> 4) * kRowBytes + (lane & 15) * 16;
      const auto fetch = [&](int i, int buf) {  // base of block i of the segment, if there is one
        const int f = f_begin + i * kWideFeat + fl;
        if (i < blocks && f < f_end)
          for (int j = 0; j < rows; j += 2) {
            const int64_t at = row_in[row0 + j];  // -1 past r.n
            if (at >= 0) cp_async16(moved + buf * kTileBytes + j * kRowBytes, static_cast<const T*>(g.base) + at + f);
          }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      const int first = (group ^ done) & 1;  // the group's blocks are those of its accumulator
      int buf = 0;
      fetch(first, 0);
      for (int i = first; i < blocks && ok; i += 2) {
        const int f = f_begin + i * kWideFeat, width = min(kWideFeat, f_end - f);
        if (bufs == 2) {
          fetch(i + 2, buf ^ 1);
          asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncwarp();  // a lane waits for its own copies, and reads a row that the others copied
        ok = mbar_wait(smem_u32(&acc_full[group]), ((done + i) >> 1) & 1);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t at = mine + buf * kTileBytes, acc = tmem + group * kWideFeat + ((uint32_t)(warp & 3) << 21);
        for (int c = 0; c < kWideFeat; c += 32) {
          uint32_t v[2][16];
          tmem_ld16(acc + c, v[0]);
          tmem_ld16(acc + c + 16, v[1]);
          uint4 y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = ld_shared(at + c * 2 + j * 16);
          tmem_ld_wait();
          if (c == kWideFeat - 32) {  // the accumulator is read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&acc_empty[group]));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float o[8];
            unpack_vec<T>(y[j], o);
#pragma unroll
            for (int q = 0; q < 8; ++q) o[q] += scale * __uint_as_float(v[j / 2][j % 2 * 8 + q]);
            st_shared(at + c * 2 + j * 16, pack_vec<T>(o));
          }
        }
        __syncwarp();
        if (fl < width) {
#pragma unroll 4
          for (int j = 0; j < rows; j += 2) {
            const int64_t to = row_out[row0 + j];
            if (to >= 0)
              *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + to + f + fl) = ld_shared(moved + buf * kTileBytes + j * kRowBytes);
          }
        }
        __syncwarp();
        if (bufs == 2) buf ^= 1; else fetch(i + 2, 0);
      }
    }
    done += blocks;
    ++segments;
    if (!ok && lane == 0) {
      failed = 1;
      atomicOr(g.err, kErrLoraWait);
    }
    __syncwarp();
    __syncthreads();  // the halves are read
    if (failed) break;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (failed) linger();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kWideFeat);
  }
}

}  // namespace
}  // namespace awqb
