// The second product of the adapters for prompts: out = base + scale * h B^T on
// tcgen05. On mma.sync the warps that issue the products also move base and out
// and were bound by their own instructions (4111 rows, rank 64, 28672 features:
// 219 us for 470 MB); here the tensor core fetches both operands from shared memory
// and the warps only turn the accumulator and stream base and out.
//
// A CTA takes 128 places of one adapter and a chunk of one slice's features. It
// writes its rows' h as two 16-bit halves into shared memory once (the layout
// that the tensor core reads: 128-byte swizzled rows of 64 k), then walks the
// chunk in blocks of 128 features: TMA brings the block of B, one warp issues the
// products of both halves with the same B (features on the accumulator's lanes,
// places on its columns, two buffers), and two groups of four warps take turns
// over 32 places at a time: the accumulator goes through shared memory, so that base
// and out move as 256 contiguous bytes of a row, base loaded one turn ahead.
#pragma once
#include "awqb_ptx.cuh"

namespace awqb {
namespace {

constexpr int kWideRows2 = 128;   // places per CTA
constexpr int kWideFeat = 128;    // features per block
constexpr int kWideThreads = 320; // 8 epilogue warps, a producer, an MMA issuer
constexpr int kAtomBytes = 128 * 128;  // 128 rows of 64 k
constexpr uint32_t kErrLoraWait = 256u;

// atoms: ceil(rank / 64). Shared memory: h (hi, lo), two blocks of B, two turning buffers.
constexpr int wide_smem(int atoms) { return 1024 + 4 * atoms * kAtomBytes + 2 * 32 * kWideFeat * 4; }

template <typename T>
__global__ void __launch_bounds__(kWideThreads) lora_second_wide_kernel(const __grid_constant__ CUtensorMap tm_b,
                                                                       const __grid_constant__ Args g, int chunks,
                                                                       int chunk, int atoms) {
  extern __shared__ uint8_t raw[];
  uint8_t* h_smem = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  uint8_t* b_smem = h_smem + 2 * atoms * kAtomBytes;
  float* turns = reinterpret_cast<float*>(b_smem + 2 * atoms * kAtomBytes);  // [2][32][kWideFeat]
  __shared__ float row_scale[kWideRows2];
  __shared__ int row_of[kWideRows2];
  __shared__ uint64_t b_full[2], b_empty[2], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Rows r = find_rows<kWideThreads, kWideRows2>(g, blockIdx.x / chunks, g.out == g.base);
  if (r.n <= 0) {
    grid_dep_wait();
    return;
  }
  const Feats feats = find_feats(g, blockIdx.x % chunks, chunk);
  const int s = feats.slice, f_begin = feats.begin, f_end = feats.end;
  const int blocks = (f_end - f_begin + kWideFeat - 1) / kWideFeat;
  for (int i = threadIdx.x; i < kWideRows2; i += kWideThreads) {
    const int tok = i < r.n ? g.order[r.p0 + i] : -1;
    row_of[i] = tok >= 0 && tok < g.M ? tok : -1;
  }
  if (r.adapter < 0) {  // rows without an adapter: out = base
    __syncthreads();
    grid_dep_wait();
    const int vecs = (f_end - f_begin) / 8;
    for (int i = threadIdx.x; i < r.n * vecs; i += kWideThreads) {
      const int tok = row_of[i / vecs], f = f_begin + i % vecs * 8;
      if (tok >= 0)
        *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + tok * g.ld_out + f) =
            *reinterpret_cast<const uint4*>(static_cast<const T*>(g.base) + tok * g.ld_base + f);
    }
    return;
  }
  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&b_full[b]), 1);
      mbar_init(smem_u32(&b_empty[b]), 1);
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), 8);
    }
    failed = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_b);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&tmem_slot), 2 * kWideRows2);
    tmem_relinquish();
  }
  grid_dep_wait();
  // h of this CTA's rows: the parts of K added in order, then split in halves
  const float scale = g.scales ? g.scales[r.adapter] : 1.f;
  const int padded = atoms * 64;
  constexpr int kBatch = 2;  // rows whose loads are in flight together
  for (int row0 = warp * kBatch; row0 < r.n; row0 += kWideThreads / 32 * kBatch) {
    float2 v[kBatch][2] = {};
    for (int part = 0; part < g.parts; ++part) {
      const float* src = g.h + ((int64_t)part * g.M + r.p0 + row0) * g.R + s * g.rank + lane * 2;
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (row0 + q < r.n && i * 64 + lane * 2 < g.rank) {
            const float2 u = *reinterpret_cast<const float2*>(src + (int64_t)q * g.R + i * 64);
            v[q][i].x += u.x, v[q][i].y += u.y;
          }
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int row = row0 + q;
      const int e = row_exponent<T>(fmaxf(fmaxf(fabsf(v[q][0].x), fabsf(v[q][0].y)), fmaxf(fabsf(v[q][1].x), fabsf(v[q][1].y))));
      const float down = ldexpf(1.f, -e);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i * 64 >= padded) continue;
        T hi[2], lo[2];
        halves<T>(v[q][i].x * down, &hi[0], &lo[0]);
        halves<T>(v[q][i].y * down, &hi[1], &lo[1]);
        const int at = i * kAtomBytes + row * 128 + ((lane * 4) ^ ((row & 7) << 4));
        *reinterpret_cast<uint32_t*>(h_smem + at) = *reinterpret_cast<uint32_t*>(hi);
        *reinterpret_cast<uint32_t*>(h_smem + atoms * kAtomBytes + at) = *reinterpret_cast<uint32_t*>(lo);
      }
      if (lane == 0 && row < kWideRows2) row_scale[row] = scale * ldexpf(1.f, e);
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  bool ok = true;
  if (warp == 8) {  // ------------------------------------------------- B
    const uint64_t keep = policy_evict_last();
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
            tc_mma_f16(tmem + b * kWideRows2, b_desc + at, h_desc + half * atoms * (kAtomBytes >> 4) + at, idesc,
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
    float* turn = turns + group * 32 * kWideFeat;
    uint4 y[4];
    const auto load_base = [&](int f, int first, uint4 (&v)[4]) {  // places first + tk + 8 j
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = first + tk + 8 * j;
        const int tok = i < r.n ? row_of[i] : -1;
        if (tok >= 0 && f < f_end)
          v[j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(g.base) + tok * g.ld_base + f);
      }
    };
    load_base(f_begin + fl, group * 32, y);
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
        const uint32_t at = tmem + b * kWideRows2 + first + ((uint32_t)(warp & 3) << 21);
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
        for (int j = 0; j < 32; ++j) turn[j * kWideFeat + tid] = __uint_as_float(v[j / 16][j % 16]);
        uint4 y_next[4];
        load_base(last ? f + kWideFeat : f, last ? group * 32 : first + 64, y_next);
        named_bar_sync(1 + group, 128);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = first + tk + 8 * j;
          const int tok = i < r.n ? row_of[i] : -1;
          if (tok >= 0 && f < f_end) {
            const float w = row_scale[i];
            const float4 p0 = *reinterpret_cast<const float4*>(turn + (tk + 8 * j) * kWideFeat + fl);
            const float4 p1 = *reinterpret_cast<const float4*>(turn + (tk + 8 * j) * kWideFeat + fl + 4);
            float o[8];
            unpack_vec<T>(y[j], o);
            o[0] += w * p0.x, o[1] += w * p0.y, o[2] += w * p0.z, o[3] += w * p0.w;
            o[4] += w * p1.x, o[5] += w * p1.y, o[6] += w * p1.z, o[7] += w * p1.w;
            *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + tok * g.ld_out + f) = pack_vec<T>(o);
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
  if (failed) {  // a wait gave up: leave copies and products in flight time to end
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 10000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kWideRows2);
  }
}

}  // namespace
}  // namespace awqb
