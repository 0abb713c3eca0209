// Tensor-core kernels of the linear cross entropy (see lce.h for the kinds and
// include/ttt_ops.h for the formulas).
//
// One persistent kernel template: each CTA walks a list of output tiles;
//   warps 0..7  epilogue: warp w owns TMEM lanes 32*(w%4)..+31 (one tile row per
//               thread) and one half of the tile's columns (w/4)
//   warp 8      TMA producer of the operand ring
//   warp 9      MMA issuer, into one of two accumulator buffers in TMEM, so that
//               a tile's products run while the previous tile is read out
// The logits never leave the chip: the statistics kinds reduce them to two
// floats per row and half tile, the gradient kinds turn them into the 16-bit
// derivative of the logits of one piece of the vocabulary, which the product
// kinds contract with w and h.
#include "attn_pipe.cuh"
#include "lce.h"

namespace ttt {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

TTT_DEV void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(smem_u32(src))
               : "memory");
}

// One TMEM column of this thread's lane.
TTT_DEV float tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;\n"
               : "=r"(r)
               : "r"(taddr)
               : "memory");
  return __uint_as_float(r);
}

// Named barrier over the 128 threads of one column half.
TTT_DEV void half_bar(int half) { asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory"); }
// The same with a vote: true if every thread's ok is (so that all leave together).
TTT_DEV bool half_all(int half, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(1 + half), "r"(ok ? 1u : 0u)
      : "memory");
  return r != 0;
}

template <int KIND>
struct LceCfg {
  static constexpr bool LOGIT = KIND <= kLceDualGrad;
  static constexpr bool DUAL = KIND == kLceDualStats || KIND == kLceDualGrad;
  static constexpr bool GRAD = KIND == kLceGrad || KIND == kLceDualGrad;
  static constexpr int BM = kLceBM, BN = DUAL ? kLceBNDual : kLceBN, BK = kLceBK;
  static constexpr int TILE_A = BM * BK * 2, TILE_B = BN * BK * 2;
  static constexpr int STAGE = (DUAL ? 2 : 1) * (TILE_A + TILE_B);
  static constexpr int NSTAGE = DUAL ? 3 : 4;
  static constexpr int PANEL = BM * 128;  // staging of one [128 x 64] 16-bit store box
  static constexpr int OFF_STORE = NSTAGE * STAGE;
  static constexpr int OFF_BAR = OFF_STORE + 2 * PANEL;
  static constexpr int NBAR = 2 * NSTAGE + 5;
  static constexpr int SMEM = OFF_BAR + NBAR * 8 + 16 + 1024;
  static constexpr int NTHREADS = 320, WARP_LOAD = 8, WARP_MMA = 9;
  static constexpr int HALF = BN / 2;  // columns (of each accumulator) per epilogue half
  static_assert(SMEM <= 232448, "tile set exceeds shared memory");
};

// Tile t of the list, and its contraction range [k0, k1) in 64-wide steps.
struct LceTile {
  int m, n, split, k0, k1;
};

template <int KIND>
TTT_DEV int lce_tiles(const LceGemm& p, int n_active) {
  using C = LceCfg<KIND>;
  const int mt = (n_active + C::BM - 1) / C::BM, dt = (p.dim + C::BN - 1) / C::BN;
  if constexpr (C::LOGIT) return mt * ((p.cols + C::BN - 1) / C::BN);
  if constexpr (KIND == kLceDH) return mt * dt * p.splits;
  return ((p.cols + C::BM - 1) / C::BM) * dt;
}
template <int KIND>
TTT_DEV LceTile lce_tile(const LceGemm& p, int n_active, int t) {
  using C = LceCfg<KIND>;
  const int mt = (n_active + C::BM - 1) / C::BM, dt = (p.dim + C::BN - 1) / C::BN;
  if constexpr (C::LOGIT) {
    // token tiles fastest: the CTAs running together share a few vocabulary tiles
    return {t % mt, t / mt, 0, 0, (p.dim + C::BK - 1) / C::BK};
  } else if constexpr (KIND == kLceDH) {
    const int s = t / (dt * mt), kt = (p.cols + C::BK - 1) / C::BK;
    return {(t / dt) % mt, t % dt, s, split_begin(kt, s, p.splits), split_begin(kt, s + 1, p.splits)};
  } else {
    return {t / dt, t % dt, 0, 0, (n_active + C::BK - 1) / C::BK};
  }
}

// Packs 64 columns of a row into the half's staging panel and stores the
// panel's box at (x, y); all 128 threads of the half call this.
template <bool BF16>
TTT_DEV void store_panel(uint8_t* panel, const CUtensorMap* map, int half, int r, int x, int y, const float (&v)[64]) {
  uint32_t w[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) w[j] = pack2<BF16>(v[2 * j], v[2 * j + 1]);
  if (r == 0) bulk_wait_read();  // the previous store has left the panel
  half_bar(half);
#pragma unroll
  for (int ch = 0; ch < 8; ++ch)
    *reinterpret_cast<uint4*>(panel + r * 128 + ((ch ^ (r & 7)) << 4)) =
        make_uint4(w[4 * ch], w[4 * ch + 1], w[4 * ch + 2], w[4 * ch + 3]);
  fence_async_smem();
  half_bar(half);
  if (r == 0) {
    tma_store_2d(map, panel, x, y);
    bulk_commit();
  }
}

template <int KIND, bool BF16>
__global__ void __launch_bounds__(LceCfg<KIND>::NTHREADS, 1) lce_gemm_kernel(const __grid_constant__ LceGemm p) {
  using C = LceCfg<KIND>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* full = bars;                       // [NSTAGE] TMA -> MMA
  uint64_t* empty = bars + C::NSTAGE;          // [NSTAGE] MMA -> TMA
  uint64_t* acc_full = bars + 2 * C::NSTAGE;   // [2] MMA -> epilogue
  uint64_t* acc_free = acc_full + 2;           // [2] epilogue (256 arrivals) -> MMA
  uint64_t* drain = acc_full + 4;              // MMA issuer's last commit
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::NBAR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::NBAR; ++i) mbar_init(bars + i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(acc_free + i, 256);
    *abort_flag = (p.err != nullptr && *reinterpret_cast<volatile int*>(p.err) != 0) ? 1 : 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (*abort_flag) return;
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Guard g{abort_flag, p.err, p.err_host};
  const int n_active = p.head->n_active;
  const int n_tiles = lce_tiles<KIND>(p, n_active);
  const bool seg0 = (p.seg_mask & 1) != 0, seg1 = (p.seg_mask & 2) != 0;

  if (warp == C::WARP_LOAD) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint32_t dual_bytes = 16384u * (2 + (seg0 ? 1 : 0) + (seg1 ? 1 : 0));
      int it = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < n_tiles; t += gridDim.x) {
        const LceTile tl = lce_tile<KIND>(p, n_active, t);
        for (int seg = 0; ok && seg < (C::LOGIT ? 1 : 2); ++seg) {
          if (!C::LOGIT && !(seg == 0 ? seg0 : seg1)) continue;
          for (int k = tl.k0; k < tl.k1; ++k, ++it) {
            const int s = it % C::NSTAGE;
            if (it >= C::NSTAGE && !(ok = mbar_wait(empty + s, ((it / C::NSTAGE) - 1) & 1, g, 0x51))) break;
            uint8_t* st = smem + s * C::STAGE;
            if constexpr (C::DUAL) {
              mbar_arrive_tx(full + s, dual_bytes);
              tma_load_2d(st, &p.a[0], full + s, k * C::BK, tl.m * C::BM);
              if (seg0) tma_load_2d(st + C::TILE_A, &p.a[1], full + s, k * C::BK, tl.m * C::BM);
              tma_load_2d(st + 2 * C::TILE_A, &p.b[0], full + s, k * C::BK, tl.n * C::BN);
              if (seg1)
                tma_load_2d(st + 2 * C::TILE_A + C::TILE_B, &p.b[1], full + s, k * C::BK, tl.n * C::BN);
            } else {
              mbar_arrive_tx(full + s, C::STAGE);
              if constexpr (KIND == kLceDW) {
                for (int q = 0; q < 2; ++q)
                  tma_load_2d(st + q * 8192, &p.a[seg], full + s, tl.m * C::BM + q * 64, k * C::BK);
              } else {
                tma_load_2d(st, &p.a[seg], full + s, k * C::BK, tl.m * C::BM);
              }
              if constexpr (C::LOGIT) {
                tma_load_2d(st + C::TILE_A, &p.b[0], full + s, k * C::BK, tl.n * C::BN);
              } else {
                for (int q = 0; q < 4; ++q)
                  tma_load_2d(st + C::TILE_A + q * 8192, &p.b[seg], full + s, tl.n * C::BN + q * 64, k * C::BK);
              }
            }
          }
        }
      }
      for (int j = max(0, it - C::NSTAGE); j < it; ++j) mbar_drain(full + j % C::NSTAGE, (j / C::NSTAGE) & 1);
    }
  } else if (warp == C::WARP_MMA) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr bool A_MN = KIND == kLceDW, B_MN = !C::LOGIT;
      constexpr uint32_t idesc = idesc_f16(C::BM, C::BN, BF16, A_MN, B_MN);
      auto da = [](uint32_t tile, int kk) { return A_MN ? desc_mnmajor(tile, C::BK, kk) : desc_kmajor(tile, C::BM, kk); };
      auto db = [](uint32_t tile, int kk) { return B_MN ? desc_mnmajor(tile, C::BK, kk) : desc_kmajor(tile, C::BN, kk); };
      int it = 0, nth = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < n_tiles; t += gridDim.x) {
        const LceTile tl = lce_tile<KIND>(p, n_active, t);
        const int steps = (tl.k1 - tl.k0) * (C::LOGIT ? 1 : (seg0 ? 1 : 0) + (seg1 ? 1 : 0));
        if (steps == 0) continue;  // the epilogue writes zeros by itself
        const int buf = nth & 1;
        if (nth >= 2 && !(ok = mbar_wait(acc_free + buf, ((nth >> 1) - 1) & 1, g, 0x52))) break;
        const uint32_t d = tmem + buf * 256;
        for (int k = 0; k < steps; ++k, ++it) {
          const int s = it % C::NSTAGE;
          if (!(ok = mbar_wait(full + s, (it / C::NSTAGE) & 1, g, 0x53))) break;
          tc_fence_after();
          const uint32_t st = smem_u32(smem + s * C::STAGE);
          if constexpr (C::DUAL) {
            const uint32_t a0 = st, a1 = st + C::TILE_A, b0 = st + 2 * C::TILE_A, b1 = b0 + C::TILE_B;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) umma_ss(d, da(a0, kk), db(b0, kk), idesc, (k | kk) ? 1u : 0u);
            if (seg0) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) umma_ss(d + C::BN, da(a1, kk), db(b0, kk), idesc, (k | kk) ? 1u : 0u);
            }
            if (seg1) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_ss(d + C::BN, da(a0, kk), db(b1, kk), idesc, (seg0 || (k | kk)) ? 1u : 0u);
            }
          } else {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_ss(d, da(st, kk), db(st + C::TILE_A, kk), idesc, (k | kk) ? 1u : 0u);
          }
          umma_commit(empty + s);
        }
        if (!ok) break;
        umma_commit(acc_full + buf);
        ++nth;
      }
      umma_commit(drain);
      mbar_drain(drain, 0);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = warp >> 2;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    uint8_t* panel = smem + C::OFF_STORE + half * C::PANEL;
    const float inv = (KIND == kLceDW) ? p.scale->inv : 1.f;
    const float mul = C::GRAD ? p.scale->scale : 1.f;
    int nth = 0;
    for (int t = blockIdx.x; t < n_tiles; t += gridDim.x) {
      const LceTile tl = lce_tile<KIND>(p, n_active, t);
      const bool have = tl.k1 > tl.k0 && (C::LOGIT || p.seg_mask != 0);
      const int buf = nth & 1;
      bool ok = true;
      if (have) {
        ok = mbar_wait(acc_full + buf, (nth >> 1) & 1, g, 0x54);
        ++nth;
      }
      if constexpr (C::GRAD) ok = half_all(half, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + lane_off + buf * 256 + half * C::HALF;
      const int slot = tl.m * C::BM + r;
      const int c0 = tl.n * C::BN + half * C::HALF;  // first column within the piece (logit kinds)

      if constexpr (KIND == kLceStats) {
        const int target = p.tgt[slot] - p.col0;
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int q = 0; q < C::HALF / 64; ++q) {
          float v[64];
          tmem_ld_nw<64>(acc + q * 64, v);
          tmem_wait_ld();
          reg_fence(v);
          const int cq = c0 + q * 64;
          if (cq + 64 > p.cols) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = cq + j < p.cols ? v[j] : -INFINITY;
          }
          float m = v[0];
#pragma unroll
          for (int j = 1; j < 64; ++j) m = fmaxf(m, v[j]);
          m = fmaxf(m, mx);
          const float sub = m == -INFINITY ? 0.f : m * kLog2e;  // nothing seen yet: all exponentials are 0
          sum *= fast_exp2(mx * kLog2e - sub);
#pragma unroll
          for (int j = 0; j < 64; ++j) sum += fast_exp2(fmaf(v[j], kLog2e, -sub));
          mx = m;
        }
        // the target's logit, for the few rows whose target lies in these columns
        unsigned hit = __ballot_sync(0xffffffffu, target >= c0 && target < min(c0 + C::HALF, p.cols));
        while (hit != 0) {
          const int src = __ffs(hit) - 1;
          hit &= hit - 1;
          const int col = __shfl_sync(0xffffffffu, target, src) - c0;
          const float z = tmem_ld1(acc + col);
          if (lane == src) p.ztgt[slot] = z;
        }
        tc_fence_before();
        mbar_arrive(acc_free + buf);
        p.part[static_cast<int64_t>(tl.n * 2 + half) * p.n_pad + slot] = make_float2(mx * kLog2e, sum);
      } else if constexpr (KIND == kLceDualStats) {
        const int target = p.tgt[slot] - p.col0;
        const float lse2 = p.lse2[slot];
        float z[64], v[64];
        tmem_ld_nw<64>(acc, z);
        tmem_ld_nw<64>(acc + C::BN, v);
        tmem_wait_ld();
        reg_fence(z);
        reg_fence(v);
        float sum = 0.f, big = 0.f;
#pragma unroll
        for (int j = 0; j < 64; ++j) {
          float x = fast_exp2(fmaf(z[j], kLog2e, -lse2)) * v[j];
          if (c0 + j >= p.cols) x = 0.f;
          sum += x;
          big = fmaxf(big, fabsf(x));
        }
        unsigned hit = __ballot_sync(0xffffffffu, target >= c0 && target < min(c0 + C::HALF, p.cols));
        while (hit != 0) {
          const int src = __ffs(hit) - 1;
          hit &= hit - 1;
          const int col = __shfl_sync(0xffffffffu, target, src) - c0;
          const float a = tmem_ld1(acc + C::BN + col);
          if (lane == src) p.ztgt[slot] = a;
        }
        tc_fence_before();
        mbar_arrive(acc_free + buf);
        p.part[static_cast<int64_t>(tl.n * 2 + half) * p.n_pad + slot] = make_float2(sum, big);
      } else if constexpr (C::GRAD) {
        const int target = p.tgt[slot] - p.col0;
        const float lse2 = p.lse2[slot], coef = p.coef[slot] * mul;
        const float rho = C::DUAL ? p.rho[slot] : 0.f;
#pragma unroll 1
        for (int q = 0; q < C::HALF / 64; ++q) {
          float v[64];
          tmem_ld_nw<64>(acc + q * 64, v);
          tmem_wait_ld();
          reg_fence(v);
          const int cq = c0 + q * 64;
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = fast_exp2(fmaf(v[j], kLog2e, -lse2));
          if constexpr (C::DUAL) {
            float d[64];
            tmem_ld_nw<64>(acc + C::BN, d);
            tmem_wait_ld();
            reg_fence(d);
            tc_fence_before();
            mbar_arrive(acc_free + buf);
#pragma unroll
            for (int j = 0; j < 64; ++j) d[j] = coef * v[j] * (d[j] - rho);
            store_panel<BF16>(panel, &p.out[1], half, r, cq, tl.m * C::BM, d);
          } else if (q == C::HALF / 64 - 1) {
            tc_fence_before();
            mbar_arrive(acc_free + buf);
          }
          const bool here = target >= cq && target < cq + 64;
          if (__any_sync(0xffffffffu, here)) {
            const int tj = here ? target - cq : -1;
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] -= j == tj ? 1.f : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] *= coef;
          store_panel<BF16>(panel, &p.out[0], half, r, cq, tl.m * C::BM, v);
        }
      } else if constexpr (KIND == kLceDH) {
        float* dst = p.acc + (static_cast<int64_t>(tl.split) * p.n_pad + slot) * p.dim_pad;
#pragma unroll 1
        for (int q = 0; q < C::HALF / 32; ++q) {
          float v[32];
          tmem_ld32(acc + q * 32, v);
          const int cq = c0 + q * 32;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            if (cq + j < p.dim_pad) {
              float4* at = reinterpret_cast<float4*>(dst + cq + j);
              float4 o = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
              if (p.accumulate) {
                const float4 old = *at;
                o.x += old.x, o.y += old.y, o.z += old.z, o.w += old.w;
              }
              *at = o;
            }
          }
        }
        tc_fence_before();
        mbar_arrive(acc_free + buf);
      } else {
        const int row = tl.m * C::BM + r;
        uint16_t* dst = p.dw + static_cast<int64_t>(row) * p.dim;
        const bool wide = (p.dim & 7) == 0;
#pragma unroll 1
        for (int q = 0; q < C::HALF / 32; ++q) {
          float v[32];
          if (have) {
            tmem_ld32(acc + q * 32, v);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          }
          const int cq = c0 + q * 32;
          if (row < p.cols) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              uint4 w;
              w.x = pack2<BF16>(v[j] * inv, v[j + 1] * inv);
              w.y = pack2<BF16>(v[j + 2] * inv, v[j + 3] * inv);
              w.z = pack2<BF16>(v[j + 4] * inv, v[j + 5] * inv);
              w.w = pack2<BF16>(v[j + 6] * inv, v[j + 7] * inv);
              if (wide) {
                if (cq + j < p.dim) *reinterpret_cast<uint4*>(dst + cq + j) = w;
              } else {
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (cq + j + e < p.dim) dst[cq + j + e] = static_cast<uint16_t>(u[e >> 1] >> ((e & 1) * 16));
              }
            }
          }
        }
        if (have) {
          tc_fence_before();
          mbar_arrive(acc_free + buf);
        }
      }
    }
    if (C::GRAD && r == 0) bulk_wait_all();  // this thread's stores have completed
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <int KIND, bool BF16>
cudaError_t launch_kind(const LceGemm& p, int sms, cudaStream_t stream) {
  using C = LceCfg<KIND>;
  auto kern = lce_gemm_kernel<KIND, BF16>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  kern<<<sms, C::NTHREADS, C::SMEM, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_lce_gemm(const LceGemm& p, int kind, bool bf16, int sms, cudaStream_t stream) {
#define TTT_LCE(K_) \
  case K_:          \
    return bf16 ? launch_kind<K_, true>(p, sms, stream) : launch_kind<K_, false>(p, sms, stream);
  switch (kind) {
    TTT_LCE(kLceStats)
    TTT_LCE(kLceGrad)
    TTT_LCE(kLceDualStats)
    TTT_LCE(kLceDualGrad)
    TTT_LCE(kLceDH)
    TTT_LCE(kLceDW)
  }
#undef TTT_LCE
  return cudaErrorInvalidValue;
}

}  // namespace ttt
