// Tensor-core kernels of the linear cross entropy (see lce.h for the kinds and
// include/ttt_ops.h for the formulas).
//
// One persistent kernel template for pairs of CTAs (clusters of two): a pair forms
// 256-row tiles with tcgen05.mma over both SMs (cta_group::2), so that each CTA
// stages its own 128 rows of A and only half of B. That halves the shared-memory
// and L2 traffic of B, which is what bounds the same tiles on single CTAs.
//   warps 0..7  epilogue: warp w owns TMEM lanes 32*(w%4)..+31 (one tile row per
//               thread) and one half of the tile's columns (w/4)
//   warp 8      TMA producer of this CTA's operands; all bytes of a stage arrive on
//               the leader's (even CTA's) barrier
//   warp 9      leader only: MMA issuer, into one of two accumulator buffers in
//               TMEM, so that a tile's products run while the previous one is read
// kLceProd's two kinds of tiles differ in length by up to a factor of ten. There the
// leader's producer takes the next tile from a global counter when it has issued the
// last load of the current one, and passes it on to the pair's other warps: taken in
// order of length by whichever pair is free, all pairs end within one short tile.
// Which pair forms a tile does not change its value.
// The logits never leave the chip: the statistics kinds reduce them to two floats
// per row and half tile, the gradient kinds turn them into the 16-bit derivative of
// the logits of one piece of the vocabulary, which kLceProd contracts with w and h.
//
// Measured at 8192 x 768 x 32000 bf16, each launch on its own: statistics 217 us (1.85
// PFLOP/s, tensor pipe 95 % active), G 258 us, both products 523 us (1.54), statistics of
// (z, A) 694 us (1.74, 99 %), G and D 773 us (85 %), their four products 1080 us (1.49).
// Back to back the GPU's power cap holds the clock near 1.35 GHz and the whole sequence
// runs at 1.25 PFLOP/s (cuBLAS sustains 1.38 there), so what is left is energy, not issue.
#include "attn_pipe.cuh"
#include "lce.h"

namespace ttt {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- pair-of-CTAs helpers
TTT_DEV uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of this CTA's shared variable `p` in CTA `rank` of the pair.
TTT_DEV uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
TTT_DEV void pair_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
TTT_DEV int ld_peer(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
TTT_DEV void st_peer(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
TTT_DEV void arrive_peer(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Acquire at pair scope, for data written by the other CTA before its arrival.
TTT_DEV void acquire_pair() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }

// 2-D tiled load into this CTA's shared memory, its bytes counted on a barrier of the pair.
TTT_DEV void load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
TTT_DEV void umma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Non-blocking look at a barrier phase.
TTT_DEV uint32_t mbar_probe(const uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done;
}

// One thread of the (converged) warp; the same one every time.
TTT_DEV bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r != 0;
}

// Arrive on `bar` of both CTAs when every product issued so far has completed.
TTT_DEV void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
TTT_DEV void tmem_alloc_pair(uint32_t* dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
TTT_DEV void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

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

template <int KIND>
struct LceCfg {
  static constexpr bool LOGIT = KIND != kLceProd;
  static constexpr bool DUAL = KIND == kLceDualStats || KIND == kLceDualGrad;
  static constexpr bool GRAD = KIND == kLceGrad || KIND == kLceDualGrad;
  static constexpr int BM = kLceBM, BN = DUAL ? kLceBNDual : kLceBN;
  // Contraction of a stage, and staging boxes of an epilogue warp. kLceGrad is bound by
  // shared memory: a pair's products read 64 bytes a cycle and their loads write 64 of
  // the 128 that it moves, and the staged G comes on top. With two boxes per warp beside
  // five short stages it keeps 84 % of the tensor pipe at dim 768, with one beside three
  // long ones 78 %, and 16 epilogue warps add nothing; the dual gradient kind needs its
  // fourth stage more than second boxes (87 % against 80 %).
  static constexpr int BK = DUAL || KIND == kLceGrad ? kLcePanel : kLceBK, PANELS = BK / kLcePanel;
  static constexpr int ROWS_A = BM / 2, ROWS_B = BN / 2;  // of a CTA
  static constexpr int TILE_A = ROWS_A * BK * 2, TILE_B = ROWS_B * BK * 2;
  static constexpr int STAGE = (DUAL ? 2 : 1) * (TILE_A + TILE_B);
  static constexpr int PANEL = 32 * 128;  // staging of one warp's [32 x 64] 16-bit store box
  static constexpr int BOXES = KIND == kLceGrad ? 2 : 1;
  static constexpr int NSTAGE = (232448 - 1024 - 256 - 8 * BOXES * PANEL) / STAGE;
  static constexpr int OFF_STORE = NSTAGE * STAGE;
  static constexpr int OFF_BAR = OFF_STORE + 8 * BOXES * PANEL;
  static constexpr int NBAR = 2 * NSTAGE + 9;
  static constexpr int SMEM = OFF_BAR + NBAR * 8 + 32 + 1024;
  static constexpr int NTHREADS = 320, WARP_LOAD = 8, WARP_MMA = 9;
  static constexpr int HALF = BN / 2;  // columns (of each accumulator) per epilogue half
  static_assert(SMEM <= 232448, "tile set exceeds shared memory");
};

// A tile of the list and its contraction range [k0, k1) in 64-wide steps.
struct LceTile {
  int m, n, split, k0, k1;
  bool dw;  // kLceProd: a tile of the weight gradient
};

struct LceSizes {
  int mt, dt, kt, nk, n_dh, n_dw, n_tiles;
  bool dw_first;
};
template <int KIND>
TTT_DEV LceSizes lce_sizes(const LceGemm& p, int n_active) {
  using C = LceCfg<KIND>;
  LceSizes s;
  s.mt = (n_active + C::BM - 1) / C::BM;
  s.dt = (p.dim + C::BN - 1) / C::BN;
  s.kt = (p.cols + C::BK - 1) / C::BK;   // steps over the piece's columns
  s.nk = (n_active + C::BK - 1) / C::BK; // steps over the rows
  if constexpr (C::LOGIT) {
    s.n_tiles = s.mt * ((p.cols + C::BN - 1) / C::BN);
  } else {
    s.n_dh = p.acc != nullptr ? s.mt * s.dt * p.splits : 0;
    s.n_dw = p.dw != nullptr ? ((p.cols + C::BM - 1) / C::BM) * s.dt : 0;
    s.n_tiles = s.n_dh + s.n_dw;
    s.dw_first = s.nk * __popc(p.seg_h) > s.kt / p.splits * __popc(p.seg_w);  // longer tiles first
  }
  return s;
}
template <int KIND>
TTT_DEV LceTile lce_tile(const LceGemm& p, const LceSizes& s, int t) {
  using C = LceCfg<KIND>;
  if constexpr (C::LOGIT) {
    // token tiles fastest: the pairs running together share a few vocabulary tiles
    return {t % s.mt, t / s.mt, 0, 0, (p.dim + C::BK - 1) / C::BK, false};
  } else {
    const bool dw = s.dw_first ? t < s.n_dw : t >= s.n_dh;
    const int i = dw ? (s.dw_first ? t : t - s.n_dh) : (s.dw_first ? t - s.n_dw : t);
    if (dw) return {i / s.dt, i % s.dt, 0, 0, s.nk, true};
    const int sp = i / (s.dt * s.mt);
    return {(i / s.dt) % s.mt, i % s.dt, sp, split_begin(s.kt, sp, p.splits), split_begin(s.kt, sp + 1, p.splits),
            false};
  }
}

// Walks the tiles of this pair: a fixed stride, or (kLceProd) what the leader's
// producer takes from the counter and writes into a two-entry ring in both CTAs'
// shared memory. Used by one warp (the epilogue) or one thread (producer, issuer).
enum LceRole { kTaker, kThread, kWarp };
template <int KIND>
struct LceWalk {
  int i = 0, pairs, pair, n_tiles;
  uint32_t rank;
  unsigned* ticket;
  volatile int* ring;
  uint64_t *full, *empty;
  // The next tile, or -1 at the end (or when aborting).
  template <LceRole ROLE>
  TTT_DEV int next(const Guard& g) {
    if constexpr (KIND != kLceProd) {
      const int t = pair + i * pairs;
      ++i;
      return t < n_tiles ? t : -1;
    } else {
      const int slot = i & 1;
      int t;
      if (ROLE == kTaker && rank == 0) {
        if (i >= 2 && !mbar_wait(empty + slot, ((i >> 1) - 1) & 1, g, 0x56)) return -1;
        t = static_cast<int>(min(atomicAdd(ticket, 1u), 0x7fffffffu));
        ring[slot] = t;
        st_peer(peer_addr(const_cast<const int*>(ring) + slot, 1), t);
        mbar_arrive(full + slot);
        arrive_peer(peer_addr(full + slot, 1));
      } else {
        bool ok = mbar_wait(full + slot, (i >> 1) & 1, g, 0x55);
        if constexpr (ROLE == kWarp) ok = __all_sync(0xffffffffu, ok);
        if (!ok) return -1;
        acquire_pair();
        t = ring[slot];
        if constexpr (ROLE == kWarp) __syncwarp();  // every lane has read the entry
        if (ROLE != kWarp || (threadIdx.x & 31) == 0) arrive_peer(peer_addr(empty + slot, 0));
      }
      ++i;
      return t < n_tiles ? t : -1;
    }
  }
};

// Packs 64 columns of this warp's 32 rows into a staging box (128-byte swizzle).
template <bool BF16>
TTT_DEV void write_box(uint8_t* box, int lane, const float (&v)[64]) {
  uint32_t w[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) w[j] = pack2<BF16>(v[2 * j], v[2 * j + 1]);
#pragma unroll
  for (int ch = 0; ch < 8; ++ch)
    *reinterpret_cast<uint4*>(box + lane * 128 + ((ch ^ (lane & 7)) << 4)) =
        make_uint4(w[4 * ch], w[4 * ch + 1], w[4 * ch + 2], w[4 * ch + 3]);
}
// ... into one of the warp's BOXES staging boxes (in turn: `turn` counts them), stored at (x, y).
template <bool BF16, int BOXES>
TTT_DEV void store_panel(uint8_t* panel, int& turn, const CUtensorMap* map, int lane, int x, int y,
                         const float (&v)[64]) {
  panel += (turn % BOXES) * 4096;
  ++turn;
  // the box's previous store has left it
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(BOXES - 1) : "memory");
  __syncwarp();
  write_box<BF16>(panel, lane, v);
  fence_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map, panel, x, y);
    bulk_commit();
  }
}

template <int KIND, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LceCfg<KIND>::NTHREADS, 1)
    lce_gemm_kernel(const __grid_constant__ LceGemm p) {
  using C = LceCfg<KIND>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* full = bars;                      // [NSTAGE] leader's: both CTAs' loads -> MMA
  uint64_t* empty = bars + C::NSTAGE;         // [NSTAGE] each CTA's: MMA -> its producer
  uint64_t* acc_full = bars + 2 * C::NSTAGE;  // [2] each CTA's: MMA -> its epilogue
  uint64_t* acc_free = acc_full + 2;          // [2] leader's: 16 epilogue warps -> MMA
  uint64_t* drain = acc_full + 4;             // each CTA's: the issuer's last commit
  uint64_t* sched_full = acc_full + 5;        // [2] each CTA's: a ring entry is there
  uint64_t* sched_empty = acc_full + 7;       // [2] leader's: its 18 readers have it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::NBAR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* ring = reinterpret_cast<volatile int*>(tmem_slot + 2);  // [2]

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  asm volatile("griddepcontrol.launch_dependents;");
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::NBAR; ++i) mbar_init(bars + i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_free + i, 16);
      mbar_init(sched_empty + i, 18);
    }
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 0) tmem_alloc_pair(tmem_slot, 512);
  // everything below reads what earlier kernels of the stream wrote
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0) *abort_flag = (p.err != nullptr && *reinterpret_cast<volatile int*>(p.err) != 0) ? 1 : 0;
  tc_fence_before();
  __syncthreads();
  pair_sync();
  tc_fence_after();
  // both CTAs work or neither does
  const bool go = *abort_flag == 0 && ld_peer(peer_addr(const_cast<const int*>(abort_flag), rank ^ 1)) == 0;
  pair_sync();
  const uint32_t tmem = *tmem_slot;
  Guard g{abort_flag, p.err, p.err_host};
  const int n_active = p.head->n_active;
  const LceSizes sz = lce_sizes<KIND>(p, n_active);
  LceWalk<KIND> walk;
  walk.pairs = static_cast<int>(gridDim.x) >> 1;
  walk.pair = static_cast<int>(blockIdx.x) >> 1;
  walk.n_tiles = sz.n_tiles;
  walk.rank = rank;
  walk.ticket = p.ticket;
  walk.ring = ring;
  walk.full = sched_full;
  walk.empty = sched_empty;
  const bool seg0 = (p.seg_w & 1) != 0, seg1 = (p.seg_w & 2) != 0;  // dual kinds
  if (C::GRAD && go && blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;  // for the products that follow

  if (go && warp == C::WARP_LOAD) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint32_t dual_bytes = 2u * (C::TILE_A * (seg0 ? 2 : 1) + C::TILE_B * (seg1 ? 2 : 1));
      const int row_a = static_cast<int>(rank) * C::ROWS_A, row_b = static_cast<int>(rank) * C::ROWS_B;
      int it = 0;
      bool ok = true;
      for (int t; ok && (t = walk.template next<kTaker>(g)) >= 0;) {
        const LceTile tl = lce_tile<KIND>(p, sz, t);
        const int segs = C::LOGIT ? 1 : (tl.dw ? p.seg_h : p.seg_w);
        for (int seg = 0; ok && seg < 2; ++seg) {
          if (!(segs >> seg & 1)) continue;
          for (int k = tl.k0; k < tl.k1; ++k, ++it) {
            const int s = it % C::NSTAGE;
            if (it >= C::NSTAGE && !(ok = mbar_wait(empty + s, ((it / C::NSTAGE) - 1) & 1, g, 0x51))) break;
            uint8_t* st = smem + s * C::STAGE;
            uint8_t* stb = st + (C::DUAL ? 2 : 1) * C::TILE_A;
            if (rank == 0) mbar_arrive_tx(full + s, C::DUAL ? dual_bytes : 2u * C::STAGE);
            const uint32_t bar = peer_addr(full + s, 0);
            const int kc = k * C::BK;
            if constexpr (C::LOGIT) {
              for (int q = 0; q < C::PANELS; ++q) {
                load_pair(st + q * C::ROWS_A * 128, &p.a[0], bar, kc + q * 64, tl.m * C::BM + row_a);
                load_pair(stb + q * C::ROWS_B * 128, &p.b[0], bar, kc + q * 64, tl.n * C::BN + row_b);
              }
              if constexpr (C::DUAL) {
                if (seg0) load_pair(st + C::TILE_A, &p.a[1], bar, kc, tl.m * C::BM + row_a);
                if (seg1) load_pair(stb + C::TILE_B, &p.b[1], bar, kc, tl.n * C::BN + row_b);
              }
            } else {
              // MN-major panels: BK rows of 64 columns; K-major ones: 128 rows of 64 columns
              const CUtensorMap* b = tl.dw ? &p.bh[seg] : &p.bw[seg];
              for (int q = 0; q < 2; ++q) {
                if (tl.dw)
                  load_pair(st + q * C::BK * 128, &p.gm[seg], bar, tl.m * C::BM + row_a + q * 64, kc);
                else
                  load_pair(st + q * C::ROWS_A * 128, &p.gk[seg], bar, kc + q * 64, tl.m * C::BM + row_a);
                load_pair(stb + q * C::BK * 128, b, bar, tl.n * C::BN + row_b + q * 64, kc);
              }
            }
          }
        }
      }
      if (rank == 0)
        for (int j = max(0, it - C::NSTAGE); j < it; ++j) mbar_drain(full + j % C::NSTAGE, (j / C::NSTAGE) & 1);
    }
  } else if (go && warp == C::WARP_MMA && rank == 0) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp walks along, so that the compiler keeps descriptors and addresses in
    // uniform registers; one thread issues. A single thread on its own took ~96 cycles a
    // product, more than a 128-wide one lasts: statistics of (z, A) 944 us, 727 like this.
    {
      const bool leader = elect_one();
      constexpr bool B_MN = !C::LOGIT;
      constexpr uint32_t id_k = idesc_f16(C::BM, C::BN, BF16, false, B_MN), id_mn = idesc_f16(C::BM, C::BN, BF16, true, B_MN);
      auto db = [](uint32_t tile, int kk) {
        return B_MN ? desc_mnmajor(tile, C::BK, kk) : desc_kmajor(tile, C::ROWS_B, kk);
      };
      constexpr int KS = C::BK / 16;
      int it = 0, nth = 0;
      bool ready = false, ok = true;  // ready: the next stage has been seen full
      for (int t; ok && (t = walk.template next<kWarp>(g)) >= 0;) {
        const LceTile tl = lce_tile<KIND>(p, sz, t);
        const int steps = (tl.k1 - tl.k0) * (C::LOGIT ? 1 : __popc(tl.dw ? p.seg_h : p.seg_w));
        if (steps == 0) continue;  // the epilogue does without the accumulators
        const int buf = nth & 1;
        if (nth >= 2 && !(ok = __all_sync(0xffffffffu, mbar_wait(acc_free + buf, ((nth >> 1) - 1) & 1, g, 0x52)))) break;
        const uint32_t d = tmem + buf * 256;
        for (int k = 0; k < steps; ++k, ++it) {
          const int s = it % C::NSTAGE;
          if (!ready && !(ok = __all_sync(0xffffffffu, mbar_wait(full + s, (it / C::NSTAGE) & 1, g, 0x53)))) break;
          tc_fence_after();
          const uint32_t st = smem_u32(smem + s * C::STAGE);
          const uint64_t* next_full = full + (it + 1) % C::NSTAGE;
          const uint32_t next_par = ((it + 1) / C::NSTAGE) & 1;
          if (leader) {
          if constexpr (C::DUAL) {
            const uint32_t a0 = st, a1 = st + C::TILE_A, b0 = st + 2 * C::TILE_A, b1 = b0 + C::TILE_B;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
              umma_pair(d, desc_kmajor(a0, C::ROWS_A, kk), db(b0, kk), id_k, (k | kk) ? 1u : 0u);
            if (seg0) {
#pragma unroll
              for (int kk = 0; kk < KS; ++kk)
                umma_pair(d + C::BN, desc_kmajor(a1, C::ROWS_A, kk), db(b0, kk), id_k, (k | kk) ? 1u : 0u);
            }
            if (seg1) {
#pragma unroll
              for (int kk = 0; kk < KS; ++kk)
                umma_pair(d + C::BN, desc_kmajor(a0, C::ROWS_A, kk), db(b1, kk), id_k, (seg0 || (k | kk)) ? 1u : 0u);
            }
          } else if (!C::LOGIT && tl.dw) {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
              umma_pair(d, desc_mnmajor(st, C::BK, kk), db(st + C::TILE_A, kk), id_mn, (k | kk) ? 1u : 0u);
          } else {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
              umma_pair(d, desc_kmajor(st, C::ROWS_A, kk), db(st + C::TILE_A, kk), id_k, (k | kk) ? 1u : 0u);
          }
          commit_pair(empty + s);
          }
          __syncwarp();
          ready = __all_sync(0xffffffffu, mbar_probe(next_full, next_par) != 0);
        }
        if (!ok) break;
        if (leader) commit_pair(acc_full + buf);
        __syncwarp();
        ++nth;
      }
      if (leader) commit_pair(drain);
      __syncwarp();
      mbar_drain(drain, 0);
    }
  } else if (go && warp < 8) {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = warp >> 2;
    const int r = static_cast<int>(rank) * C::ROWS_A + quarter * 32 + lane;  // row of the tile
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    uint8_t* panel = smem + C::OFF_STORE + warp * C::BOXES * C::PANEL;
    int turn = 0;
    const uint32_t free_leader = peer_addr(acc_free, 0);
    const float mul = C::GRAD ? p.coef.scale() : (KIND == kLceProd ? p.coef.out() : 1.f);
    int nth = 0;
    for (int t; (t = walk.template next<kWarp>(g)) >= 0;) {
      const LceTile tl = lce_tile<KIND>(p, sz, t);
      const bool have = tl.k1 > tl.k0 && (C::LOGIT || (tl.dw ? p.seg_h : p.seg_w) != 0);
      const int buf = nth & 1;
      if (have) {
        if (!__all_sync(0xffffffffu, mbar_wait(acc_full + buf, (nth >> 1) & 1, g, 0x54))) break;
        ++nth;
      }
      tc_fence_after();
      // the accumulators are in registers: the issuer may use the buffer again
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_peer(free_leader + buf * 8);
      };
      const uint32_t acc = tmem + lane_off + buf * 256 + half * C::HALF;
      const int slot = tl.m * C::BM + r;
      const int c0 = tl.n * C::BN + half * C::HALF;  // first column of this half

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
          // Nothing seen yet: all exponentials are 0. The maximum's product with log2 e is rounded alike
          // here and in what is written out, so that its rounding cancels in the loss.
          const float sub = m == -INFINITY ? 0.f : __fmul_rn(m, kLog2e);
          sum *= fast_exp2(__fmul_rn(mx, kLog2e) - sub);
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
        release();
        p.part[static_cast<int64_t>(tl.n * 2 + half) * p.n_pad + slot] = make_float2(__fmul_rn(mx, kLog2e), sum);
      } else if constexpr (KIND == kLceDualStats) {
        const int target = p.tgt[slot] - p.col0;
        const float top2 = p.top2[slot], inv_l = p.inv_l[slot];
        float z[64], v[64];
        tmem_ld_nw<64>(acc, z);
        tmem_ld_nw<64>(acc + C::BN, v);
        tmem_wait_ld();
        reg_fence(z);
        reg_fence(v);
        float sum = 0.f, big = 0.f;
#pragma unroll
        for (int j = 0; j < 64; ++j) {
          float x = fast_exp2(fmaf(z[j], kLog2e, -top2)) * v[j];
          if (c0 + j >= p.cols) x = 0.f;
          sum += x;
          big = fmaxf(big, fabsf(x));
        }
        sum *= inv_l;
        big *= inv_l;
        unsigned hit = __ballot_sync(0xffffffffu, target >= c0 && target < min(c0 + C::HALF, p.cols));
        while (hit != 0) {
          const int src = __ffs(hit) - 1;
          hit &= hit - 1;
          const int col = __shfl_sync(0xffffffffu, target, src) - c0;
          const float a = tmem_ld1(acc + C::BN + col);
          if (lane == src) p.ztgt[slot] = a;
        }
        release();
        p.part[static_cast<int64_t>(tl.n * 2 + half) * p.n_pad + slot] = make_float2(sum, big);
      } else if constexpr (C::GRAD) {
        const int target = p.tgt[slot] - p.col0;
        const float top2 = p.top2[slot], coef = slot < n_active ? p.coef.row(slot) * mul : 0.f;
        const float coef_l = coef * p.inv_l[slot];  // c p = coef_l * exp2(z log2 e - top2)
        const float rho = C::DUAL ? p.rho[slot] : 0.f;
        const int row0 = tl.m * C::BM + static_cast<int>(rank) * C::ROWS_A + quarter * 32;
#pragma unroll 1
        for (int q = 0; q < C::HALF / 64; ++q) {
          float v[64];
          tmem_ld_nw<64>(acc + q * 64, v);
          tmem_wait_ld();
          reg_fence(v);
          const int cq = c0 + q * 64;
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = fast_exp2(fmaf(v[j], kLog2e, -top2));
          if constexpr (C::DUAL) {
            float d[64];
            tmem_ld_nw<64>(acc + C::BN, d);
            tmem_wait_ld();
            reg_fence(d);
            release();
#pragma unroll
            for (int j = 0; j < 64; ++j) d[j] = coef_l * v[j] * (d[j] - rho);
            store_panel<BF16, C::BOXES>(panel, turn, &p.out[1], lane, cq, row0, d);
          } else if (q == C::HALF / 64 - 1) {
            release();
          }
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] *= coef_l;
          const bool here = target >= cq && target < cq + 64;
          if (__any_sync(0xffffffffu, here)) {
            const int tj = here ? target - cq : -1;
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] -= j == tj ? coef : 0.f;
          }
          store_panel<BF16, C::BOXES>(panel, turn, &p.out[0], lane, cq, row0, v);
        }
      } else if (!tl.dw) {
        // A share without columns adds nothing to the partial rows. Only a last piece can be that
        // short (the plan gives every share of the first one some steps), and an earlier piece
        // has written them.
        if (!have) continue;
        float* dst = p.acc + (static_cast<int64_t>(tl.split) * p.n_pad + slot) * p.dim_pad;
#pragma unroll 1
        for (int q = 0; q < C::HALF / 32; ++q) {
          float v[32];
          tmem_ld32(acc + q * 32, v);
          if (q == C::HALF / 32 - 1) release();
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
      } else {
        const bool boxes = (p.dim & 7) == 0;  // else the rows are not aligned for tensor-map stores
        const int row0 = tl.m * C::BM + static_cast<int>(rank) * C::ROWS_A + quarter * 32;
#pragma unroll 1
        for (int q = 0; q < C::HALF / 64; ++q) {
          float v[64];
          if (have) {
            tmem_ld_nw<64>(acc + q * 64, v);
            tmem_wait_ld();
            reg_fence(v);
            if (q == C::HALF / 64 - 1) release();
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] *= mul;
          } else {  // no row takes part: zeros, whatever the upstream value is
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = 0.f;
          }
          const int cq = c0 + q * 64;
          if (cq >= p.dim || row0 >= p.cols) continue;
          if (boxes) {
            store_panel<BF16, C::BOXES>(panel, turn, &p.dw_out, lane, cq, row0, v);
          } else {
            // through the staging box as well, then row by row: consecutive lanes write
            // consecutive columns, a pair each where rows start on 4 bytes
            __syncwarp();
            write_box<BF16>(panel, lane, v);
            __syncwarp();
            auto at = [&](int i, int c) { return panel + i * 128 + (((c >> 3) ^ (i & 7)) << 4) + (c & 7) * 2; };
            const int rows = min(32, p.cols - row0), cols = min(64, p.dim - cq);
            uint16_t* dst = p.dw + static_cast<int64_t>(row0) * p.dim + cq;
            if ((p.dim & 1) == 0) {
              if (2 * lane < cols) {
#pragma unroll 8
                for (int i = 0; i < rows; ++i)
                  *reinterpret_cast<uint32_t*>(dst + static_cast<int64_t>(i) * p.dim + 2 * lane) =
                      *reinterpret_cast<const uint32_t*>(at(i, 2 * lane));
              }
            } else {
#pragma unroll 8
              for (int i = 0; i < rows; ++i) {
                uint16_t* to = dst + static_cast<int64_t>(i) * p.dim + lane;
                if (lane < cols) to[0] = *reinterpret_cast<const uint16_t*>(at(i, lane));
                if (lane + 32 < cols) to[32] = *reinterpret_cast<const uint16_t*>(at(i, lane + 32));
              }
            }
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();  // this thread's stores have completed
  }

  // No CTA leaves while the other may still signal its barriers. After an abort, a
  // millisecond lets this CTA's own loads land before its shared memory is given up.
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0 && go) {
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 1000000ull) {
    }
  }
  pair_sync();
  tc_fence_after();
  if (warp == 0) tmem_dealloc_pair(tmem, 512);
}

template <int KIND, bool BF16>
cudaError_t launch_kind(const LceGemm& p, int sms, cudaStream_t stream) {
  using C = LceCfg<KIND>;
  auto kern = lce_gemm_kernel<KIND, BF16>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute early;  // the prologue may overlap the previous kernel's end (griddepcontrol.wait)
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(sms < 2 ? 2 : sms & ~1));
  cfg.blockDim = dim3(C::NTHREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
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
    TTT_LCE(kLceProd)
  }
#undef TTT_LCE
  return cudaErrorInvalidValue;
}

}  // namespace ttt
