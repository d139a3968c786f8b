// Causal attention over packed sequences with grouped heads, on the 5th-generation tensor
// cores:  o_i = sum_j p_ij v_j,  p_ij = 2^(c2 q_i . k_j - lse2_i)  (log2 units), one pass over
// the keys with a running maximum and sum.
//
// A row tile is 128 / G tokens times the G heads of one kv head (128 rows, brought in by one
// 3-D tensor-map box), so that the group shares its K and V; a work item is two row tiles of
// one sequence with the same 128-key tiles of K and V.  One CTA to an SM stays for the whole
// call and takes every gridDim-th item, back and forth, the items with the most keys first.
// Warp roles (384 threads):
//   warp 0      TMA: Q of an item, K and V through two rings, on into the next item;
//   warp 1      issues tcgen05.mma: S_i = Q_i K_j^T (128 x 128, TMEM), O_i += P_i V_j with P_i
//               read from TMEM over its scores; while one tile's softmax runs, the tensor
//               cores have the other tile's P V and the next scores, and while an item's
//               outputs are written, the next item's first scores;
//   warp 2      clears the rows of a sequence's last V tile that belong to the next sequence
//               (0 x their Inf or NaN would reach this one);
//   warp 3      finds the items (which sequence, which keys) and hands them to the others
//               through shared memory, a few ahead;
//   warps 4-7   softmax of row tile 0, warps 8-11 of row tile 1: one thread a row, with the
//               registers that the other warps give up; P leaves in two halves, so that P V
//               of the first runs while the second is computed.
// The running maximum moves, and O is rescaled in TMEM, only past a margin of 2^8; the sums
// are kept in fp32 from the unrounded weights, P is rounded to the inputs' 16-bit type (the
// same relative rounding as the output's: 2.0e-3 off in all against 1.5e-3 of the output's rounding
// alone, bf16).  O is added up in fp32 in TMEM, where a product loses what lies below some 2^-25 of
// the sum so far.  Over very many keys of like weight this adds up, towards zero: measured on
// weights that are all equal 2e-4 (2^17 keys), 5e-4 (2^18), 2.6e-3 (2^20), 1.2e-2 (2^22), below f16's own
// rounding up to 2^17 keys and bf16's up to 2^19.  Parts of a key range (n_splits) are added outside.
// Bound at D = 128: a 128 x 128 tile takes 1024 clocks of the tensor cores and 1024 clocks of
// the exponential unit (16 a clock), which the two row tiles overlap.  Taking 2 of 8 weights
// from a polynomial on the FMA pipe instead was slower (2161 against 1798 us for 16384
// tokens, 32 / 8 heads): the added instructions cost more issue slots and power than they save.
// Measured (32 / 8 heads, D = 128, bf16): 4096 tokens 124 us (1110 TFLOP/s of causal work), 16384
// tokens 1770 to 2000 us (1100 to 1250, by the box's power: at 985 W the SMs run at 1.58 GHz); both units are active 59% of the
// time.  What is in the way is TMEM, which loads of scores share with running products, and the
// wait of a row tile for its own P V and next scores.
// Few rows: the key range is cut into n_splits parts, whose normalised outputs and lse a second
// kernel merges.
#include <cstdio>
#include <type_traits>

#include "launchers.cuh"
#include "packed_tiles.cuh"
#include "sparse_attention_mma.cuh"
#include "umma.cuh"

namespace linattn {

namespace {

struct PackedArgs {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t Nq, Nk;
  int max_q;         // rows of a sequence at most: later ones are not written
  int S, Hq, Hkv, G, tokens;  // tokens of a row tile (floor(128 / G))
  int inv_g;         // ceil(2^16 / G): (r inv_g) >> 16 = r / G for r < 128
  int causal;
  float scale_log2;
  void* out;
  int64_t ot, oh;
  float* lse;        // (N_q, H_q) or NULL
  int n_splits;
  // parts of a cut key range, rows next to one another as a row tile has them (row = token G + head
  // of the group), so that a warp's rows are written and read together
  float4* part_o;    // (n_splits, H_kv, D / 4, N_q G) four channels of a row
  float* part_lse;   // (n_splits, H_kv, N_q G)
  int64_t items;     // at most: tiles x H_kv x n_splits
  uint64_t item_ns;  // limit of a wait for an item's end
  int32_t* status;
};

constexpr int PA_THREADS = 384;
constexpr int PA_ITEMS = 3;  // items handed out ahead
// Registers: 168 a thread at launch; the loading and issuing warpgroup gives up what the two
// softmax warpgroups take (88 + 2 x 208 = 3 x 168).
constexpr int PA_REGS_LOW = 88, PA_REGS_HIGH = 208;

template <int D>
struct PackedSmem {
  static constexpr int TILE = 128 * D * 2;           // Q, K or V tile
  static constexpr int KS = D == 128 ? 2 : 4;        // K ring stages
  static constexpr int VS = D == 128 ? 2 : 4;        // V ring stages
  static constexpr int OUT = 8 * 4096;               // outputs on their way: 32 rows x 64 channels a softmax warp
  static constexpr int BYTES = 1024 + TILE * (2 + KS + VS) + OUT;
};

// One work item: two row tiles of a sequence, a kv head, a part of the keys.
struct PackedItem {
  int q_first, lq, k_first, lk, t0, shift, kvh, split;
  int j0, n0, n1, n;  // first key tile, key tiles of each row tile and of both
  int ragged;         // the key tile that another sequence's rows end, or -1
  int more;           // 0: no item any more
};

// Up to 64 sequences, two to a lane: the pairs of row tiles of all of them from the longest
// key range to the shortest.  Pair x of a sequence has about (x + base) units of keys, so the
// pairs at or above a level are counted in closed form and a level is found by bisection.
// (Sequence after sequence, the static shares of a ragged batch were 35% apart.)
struct PackedOrder {
  int first[2], n[2], other_first[2], other_n[2], base[2], pairs[2];
  bool sound[2];
  int levels;
  __device__ __forceinline__ void load(const PackedArgs& p) {
    const int lane = threadIdx.x & 31;
    levels = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int s = lane + 32 * e;
      first[e] = n[e] = other_first[e] = other_n[e] = 0;
      sound[e] = true;
      if (s < p.S) {
        sound[e] = packed_range(p.cu_q, s, p.Nq, &first[e], &n[e]);
        sound[e] &= packed_range(p.cu_k, s, p.Nk, &other_first[e], &other_n[e]);
      }
      pairs[e] = (min(n[e], p.max_q) + 2 * p.tokens - 1) / (2 * p.tokens);
      base[e] = max(0, other_n[e] - n[e]) / (2 * p.tokens);
      levels = max(levels, base[e] + pairs[e]);
    }
    levels = __reduce_max_sync(0xffffffffu, levels);
  }
  __device__ __forceinline__ int above(int level) const {  // pairs at this level or over it
    int c = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) c += max(0, min(pairs[e], base[e] + pairs[e] - level));
    return __reduce_add_sync(0xffffffffu, c);
  }
  __device__ __forceinline__ bool find(int64_t idx, PackedTile* t) const {
    if (idx >= above(0)) return false;
    int lo = 0, hi = levels;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (idx < above(mid)) lo = mid;
      else hi = mid;
    }
    int rank = static_cast<int>(idx) - above(lo + 1);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool here = lo >= base[e] && lo < base[e] + pairs[e];
      const unsigned mask = __ballot_sync(0xffffffffu, here);
      const unsigned below = mask & ((1u << (threadIdx.x & 31)) - 1u);
      const unsigned owner = __ballot_sync(0xffffffffu, here && __popc(below) == rank);
      if (owner) {
        const int l = __ffs(owner) - 1;
        t->tile = lo - __shfl_sync(0xffffffffu, base[e], l);
        t->first = __shfl_sync(0xffffffffu, first[e], l);
        t->n = __shfl_sync(0xffffffffu, n[e], l);
        t->other_first = __shfl_sync(0xffffffffu, other_first[e], l);
        t->other_n = __shfl_sync(0xffffffffu, other_n[e], l);
        t->sound = __shfl_sync(0xffffffffu, sound[e] ? 1 : 0, l) != 0;
        return true;
      }
      rank -= __popc(mask);
    }
    return false;
  }
};

// The item of this CTA's `turn`-th turn, back and forth over the CTAs (items get smaller: always
// the same order would give the first CTA the largest of every turn).  All lanes of a warp
// together; false past the last item.
__device__ __forceinline__ bool packed_item(const PackedArgs& p, const PackedOrder& order, int64_t turn, PackedItem* w) {
  const int64_t item = turn * gridDim.x + ((turn & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  if (item >= p.items) return false;
  const int per = p.Hkv * p.n_splits;
  const int64_t at = item / per;
  const int rest = static_cast<int>(item - at * per);
  w->kvh = rest / p.n_splits;
  w->split = rest - w->kvh * p.n_splits;
  PackedTile t;
  if (p.S <= 64) {
    if (!order.find(at, &t)) return false;
  } else {  // sequence after sequence, each from its end
    if (!packed_tile(p.cu_q, p.cu_k, p.S, p.Nq, p.Nk, 2 * p.tokens, p.max_q, at, &t)) return false;
    t.tile = (min(t.n, p.max_q) + 2 * p.tokens - 1) / (2 * p.tokens) - 1 - t.tile;
  }
  if (!t.sound && (threadIdx.x & 31) == 0) report(p.status, LINATTN_DEV_BAD_ID);
  w->q_first = t.first;
  w->lq = min(t.n, p.max_q);
  w->k_first = t.other_first;
  w->lk = t.other_n;
  w->t0 = t.tile * 2 * p.tokens;
  w->shift = w->lk - t.n;  // token t reads keys up to t + shift
  int nt[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = w->t0 + i * p.tokens, end = min(w->lq, first + p.tokens);
    const int keys = first >= end ? 0 : p.causal ? max(0, min(w->lk, end + w->shift)) : w->lk;
    nt[i] = (keys + 127) >> 7;
  }
  int j0 = 0, j1 = max(nt[0], nt[1]);
  if (p.n_splits > 1) {
    const int share = (j1 + p.n_splits - 1) / p.n_splits;
    j0 = min(j1, w->split * share);
    j1 = min(j1, j0 + share);
  }
  w->j0 = j0;
  w->n0 = max(0, min(nt[0], j1) - j0);
  w->n1 = max(0, min(nt[1], j1) - j0);
  w->n = max(w->n0, w->n1);
  w->ragged = (w->lk & 127) && j0 + w->n == (w->lk + 127) >> 7 ? w->n - 1 : -1;
  return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(PA_THREADS, 1)
    packed_attention_kernel(const PackedArgs p, const __grid_constant__ CUtensorMap tmq,
                            const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
  using M = MmaOp<T>;
  using SM = PackedSmem<D>;
  constexpr int KS = SM::KS, VS = SM::VS, HALVES = D / 64, TILE = SM::TILE;
  constexpr int AB = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  constexpr uint32_t IDESC_S = umma_idesc(AB, 128, 128, 0);
  constexpr uint32_t IDESC_O = umma_idesc(AB, 128, D, 1);
  extern __shared__ __align__(128) uint8_t asmem_raw[];
  uint8_t* sq = asmem_raw + ((1024 - (smem_u32(asmem_raw) & 1023)) & 1023);  // two row tiles
  uint8_t* sk = sq + 2 * TILE;
  uint8_t* sv_ring = sk + KS * TILE;
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], v_ragged[VS],
      s_full[2], p_full[2][2], pv_done[2], i_full[PA_ITEMS], i_empty[PA_ITEMS], last;
  __shared__ PackedItem items[PA_ITEMS];
  __shared__ uint32_t tmem_sh;
  __shared__ int dead;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int boxb = p.tokens * p.G * 128;
  PackedItem ahead;
  PackedOrder order;
  if (warp == 3) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the offsets may be the previous kernel's
    if (p.S <= 64) order.load(p);
    ahead.more = packed_item(p, order, 0, &ahead) ? 1 : 0;
  }
  if (tid == 0) {
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
      mbar_init(&v_ragged[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s][0], 128);
      mbar_init(&p_full[s][1], 128);
      mbar_init(&pv_done[s], 1);
    }
    for (int s = 0; s < PA_ITEMS; ++s) {
      mbar_init(&i_full[s], 1);
      mbar_init(&i_empty[s], PA_THREADS / 32 - 1);
    }
    mbar_init(&last, 1);
    dead = 0;
    mbar_fence_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_sh)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  asm volatile("griddepcontrol.wait;" ::: "memory");  // so may q, k and v, and out may be in use
  __syncthreads();
  tc_fence_after();
  // A wait for another warp's end of an item, not of a tile: a part of 2^27 keys takes seconds.
  auto item_wait = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, p.item_ns)) != 0;
  };
  // the item of a turn, and its slot's return
  auto take = [&](int turn, bool* ok) -> const PackedItem* {
    const int slot = turn % PA_ITEMS;
    *ok = *ok && item_wait(&i_full[slot], static_cast<uint32_t>((turn / PA_ITEMS) & 1));
    return *ok && items[slot].more ? &items[slot] : nullptr;
  };
  auto give_back = [&](int turn) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&i_empty[turn % PA_ITEMS]);
  };
  // columns [128 i, 128 i + 128): S / P of row tile i; [256 + 128 i, ...): O of row tile i
  const uint32_t tmem = tmem_sh;

  if (warp < 4) {
    regs_dec<PA_REGS_LOW>();
    if (warp == 0) {
      int kc = 0, vc = 0, qc[2] = {0, 0};  // loads so far: K and V tiles, Q of each row tile
      // a bit for each V stage: whether its last load was a ragged tile, and the parity of its ragged loads
      uint32_t ragged = 0, ragged_par = 0;
      bool ok = true;
      for (int turn = 0;; ++turn) {
        const PackedItem* item = take(turn, &ok);
        if (!item) break;
        const PackedItem& w = *item;
        if (lane == 0) {
          auto load_q = [&](int i) {
            if (qc[i] > 0) ok = ok && mbar_wait_bounded(&q_empty[i], static_cast<uint32_t>((qc[i] - 1) & 1));
            if (!ok || dead) return;
            mbar_arrive_expect_tx(&q_full[i], boxb * HALVES);
            for (int c = 0; c < HALVES; ++c)
              tma_load_3d(sq + i * TILE + c * 16384, &tmq, 64 * c, w.kvh * p.G, w.q_first + w.t0 + i * p.tokens, &q_full[i]);
            ++qc[i];
          };
          auto load_k = [&](int j) {
            const int st = kc % KS;
            if (kc >= KS) ok = ok && mbar_wait_bounded(&k_empty[st], static_cast<uint32_t>((kc / KS - 1) & 1));
            if (!ok || dead) return;
            mbar_arrive_expect_tx(&k_full[st], TILE);
            for (int c = 0; c < HALVES; ++c)
              tma_load_3d(sk + st * TILE + c * 16384, &tmk, 64 * c, w.kvh, w.k_first + (w.j0 + j) * 128, &k_full[st]);
            ++kc;
          };
          auto load_v = [&](int j) {
            const int st = vc % VS;
            if (vc >= VS) ok = ok && mbar_wait_bounded(&v_empty[st], static_cast<uint32_t>((vc / VS - 1) & 1));
            if (!ok || dead) return;
            // A ragged V tile goes to warp 2 first, which passes it on.  Each stage has its barrier for
            // that: v_empty orders a stage's loads, while ragged tiles of short items next to one
            // another are in flight together.
            const bool to_clear = j == w.ragged;
            ragged = (ragged & ~(1u << st)) | (static_cast<uint32_t>(to_clear) << st);
            ragged_par ^= static_cast<uint32_t>(to_clear) << st;
            uint64_t* bar = to_clear ? &v_ragged[st] : &v_full[st];
            mbar_arrive_expect_tx(bar, TILE);
            for (int c = 0; c < HALVES; ++c)
              tma_load_3d(sv_ring + st * TILE + c * 16384, &tmv, 64 * c, w.kvh, w.k_first + (w.j0 + j) * 128, bar);
            ++vc;
          };
          if (w.n > 0) {
            if (w.n0 > 0) load_q(0);
            load_k(0);
            if (w.n1 > 0) load_q(1);
            for (int j = 0; ok && !dead && j < w.n; ++j) {
              load_v(j);
              if (j + 1 < w.n) load_k(j + 1);
            }
          }
          if (!ok) report(p.status, LINATTN_DEV_TIMEOUT);
          if (dead) ok = false;
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        give_back(turn);
      }
      if (!ok && lane == 0) {  // the copies in flight land before the CTA gives up its shared memory
        dead = 1;
        for (int i = 0; i < 2; ++i)
          if (qc[i] > 0) (void)mbar_wait_bounded(&q_full[i], static_cast<uint32_t>((qc[i] - 1) & 1), 200000000ull);
        for (int j = kc > KS ? kc - KS : 0; j < kc; ++j)
          (void)mbar_wait_bounded(&k_full[j % KS], static_cast<uint32_t>((j / KS) & 1), 200000000ull);
        for (int j = vc > VS ? vc - VS : 0; j < vc; ++j) {
          const int st = j % VS;
          if ((ragged >> st) & 1u) (void)mbar_wait_bounded(&v_ragged[st], ((ragged_par >> st) & 1u) ^ 1u, 200000000ull);
          else (void)mbar_wait_bounded(&v_full[st], static_cast<uint32_t>((j / VS) & 1), 200000000ull);
        }
      }
    } else if (warp == 1) {
      int kc = 0, vc = 0, qc0 = 0, qc1 = 0, pc0 = 0, pc1 = 0;  // tiles so far: K, V, Q and P of each row tile
      bool ok = true;
      const uint64_t q_desc = umma_desc(smem_u32(sq), 16, 1024), k_desc = umma_desc(smem_u32(sk), 16, 1024),
                     v_desc = umma_desc(smem_u32(sv_ring), 16384, 1024);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      for (int turn = 0;; ++turn) {
        const PackedItem* item = take(turn, &ok);
        if (!item) break;
        const PackedItem w = *item;
        give_back(turn);
        if (w.n > 0) {
          auto scores = [&](int i, int j) {  // S_i of the item's key tile j
            const uint64_t a0 = q_desc + i * (TILE >> 4), b0 = k_desc + ((kc + j) % KS) * (TILE >> 4);
            if (elect_lane()) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
                umma_f16(tm + i * 128, a0 + off, b0 + off, IDESC_S, kk > 0 ? 1u : 0u);
              }
              umma_commit(&s_full[i]);
              if (j + 1 == (i ? w.n1 : w.n0)) umma_commit(&q_empty[i]);
            }
          };
          auto key_tile = [&](int j) {
            ok = ok && warp_wait(&k_full[(kc + j) % KS], static_cast<uint32_t>(((kc + j) / KS) & 1));
            if (ok) tc_fence_after();
          };
          key_tile(0);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (ok && (i ? w.n1 : w.n0) > 0) {
              ok = warp_wait(&q_full[i], static_cast<uint32_t>((i ? qc1++ : qc0++) & 1));
              if (ok) {
                tc_fence_after();
                scores(i, 0);
              }
            }
          if (ok && elect_lane()) umma_commit(&k_empty[kc % KS]);
          for (int j = 0; ok && j < w.n; ++j) {
            bool v_there = false, k_there = false;
            const uint64_t vd = v_desc + ((vc + j) % VS) * (TILE >> 4);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int ni = i ? w.n1 : w.n0;
              if (!ok || j >= ni) continue;
              if (!v_there) ok = warp_wait(&v_full[(vc + j) % VS], static_cast<uint32_t>(((vc + j) / VS) & 1));
              v_there = true;
#pragma unroll
              for (int h = 0; h < 2; ++h) {  // the first 64 keys while the others' weights are computed
                ok = ok && warp_wait(&p_full[i][h], static_cast<uint32_t>((i ? pc1 : pc0) & 1));
                if (!ok) break;
                tc_fence_after();
                if (elect_lane()) {
#pragma unroll
                  for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                    umma_f16_ts(tm + 256 + i * 128, tm + i * 128 + 8 * kk, vd + kk * (2048 >> 4), IDESC_O,
                                (j > 0 || kk > 0) ? 1u : 0u);
                  if (h == 1) umma_commit(&pv_done[i]);
                }
              }
              if (!ok) break;
              i ? ++pc1 : ++pc0;
              if (j + 1 < ni) {
                if (!k_there) key_tile(j + 1);
                k_there = true;
                if (ok) scores(i, j + 1);
              }
            }
            if (ok && elect_lane()) {
              umma_commit(&v_empty[(vc + j) % VS]);
              if (k_there) umma_commit(&k_empty[(kc + j + 1) % KS]);
            }
          }
          if (!ok && lane == 0) {
            report(p.status, LINATTN_DEV_TIMEOUT);
            dead = 1;
          }
          kc += w.n;
          vc += w.n;
        }
      }
    } else if (warp == 2) {
      int vc = 0;
      uint32_t par = 0;  // a bit for each V stage: of its ragged tiles
      bool ok = true;
      for (int turn = 0;; ++turn) {
        const PackedItem* item = take(turn, &ok);
        if (!item) break;
        const PackedItem& w = *item;
        if (w.ragged >= 0) {
          const int st = (vc + w.ragged) % VS;
          ok = item_wait(&v_ragged[st], (par >> st) & 1u);
          par ^= 1u << st;
          if (ok) {
            const int from = (w.lk & 127) * 8;  // 16-byte pieces of the 128-byte rows of one channel half
            uint8_t* t = sv_ring + st * TILE;
            for (int c = 0; c < HALVES; ++c)
              for (int x = from + lane; x < 1024; x += 32)
                *reinterpret_cast<uint4*>(t + c * 16384 + x * 16) = make_uint4(0u, 0u, 0u, 0u);
            umma_fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[st]);
          }
        }
        vc += w.n;
        give_back(turn);
      }
    } else {
      for (int turn = 0;; ++turn) {
        if (turn > 0) ahead.more = packed_item(p, order, turn, &ahead) ? 1 : 0;
        if (turn >= PA_ITEMS && !item_wait(&i_empty[turn % PA_ITEMS], static_cast<uint32_t>((turn / PA_ITEMS - 1) & 1))) {
          if (lane == 0) {
            report(p.status, LINATTN_DEV_TIMEOUT);
            dead = 1;
          }
          break;
        }
        if (lane == 0) {
          items[turn % PA_ITEMS] = ahead;
          mbar_arrive(&i_full[turn % PA_ITEMS]);
        }
        if (!ahead.more) break;
      }
    }
  } else {
    regs_inc<PA_REGS_HIGH>();
    const int i = (warp >> 2) - 1, r = tid & 127;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
    const uint32_t s_addr = lane_addr + i * 128, o_addr = lane_addr + 256 + i * 128;
    const int rt = (r * p.inv_g) >> 16, rg = r - rt * p.G;
    const float sl = p.scale_log2;
    const uint64_t sl2 = pack_f2(sl, sl);
    int sc = 0;  // score tiles so far
    bool ok = true;
    for (int turn = 0;; ++turn) {
      const PackedItem* item = take(turn, &ok);
      if (!item) break;
      const PackedItem& w = *item;
      const int ni = i ? w.n1 : w.n0, t = w.t0 + i * p.tokens + rt;
      const bool row_ok = rt < p.tokens && t < w.lq;
      const int klim = (!row_ok ? 0 : p.causal ? max(0, min(w.lk, t + w.shift + 1)) : w.lk) - w.j0 * 128;  // keys this row reads
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < ni; ++j, ++sc) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&s_full[i], static_cast<uint32_t>(sc & 1)))) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sv[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(s_addr + q * 32, sv[q]);
        tmem_wait_ld();
        const int lim = klim - j * 128;
        if (!__all_sync(0xffffffffu, lim >= 128)) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= lim) sv[c >> 5][c & 31] = 0xff800000u;  // -inf
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; c += 2)
          mx4[(c >> 1) & 3] = fmaxf(fmaxf(mx4[(c >> 1) & 3], __uint_as_float(sv[c >> 5][c & 31])),
                                    __uint_as_float(sv[c >> 5][(c & 31) + 1]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl;
        const bool grow = mx > m + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? (m == -INFINITY ? 0.f : ex2_approx(m - mx)) : 1.f;
          if (j > 0) {  // O holds the tiles before this one once their P V is done
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&pv_done[i], static_cast<uint32_t>((sc - 1) & 1)))) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t ov[32];
              tmem_ld32(o_addr + c * 32, ov);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
              tmem_st32(o_addr + c * 32, ov);
            }
            tmem_wait_st();
          }
          l *= alpha;
          if (grow) m = mx;
        }
        const float neg = m == -INFINITY ? 0.f : -m;  // nothing read yet: every score is -inf, P = 0
        const uint64_t neg2 = pack_f2(neg, neg);
        uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int h = 0; h < 4; ++h) {  // keys [32 h, 32 h + 32)
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = unpack_f2(
                fma_f2(pack_f2(__uint_as_float(sv[h][2 * e]), __uint_as_float(sv[h][2 * e + 1])), sl2, neg2));
            const float y0 = ex2_approx(x.x), y1 = ex2_approx(x.y);
            pk[e] = M::pack(y0, y1);
            sum[e & 3] = add_f2(sum[e & 3], pack_f2(y0, y1));
          }
          tmem_st16(s_addr + h * 16, pk);
          if (h & 1) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[i][h >> 1]);
          }
        }
        const float2 ts = unpack_f2(add_f2(add_f2(sum[0], sum[1]), add_f2(sum[2], sum[3])));
        l += ts.x + ts.y;
      }
      if (ok && ni > 0)
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pv_done[i], static_cast<uint32_t>((sc - 1) & 1)));
      if (!ok) break;
      tc_fence_after();
      const float inv = l != 0.f ? 1.f / l : 0.f;
      const float lse = l != 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
      const int64_t token = static_cast<int64_t>(w.q_first) + t;
      if (p.n_splits > 1) {
        const int64_t rows = p.Nq * p.G, at = token * p.G + rg;
        const int64_t part = static_cast<int64_t>(w.split) * p.Hkv + w.kvh;
        if (row_ok) p.part_lse[part * rows + at] = lse;
        float4* dst = p.part_o + part * (D / 4) * rows + at;
#pragma unroll 1
        for (int c = 0; c < (ni > 0 ? D / 32 : 0); ++c) {
          uint32_t ov[32];
          tmem_ld32(o_addr + c * 32, ov);
          tmem_wait_ld();
          if (row_ok) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[(c * 8 + e) * rows] =
                  make_float4(__uint_as_float(ov[4 * e]) * inv, __uint_as_float(ov[4 * e + 1]) * inv,
                              __uint_as_float(ov[4 * e + 2]) * inv, __uint_as_float(ov[4 * e + 3]) * inv);
          }
        }
      } else {
        const int head = w.kvh * p.G + rg;
        if (row_ok && p.lse) p.lse[token * p.Hq + head] = lse;
        T* out = static_cast<T*>(p.out);
        if (__all_sync(0xffffffffu, row_ok)) {
          // 64 channels at a time through shared memory (16-byte pieces, swizzled by the row), then
          // four whole rows a store; a row to a thread takes 32 lines a store (a prompt of 4096
          // tokens 123.8 against 126.0 us, a batch of 9 sequences 116.7 against 121.3)
          uint8_t* st = sv_ring + VS * TILE + (i * 4 + (warp & 3)) * 4096;
#pragma unroll 1
          for (int c = 0; c < HALVES; ++c) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t ov[16];
              if (ni > 0) {  // warp-uniform
                tmem_ld16(o_addr + c * 64 + q * 16, ov);
                tmem_wait_ld();
              }
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  y[e] = l != 0.f ? M::pack(__uint_as_float(ov[h * 8 + 2 * e]) * inv, __uint_as_float(ov[h * 8 + 2 * e + 1]) * inv) : 0u;
                *reinterpret_cast<uint4*>(st + lane * 128 + (((2 * q + h) ^ (lane & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
              }
            }
            __syncwarp();
            const int piece = lane & 7;
#pragma unroll 4
            for (int x = 0; x < 32; x += 4) {
              const int rw = x + (lane >> 3), rr = 32 * (warp & 3) + rw, tt = (rr * p.inv_g) >> 16;  // rr / G
              *reinterpret_cast<uint4*>(out + (static_cast<int64_t>(w.q_first) + w.t0 + i * p.tokens + tt) * p.ot +
                                        (static_cast<int64_t>(w.kvh) * p.G + rr - tt * p.G) * p.oh + c * 64 + piece * 8) =
                  *reinterpret_cast<const uint4*>(st + rw * 128 + ((piece ^ (rw & 7)) << 4));
            }
            __syncwarp();
          }
        } else if (__any_sync(0xffffffffu, row_ok)) {
          // few rows: each thread writes its own, without the wait in between (27 rows of three
          // sequences 9.0 us, by way of shared memory 9.5)
          T* dst = out + token * p.ot + head * p.oh;
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t ov[16];
            if (ni > 0) {  // warp-uniform
              tmem_ld16(o_addr + c * 16, ov);
              tmem_wait_ld();
            }
            if (row_ok) {
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  y[e] = l != 0.f ? M::pack(__uint_as_float(ov[q * 8 + 2 * e]) * inv, __uint_as_float(ov[q * 8 + 2 * e + 1]) * inv) : 0u;
                *reinterpret_cast<uint4*>(dst + c * 16 + q * 8) = make_uint4(y[0], y[1], y[2], y[3]);
              }
            }
          }
        }
      }
      tc_fence_before();  // the next item's first P V overwrites O after this warp's next P
      give_back(turn);
    }
    if (!ok) {
      report(p.status, LINATTN_DEV_TIMEOUT);
      dead = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (dead && tid == 32) {  // MMAs may still be in flight: wait for them before TMEM goes
    umma_commit(&last);
    (void)mbar_wait_bounded(&last, 0, 200000000ull);
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Merge of the parts of a key range: 32 rows to a block, a lane to a row, and 8 of their channels to
// a warp.  A row's weights 2^(lse_s - max) are found by its lane in every warp; the parts are added
// in their order.  Rows that the parts do not cover (no sequence's) are left alone.
template <typename T, int D>
__global__ void __launch_bounds__(4 * D) packed_merge_kernel(const PackedArgs p) {
  using M = MmaOp<T>;
  constexpr int QUADS = 2;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = blockIdx.y;
  const int64_t rows = p.Nq * p.G, row0 = static_cast<int64_t>(blockIdx.x) * 32 + lane, row = lmin(row0, rows - 1);
  PackedOwner owner;
  owner.load(p.cu_q, p.S, p.Nq, p.max_q);
  const float* lse = p.part_lse + kvh * rows + row;
  const int64_t next = p.Hkv * rows;  // to the next part
  float mx = -INFINITY, sum = 0.f;
#pragma unroll 8
  for (int s = 0; s < p.n_splits; ++s) mx = fmaxf(mx, lse[s * next]);
  const float4* src = p.part_o + (static_cast<int64_t>(kvh) * (D / 4) + warp * QUADS) * rows + row;
  float4 acc[QUADS];
#pragma unroll
  for (int q = 0; q < QUADS; ++q) acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int STEP = 8;  // parts whose loads go out together
  for (int s0 = 0; s0 < p.n_splits; s0 += STEP) {
    // a part that reads nothing has no weight (its o is not written); one of NaN keeps it
    float f[STEP];
    float4 o[STEP][QUADS];
#pragma unroll
    for (int e = 0; e < STEP; ++e) {
      const float part = s0 + e < p.n_splits ? lse[(s0 + e) * next] : -INFINITY;
      f[e] = part == -INFINITY ? 0.f : ex2_approx((part - mx) * 1.4426950408889634f);
#pragma unroll
      for (int q = 0; q < QUADS; ++q)
        o[e][q] = part == -INFINITY ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldg(src + (s0 + e) * (D / 4) * next + q * rows);
    }
#pragma unroll
    for (int e = 0; e < STEP; ++e) {
      sum += f[e];
#pragma unroll
      for (int q = 0; q < QUADS; ++q) {
        acc[q].x += f[e] * o[e][q].x;
        acc[q].y += f[e] * o[e][q].y;
        acc[q].z += f[e] * o[e][q].z;
        acc[q].w += f[e] * o[e][q].w;
      }
    }
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  const int64_t token = row / p.G;
  if (!owner.has(token) || row0 >= rows) return;
  const int head = kvh * p.G + static_cast<int>(row - token * p.G);
  T* dst = static_cast<T*>(p.out) + token * p.ot + head * p.oh + warp * QUADS * 4;
  *reinterpret_cast<uint4*>(dst) = make_uint4(M::pack(acc[0].x * inv, acc[0].y * inv), M::pack(acc[0].z * inv, acc[0].w * inv),
                                              M::pack(acc[1].x * inv, acc[1].y * inv), M::pack(acc[1].z * inv, acc[1].w * inv));
  if (p.lse && warp == 0) p.lse[token * p.Hq + head] = sum != 0.f ? mx + logf(sum) : -INFINITY;
}

int packed_fail(int code, const char* what) {
  char msg[256];
  snprintf(msg, sizeof(msg), "packed_attention: %s", what);
  return set_error(code, msg);
}

template <typename T, int D>
cudaError_t launch_packed(const PackedArgs& p, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, unsigned grid,
                          cudaStream_t st) {
  auto kern = packed_attention_kernel<T, D>;
  static int allowed[64] = {};
  const cudaError_t e = allow_smem(kern, PackedSmem<D>::BYTES, allowed);
  if (e != cudaSuccess) return e;
  const cudaError_t launched = launch_ahead(kern, dim3(grid), PA_THREADS, PackedSmem<D>::BYTES, st, p, q, k, v);
  if (launched != cudaSuccess || p.n_splits == 1) return launched;
  return launch_ahead(packed_merge_kernel<T, D>, dim3(static_cast<unsigned>((p.Nq * p.G + 31) / 32), static_cast<unsigned>(p.Hkv)),
                      4 * D, 0, st, p);
}

int64_t packed_tiles(int64_t N_q, int64_t G, int64_t S, int64_t max_q) {
  const int64_t rows = 2 * (128 / G);
  return lmin(N_q / rows + S, S * ((max_q + rows - 1) / rows));
}

}  // namespace

}  // namespace linattn

using namespace linattn;

extern "C" int32_t linattn_packed_attention_splits(int64_t N_q, int64_t Hq, int64_t Hkv, int64_t S, int64_t max_q,
                                                   int64_t max_k) {
  if (N_q < 1 || Hkv < 1 || Hq < Hkv || Hq / Hkv > 128 || S < 1 || max_q < 1) return 1;
  // Time of n parts to a key range, in key tiles of a work item (1.7 to 2 us): the longest item's, or
  // what the items of a CTA come to where they are more; 1.5 for each item's start and end, and
  // with parts 2.5 for the merge and their bytes, written and read (a tile's time moves 12
  // MB).  The mean item reads what its sequence has before its queries and half of the rest;
  // sequences are taken to be as unlike in keys as in queries.  Measured in us, by parts:
  //   384 queries on 15737 keys, 2 kv heads, D = 64: 1: 197, 4: 61, 6: 47, 8: 65, 12: 52, 18: 54
  //   1 query on 30000 keys, 8 kv heads, D = 128: 1: 437, 8: 67, 16: 44, 18: 44, 24: 57
  //   700 queries on 3000 keys, 8 kv heads: 1: 64, 2: 72, 3: 63, 5: 71, 8: 83
  //   prompts of 2118, 777, 283 and 315 tokens, 2 kv heads: 1: 43, 2: 35, 3: 30, 4: 30, 8: 36
  //   a prompt of 1500 tokens, 8 kv heads: 1: 32, 2: 60
  const double sms = sm_count(), items = static_cast<double>(packed_tiles(N_q, Hq / Hkv, S, max_q) * Hkv);
  const double longest = (max_k + 127) / 128;
  const double even = lmin(N_q, S * max_q) / static_cast<double>(S * max_q);
  const double mean = even * (max_k - 0.5 * lmin(max_q, max_k)) / 128;
  const double bytes = 1024.0 * N_q * Hq;
  int best = 1;
  double least = 0;
  for (int n = 1; n <= 32 && n <= longest; ++n) {
    const int64_t rounds = static_cast<int64_t>((items * n + sms - 1) / sms);
    const double share = mean / n < 1 ? 1 : mean / n;
    const double most = rounds * share > longest / n ? rounds * share : longest / n;
    const double time = most + 1.5 * rounds + (n > 1 ? 2.5 + n * bytes / 12e6 : 0.0);
    if (n == 1 || time < least) {
      least = time;
      best = n;
    }
  }
  return best;
}

extern "C" int64_t linattn_packed_attention_workspace(int64_t N_q, int64_t Hq, int64_t D, int32_t n_splits) {
  return n_splits > 1 ? static_cast<int64_t>(n_splits) * N_q * Hq * (D + 1) * 4 : 0;
}

extern "C" int linattn_packed_attention(const void* q, const void* k, const void* v, int32_t dtype, int64_t N_q, int64_t N_k,
                                        int64_t Hq, int64_t Hkv, int64_t D, const int64_t* q_strides,
                                        const int64_t* k_strides, const int64_t* v_strides, const int32_t* cu_q,
                                        const int32_t* cu_k, int64_t S, int64_t max_q, int64_t max_k, int32_t causal,
                                        float scale, void* out, const int64_t* out_strides, float* lse, int32_t n_splits,
                                        void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (!q_strides || !k_strides || !v_strides || !out_strides || !cu_q || !cu_k) return packed_fail(LINATTN_EINVAL, "NULL pointer");
  if (dtype != LINATTN_BF16 && dtype != LINATTN_F16) return packed_fail(LINATTN_EUNSUPPORTED, "q, k and v must be bf16 or f16");
  if (D != 64 && D != 128) return packed_fail(LINATTN_EUNSUPPORTED, "head_dim must be 64 or 128");
  if (Hkv < 1 || Hq < 1 || Hq % Hkv) return packed_fail(LINATTN_EINVAL, "H_q must be a multiple of H_kv");
  if (Hq / Hkv > 128) return packed_fail(LINATTN_EUNSUPPORTED, "at most 128 query heads to a kv head");
  if (N_q < 0 || N_k < 0 || S < 0 || max_q < 0 || max_k < 0 || n_splits < 1)
    return packed_fail(LINATTN_EINVAL, "sizes must not be negative");
  if (N_q >= (int64_t(1) << 30) || N_k >= (int64_t(1) << 30)) return packed_fail(LINATTN_EUNSUPPORTED, "at most 2^30 rows");
  if (n_splits > 1 && Hkv > 65535) return packed_fail(LINATTN_EUNSUPPORTED, "at most 65535 kv heads with parts");
  if (!(scale > 0.f) || scale > 1e30f) return packed_fail(LINATTN_EINVAL, "scale must be positive and finite");
  if (N_q == 0 || S == 0) return LINATTN_OK;
  if (!q || !out || (N_k > 0 && (!k || !v))) return packed_fail(LINATTN_EINVAL, "NULL pointer");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) % 16)
    return packed_fail(LINATTN_EINVAL, "q, k, v and out must be 16-byte aligned");
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] % 8 || k_strides[i] % 8 || v_strides[i] % 8 || out_strides[i] % 8)
      return packed_fail(LINATTN_EINVAL, "strides must be multiples of 16 bytes");
  if (n_splits > 1 && (!workspace || workspace_bytes < linattn_packed_attention_workspace(N_q, Hq, D, n_splits) ||
                       reinterpret_cast<uintptr_t>(workspace) % 16))
    return packed_fail(LINATTN_EINVAL, "workspace too small or not 16-byte aligned");
  PackedArgs p;
  p.G = static_cast<int>(Hq / Hkv);
  p.tokens = 128 / p.G;
  p.inv_g = (65536 + p.G - 1) / p.G;
  const CUtensorMapDataType cu = dtype == LINATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tq, tk, tv;
  const int64_t qd[3] = {D, Hq, N_q}, qs[2] = {q_strides[1] * 2, q_strides[0] * 2};
  const int64_t kd[3] = {D, Hkv, lmax(N_k, 1)}, ks[2] = {k_strides[1] * 2, k_strides[0] * 2}, vs[2] = {v_strides[1] * 2, v_strides[0] * 2};
  const int qbox[3] = {64, p.G, p.tokens}, kbox[3] = {64, 1, 128};
  const bool keys = N_k > 0;  // without keys no tile is read
  if (!tensor_map_3d(&tq, q, cu, qd, qs, qbox) || !tensor_map_3d(&tk, keys ? k : q, cu, kd, ks, kbox) ||
      !tensor_map_3d(&tv, keys ? v : q, cu, kd, vs, kbox))
    return packed_fail(LINATTN_ECUDA, "tensor map encoding failed");
  p.cu_q = cu_q; p.cu_k = cu_k; p.Nq = N_q; p.Nk = N_k; p.max_q = static_cast<int>(lmin(max_q, N_q));
  p.S = static_cast<int>(S); p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(Hkv);
  p.causal = causal ? 1 : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = out; p.ot = out_strides[0]; p.oh = out_strides[1];
  p.lse = lse;
  p.n_splits = n_splits;
  p.part_o = static_cast<float4*>(workspace);
  p.part_lse = n_splits > 1 ? static_cast<float*>(workspace) + n_splits * N_q * Hq * D : nullptr;
  p.status = status;
  const int64_t tiles = packed_tiles(N_q, p.G, S, max_q);
  if (Hkv > 65535 || n_splits > 32) return packed_fail(LINATTN_EUNSUPPORTED, "more than 65535 kv heads, or than 32 splits");
  if (tiles == 0) return LINATTN_OK;
  p.items = tiles * Hkv * n_splits;
  // 2 s as every wait; a key tile of an item takes about 2 us, and two items may lie ahead
  p.item_ns = 2000000000ull + static_cast<uint64_t>(N_k / 128 / n_splits) * 8000ull;
  const unsigned grid = static_cast<unsigned>(lmin(sm_count(), p.items));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == LINATTN_BF16) e = D == 128 ? launch_packed<__nv_bfloat16, 128>(p, tq, tk, tv, grid, st) : launch_packed<__nv_bfloat16, 64>(p, tq, tk, tv, grid, st);
  else e = D == 128 ? launch_packed<__half, 128>(p, tq, tk, tv, grid, st) : launch_packed<__half, 64>(p, tq, tk, tv, grid, st);
  return e == cudaSuccess ? LINATTN_OK : packed_fail(LINATTN_ECUDA, cudaGetErrorString(e));
}
