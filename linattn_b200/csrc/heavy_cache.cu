// Heavy-hitter cache: a fixed number M of slots per (sequence, kv head) that keep a
// token's K and V rows, the attention weight it has received (`mass`) and its position.
//
//   load     a prompt of n tokens is cut to M: the first `sinks`, the last `recent` and, of
//            the rest, the ones of most mass (lowest position on ties), in ascending order;
//   append   one new token: the next empty slot, or in a full cache the slot of least mass
//            (lowest slot on ties) among those with sinks <= position <= now - recent.
//
// Attention does not depend on the order of its keys (rotary phases are in K already), so an
// append overwrites one slot in place and nothing else moves.
#include <cooperative_groups.h>

#include <cstdio>

#include "launchers.cuh"
#include "packed_tiles.cuh"

namespace cg = cooperative_groups;

namespace linattn {

namespace {

struct HeavyCacheArgs {
  uint4* k;        // (B, H, M, D) rows of `pieces` 16-byte pieces
  uint4* v;
  float* mass;     // (B, H, M)
  int32_t* pos;    // (B, H, M)
  int32_t* seen;   // (B) tokens taken so far; min(seen, M) slots are in use
  int B, H, M, pieces, sinks, recent;
  int32_t* status;
};

// larger mass -> larger key, every NaN above +inf (a NaN weight is not evidence of being unused)
__device__ __forceinline__ uint32_t mass_key(float f) { return f != f ? 0xffffffffu : float_key(f); }

// ---------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------
// One CTA per (sequence, kv head).  A pass over the head's masses and positions (8 bytes a
// slot) gives the least (key, slot) by one 64-bit minimum; the row is then written by the
// first threads.  Several new tokens are taken one after the other.  The last CTA of a
// sequence (a ticket) moves `seen`, which every CTA of the sequence has read before its
// ticket was drawn.  Bound by a launch's latency for few units (8 heads of 512 slots: 3.2 us)
// and by HBM and L2 for many (64 x 8 x 4096 slots, 17 MB: 5.7 us; both in a graph).
constexpr int APPEND_THREADS = 256;

__global__ void __launch_bounds__(APPEND_THREADS) heavy_append_kernel(const HeavyCacheArgs c,
                                                                      const uint4* __restrict__ k_new,
                                                                      const uint4* __restrict__ v_new, int64_t kb,
                                                                      int64_t kh, int64_t kt, int64_t vb, int64_t vh,
                                                                      int64_t vt, int t_new, int32_t* __restrict__ ticket) {
  __shared__ unsigned long long best[APPEND_THREADS / 32];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int64_t unit = static_cast<int64_t>(b) * c.H + h;
  float* mass = c.mass + unit * c.M;
  int32_t* pos = c.pos + unit * c.M;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = c.seen[b];
  for (int t = 0; t < t_new; ++t) {
    const int now = n + t;
    int slot = now;
    if (now >= c.M) {
      unsigned long long least = ~0ull;
      auto take = [&](float m, int p, int i) {
        if (p >= c.sinks && p <= now - c.recent) {
          const unsigned long long key = (static_cast<unsigned long long>(mass_key(m)) << 32) | static_cast<unsigned>(i);
          least = key < least ? key : least;
        }
      };
      if ((c.M & 3) == 0) {  // the head's masses and positions start on 16 bytes
#pragma unroll 4
        for (int i = tid; i < (c.M >> 2); i += APPEND_THREADS) {
          const float4 m = reinterpret_cast<const float4*>(mass)[i];
          const int4 p = reinterpret_cast<const int4*>(pos)[i];
          take(m.x, p.x, 4 * i);
          take(m.y, p.y, 4 * i + 1);
          take(m.z, p.z, 4 * i + 2);
          take(m.w, p.w, 4 * i + 3);
        }
      } else {
        for (int i = tid; i < c.M; i += APPEND_THREADS) take(mass[i], pos[i], i);
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, least, o);
        least = other < least ? other : least;
      }
      if ((tid & 31) == 0) best[tid >> 5] = least;
      __syncthreads();
      least = best[0];
#pragma unroll
      for (int w = 1; w < APPEND_THREADS / 32; ++w) least = best[w] < least ? best[w] : least;
      slot = least == ~0ull ? -1 : static_cast<int>(least & 0xffffffffu);
    }
    if (slot >= 0) {
      for (int i = tid; i < 2 * c.pieces; i += APPEND_THREADS) {
        const bool is_v = i >= c.pieces;
        const int e = is_v ? i - c.pieces : i;
        const uint4* src = is_v ? v_new + b * vb + h * vh + t * vt : k_new + b * kb + h * kh + t * kt;
        (is_v ? c.v : c.k)[(unit * c.M + slot) * c.pieces + e] = __ldg(src + e);
      }
      if (tid == 0) {
        mass[slot] = 0.f;
        pos[slot] = now;
      }
    } else if (tid == 0) {
      report(c.status, LINATTN_DEV_BAD_ID);  // positions that no append or load has written: nothing may go
    }
    if (t + 1 < t_new) __syncthreads();  // the next token's search sees this one's slot
  }
  __syncthreads();  // every thread has read seen[b]
  if (tid == 0) {
    __threadfence();
    if (atomicAdd(ticket + b, 1) == c.H - 1) {
      ticket[b] = 0;
      c.seen[b] = n + t_new;
    }
  }
}

// ---------------------------------------------------------------------------------
// load
// ---------------------------------------------------------------------------------
// Selection: a cluster per (sequence, kv head), each CTA a contiguous part of the prompt, each
// thread 16 tokens next to one another, whose keys stay in registers (parts of more than
// 8192 tokens are read again for every pass).  The R-th largest mass of the candidates is found
// digit by digit (11 + 11 + 10 bits: the first digit of positive floats is spread over enough
// bins that the shared-memory atomics rarely meet).  The CTAs read one another's histograms
// over distributed shared memory in two steps, the sums of 64 groups of bins and then the 32
// bins of the group that holds the R-th: one remote load a thread and step, where reading
// all 2048 bins of 8 CTAs took most of the time (16 ragged prompts, 8 heads: 247 us).  Once a
// bin holds 1024 candidates or fewer (mostly after the first digit) they are ranked against one
// another instead.  Then every CTA knows how many kept tokens lie before its part and writes
// the positions and masses of its own in order.  The rows are moved by a second kernel, spread
// evenly over the GPU: what is kept is not spread evenly over the prompt (`recent` tokens all
// lie at its end).  Measured, both kernels in a graph: 32768 tokens to 2048 slots, 8 heads,
// D = 128 15.1 us, 16 ragged prompts to 1024 slots, D = 64 21.1 us, most of it barriers and remote
// reads of the selection.
constexpr int SEL_THREADS = 512;
constexpr int SEL_PER = 16;                        // tokens of a thread in one round
constexpr int SEL_ROUND = SEL_THREADS * SEL_PER;   // tokens of a CTA in one round
constexpr int SEL_BINS = 2048;
constexpr int SEL_GROUPS = 64;                     // groups of 32 bins
constexpr int SEL_LIST = 1024;                     // candidates that are ranked against one another at most

struct HeavyLoadArgs {
  const float* mass;   // (H, N)
  int64_t mass_stride;
  const int32_t* cu;   // (S + 1)
  const int32_t* rows; // (S) cache rows, or NULL: sequence s fills row s
  int64_t N;
};

// the tokens [first, first + n) of sequence s, whatever `cu` holds
__device__ __forceinline__ bool sequence_range(const int32_t* cu, int s, int64_t N, int64_t* first, int* n) {
  const int64_t a = cu[s], b = cu[s + 1];
  const int64_t lo = lmin(lmax(a, 0), N), hi = lmin(lmax(b, lo), N);
  *first = lo;
  *n = static_cast<int>(hi - lo);
  return a == lo && b == hi;
}

// Inclusive sums over a warp from the highest lane down.
__device__ __forceinline__ uint32_t sum_from_above(uint32_t x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_down_sync(0xffffffffu, x, o);
    if (lane + o < 32) x += y;
  }
  return x;
}

__global__ void __launch_bounds__(SEL_THREADS, 2) heavy_select_kernel(const HeavyCacheArgs c, const HeavyLoadArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ __align__(16) uint32_t hist[SEL_BINS];
  __shared__ uint32_t groups[SEL_GROUPS];   // sums of this CTA's bins
  __shared__ uint32_t totals[SEL_GROUPS];   // of all CTAs: groups, then the bins of one group
  __shared__ uint32_t scan[SEL_THREADS / 32 + 1];
  __shared__ uint32_t picked[3];            // group or bin that holds the R-th largest, how many lie above it and in it
  // the candidates of that bin, of this CTA and of all (key over complemented position: the
  // larger word comes first), and those that stay
  __shared__ uint64_t own_list[SEL_LIST], all_list[SEL_LIST];
  __shared__ uint32_t counts[8];
  __shared__ uint32_t stays[SEL_ROUND / 32];
  __shared__ uint32_t own_n, kept_n;
  __shared__ uint32_t above[2];             // this CTA's candidates over the threshold / equal to it
  const int tid = threadIdx.x, lane = tid & 31, cl = static_cast<int>(cluster.num_blocks()),
            rank = static_cast<int>(cluster.block_rank());
  asm volatile("griddepcontrol.wait;" ::: "memory");               // started ahead of the previous kernel's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the row copies wait for this kernel's end
  const int unit_in = blockIdx.x / cl;
  const int h = unit_in % c.H, s = unit_in / c.H;
  int64_t first;
  int n;
  const bool sound = sequence_range(a.cu, s, a.N, &first, &n);
  const int b = a.rows ? a.rows[s] : s;
  const bool row_ok = b >= 0 && b < c.B;
  if (tid == 0 && rank == 0 && (!sound || !row_ok)) report(c.status, LINATTN_DEV_BAD_ID);
  if (!row_ok) return;  // the whole cluster
  const float* mass = a.mass + h * a.mass_stride + first;
  const int64_t unit = static_cast<int64_t>(b) * c.H + h;
  float* out_mass = c.mass + unit * c.M;
  int32_t* out_pos = c.pos + unit * c.M;
  // part of this CTA
  const int part = (n + cl - 1) / cl;
  const int lo = min(n, rank * part), hi = min(n, lo + part);
  if (h == 0 && rank == 0 && tid == 0) c.seen[b] = n;
  if (n <= c.M) {  // everything stays
    for (int i = lo + tid; i < hi; i += SEL_THREADS) {
      out_mass[i] = mass[i];
      out_pos[i] = i;
    }
    return;
  }
  const int c_lo = c.sinks, c_hi = n - c.recent;  // candidates [c_lo, c_hi): c_hi - c_lo > M - sinks - recent
  const int want = c.M - c.sinks - c.recent;
  uint32_t prefix = 0, left = static_cast<uint32_t>(want);
  // the masses of this thread's tokens of one round: with a few tokens to a thread they sit
  // close together, so that every thread has some
  const int rounds = (part + SEL_ROUND - 1) / SEL_ROUND;
  const int per = rounds <= 1 ? (part + SEL_THREADS - 1) / SEL_THREADS : SEL_PER;
  float m[SEL_PER];
  int base = 0;
  auto fetch = [&](int r) {
    base = lo + r * SEL_ROUND + tid * per;
#pragma unroll
    for (int e = 0; e < SEL_PER; ++e) m[e] = e < per && base + e < hi ? __ldg(mass + base + e) : 0.f;
  };
  auto candidate = [&](int e) { return e < per && base + e < hi && base + e >= c_lo && base + e < c_hi; };
  if (rounds == 1) fetch(0);
  int listed = -1;  // digits below this bit are left to the list
  if (want > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass == 2 ? 1023u : 2047u;
      for (int i = tid; i < SEL_BINS; i += SEL_THREADS) hist[i] = 0;
      __syncthreads();
      for (int r = 0; r < rounds; ++r) {
        if (rounds > 1) fetch(r);
#pragma unroll
        for (int e = 0; e < SEL_PER; ++e) {
          const uint32_t key = mass_key(m[e]);
          if (candidate(e) && (pass == 0 || (key >> (pass == 1 ? 21 : 10)) == prefix))
            atomicAdd(&hist[(key >> shift) & digits], 1u);
        }
      }
      __syncthreads();
      {  // 8 threads a group, 4 bins a thread
        const uint4 x = reinterpret_cast<const uint4*>(hist)[tid];
        uint32_t t = x.x + x.y + x.z + x.w;
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        if ((tid & 7) == 0) groups[tid >> 3] = t;
      }
      cluster.sync();
      {  // thread (group, CTA)
        uint32_t t = (tid & 7) < cl ? cluster.map_shared_rank(groups, tid & 7)[tid >> 3] : 0u;
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        if ((tid & 7) == 0) totals[tid >> 3] = t;
      }
      __syncthreads();
      if (tid < 32) {  // two groups a lane
        const uint32_t t0 = totals[2 * lane], t1 = totals[2 * lane + 1];
        const uint32_t over = sum_from_above(t0 + t1) - t0 - t1;
        if (over < left && left <= over + t1) {
          picked[0] = 2 * lane + 1;
          picked[1] = over;
        } else if (over + t1 < left && left <= over + t1 + t0) {
          picked[0] = 2 * lane;
          picked[1] = over + t1;
        }
      }
      __syncthreads();
      const uint32_t group = picked[0];
      left -= picked[1];
      if (tid < 256) {  // thread (bin of the group, CTA)
        uint32_t t = (tid & 7) < cl ? cluster.map_shared_rank(hist, tid & 7)[group * 32 + (tid >> 3)] : 0u;
        t += __shfl_xor_sync(0xffffffffu, t, 1);
        t += __shfl_xor_sync(0xffffffffu, t, 2);
        t += __shfl_xor_sync(0xffffffffu, t, 4);
        if ((tid & 7) == 0) totals[tid >> 3] = t;
      }
      __syncthreads();
      if (tid < 32) {
        const uint32_t t = totals[lane], over = sum_from_above(t) - t;
        if (over < left && left <= over + t) {
          picked[0] = group * 32 + lane;
          picked[1] = over;
          picked[2] = t;
        }
      }
      cluster.sync();  // picked[] is there, and every CTA has read the histograms
      prefix = pass == 0 ? picked[0] : (prefix << (pass == 1 ? 11 : 10)) | picked[0];
      left -= picked[1];
      if (rounds == 1 && picked[2] <= SEL_LIST) {
        listed = shift;
        break;
      }
    }
  }
  if (listed >= 0) {
    // Few enough candidates share the threshold's digits: every CTA gets all of them, and each of
    // its own stays if fewer than `left` come before it (larger key, or equal and lower position).
    if (tid == 0) own_n = 0;
    for (int i = tid; i < SEL_ROUND / 32; i += SEL_THREADS) stays[i] = 0;
    __syncthreads();
    uint32_t keep = 0;  // one bit a token
#pragma unroll
    for (int e = 0; e < SEL_PER; ++e) {
      const int i = base + e;
      const uint32_t digits = mass_key(m[e]) >> listed;
      if (candidate(e)) {
        keep |= static_cast<uint32_t>(digits > prefix) << e;
        if (digits == prefix) {
          const uint32_t at = atomicAdd(&own_n, 1u);
          own_list[at] = (static_cast<uint64_t>(mass_key(m[e])) << 32) | ~static_cast<uint32_t>(i);
        }
      } else {
        keep |= static_cast<uint32_t>(e < per && i < hi) << e;
      }
    }
    cluster.sync();
    if (tid < cl) counts[tid] = *cluster.map_shared_rank(&own_n, tid);
    __syncthreads();
    uint32_t all = 0, mine_at = 0;
    const int from = tid / (SEL_THREADS / cl);  // a group of threads copies one CTA's list
    for (int r = 0; r < cl; ++r) {
      if (r == from) mine_at = all;
      all += counts[r];
    }
    for (uint32_t x = tid % (SEL_THREADS / cl); x < counts[from]; x += SEL_THREADS / cl)
      all_list[mine_at + x] = cluster.map_shared_rank(own_list, from)[x];
    __syncthreads();
    for (uint32_t x0 = 0; x0 < own_n; x0 += SEL_THREADS / 8) {  // eight threads a candidate
      const uint32_t x = x0 + tid / 8;
      const uint64_t me = x < own_n ? own_list[x] : ~0ull;
      uint32_t before = 0;
#pragma unroll 4
      for (uint32_t y = tid & 7; y < all; y += 8) before += all_list[y] > me;
      before += __shfl_xor_sync(0xffffffffu, before, 1);
      before += __shfl_xor_sync(0xffffffffu, before, 2);
      before += __shfl_xor_sync(0xffffffffu, before, 4);
      if (x < own_n && (tid & 7) == 0 && before < left) {
        const uint32_t at = ~static_cast<uint32_t>(me) - static_cast<uint32_t>(lo);
        atomicOr(&stays[at >> 5], 1u << (at & 31));
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < SEL_PER; ++e) {
      const int i = tid * per + e;
      if (e < per && base + e < hi) keep |= ((stays[i >> 5] >> (i & 31)) & 1u) << e;
    }
    uint32_t total;
    uint32_t slot = block_exclusive_scan<SEL_THREADS>(__popc(keep), scan, &total);
    if (tid == 0) kept_n = total;
    cluster.sync();
    for (int r = 0; r < rank; ++r) slot += *cluster.map_shared_rank(&kept_n, r);
#pragma unroll
    for (int e = 0; e < SEL_PER; ++e)
      if ((keep >> e) & 1u) {
        if (slot < static_cast<uint32_t>(c.M)) {
          out_mass[slot] = m[e];
          out_pos[slot] = base + e;
        }
        ++slot;
      }
    cluster.sync();  // kept_n is read by the other CTAs
    return;
  }
  // prefix is the threshold key; `left` of its equals stay, the lowest ones
  const uint32_t thr = prefix, ties = left;
  if (tid < 2) above[tid] = 0;
  __syncthreads();
  if (want > 0) {
    uint32_t gt = 0, eq = 0;
    for (int r = 0; r < rounds; ++r) {
      if (rounds > 1) fetch(r);
#pragma unroll
      for (int e = 0; e < SEL_PER; ++e) {
        const uint32_t key = mass_key(m[e]);
        gt += candidate(e) && key > thr;
        eq += candidate(e) && key == thr;
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      gt += __shfl_xor_sync(0xffffffffu, gt, o);
      eq += __shfl_xor_sync(0xffffffffu, eq, o);
    }
    if (lane == 0) {
      atomicAdd(&above[0], gt);
      atomicAdd(&above[1], eq);
    }
  }
  cluster.sync();
  uint32_t gt_before = 0, eq_before = 0;
  for (int r = 0; r < rank; ++r) {
    const uint32_t* o = cluster.map_shared_rank(above, r);
    gt_before += o[0];
    eq_before += o[1];
  }
  // kept tokens before this part: sinks, candidates, and those `recent` ones that lie before it
  uint32_t at = static_cast<uint32_t>(min(lo, c_lo)) + gt_before + min(eq_before, ties) +
                static_cast<uint32_t>(max(0, lo - c_hi));
  uint32_t eq_at = eq_before;
  for (int r = 0; r < rounds; ++r) {
    if (rounds > 1) fetch(r);
    uint32_t keep = 0, eq = 0;  // one bit a token
#pragma unroll
    for (int e = 0; e < SEL_PER; ++e) {
      const int i = base + e;
      const uint32_t key = mass_key(m[e]);
      const bool in = e < per && i < hi, cand = candidate(e) && want > 0;
      keep |= static_cast<uint32_t>(in && (i < c_lo || i >= c_hi || (cand && key > thr))) << e;
      eq |= static_cast<uint32_t>(cand && key == thr) << e;
    }
    // the ties before a token decide whether it stays; one scan carries both counts
    uint32_t total;
    const uint32_t x = block_exclusive_scan<SEL_THREADS>(__popc(keep) | (__popc(eq) << 16), scan, &total);
    uint32_t eq_here = eq_at + (x >> 16);
    uint32_t slot = at + (x & 0xffffu) + (min(eq_here, ties) - min(eq_at, ties));
#pragma unroll
    for (int e = 0; e < SEL_PER; ++e) {
      const bool tie = (eq >> e) & 1u;
      if (((keep >> e) & 1u) || (tie && eq_here < ties)) {
        if (slot < static_cast<uint32_t>(c.M)) {
          out_mass[slot] = m[e];
          out_pos[slot] = base + e;
        }
        ++slot;
      }
      eq_here += tie;
    }
    at += (total & 0xffffu) + (min(eq_at + (total >> 16), ties) - min(eq_at, ties));
    eq_at += total >> 16;
  }
  cluster.sync();  // `above` is read by the other CTAs
}

// Rows of the kept tokens, by the positions that the selection has written.  A group of
// `pieces` threads moves one row of K and of V, 16 bytes a thread, two rows in flight (16 ragged
// prompts to 1024 slots, 8 heads, D = 64: 2 / 4 / 8 rows 26.1 / 28.7 / 34.2 us for the whole load).
constexpr int GATHER_THREADS = 256;
constexpr int GATHER_ROWS = 2;

__global__ void __launch_bounds__(GATHER_THREADS) heavy_gather_kernel(const HeavyCacheArgs c, const HeavyLoadArgs a,
                                                                      const uint4* __restrict__ k, int64_t kn, int64_t kh,
                                                                      const uint4* __restrict__ v, int64_t vn, int64_t vh) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int s = blockIdx.z, h = blockIdx.y;
  const int b = a.rows ? a.rows[s] : s;
  if (b < 0 || b >= c.B) return;
  const int64_t unit = static_cast<int64_t>(b) * c.H + h;
  const int per = GATHER_THREADS / c.pieces;  // rows of one step of the block
  const int e = threadIdx.x % c.pieces, r = threadIdx.x / c.pieces;
  const int base = blockIdx.x * (per * GATHER_ROWS);
  if (r >= per) return;
  int p[GATHER_ROWS];
#pragma unroll
  for (int j = 0; j < GATHER_ROWS; ++j) {  // beside the offsets, before it is known how many slots are used
    const int slot = base + j * per + r;
    p[j] = slot < c.M ? c.pos[unit * c.M + slot] : 0;
  }
  int64_t first;
  int n;
  sequence_range(a.cu, s, a.N, &first, &n);
  const int used = min(n, c.M);
  uint4 kk[GATHER_ROWS], vv[GATHER_ROWS];
#pragma unroll
  for (int j = 0; j < GATHER_ROWS; ++j) {
    const int slot = base + j * per + r;
    if (slot < used) {
      const int64_t at = first + min(max(p[j], 0), n - 1);
      kk[j] = __ldg(k + at * kn + h * kh + e);
      vv[j] = __ldg(v + at * vn + h * vh + e);
    }
  }
#pragma unroll
  for (int j = 0; j < GATHER_ROWS; ++j) {
    const int slot = base + j * per + r;
    if (slot < used) {
      c.k[(unit * c.M + slot) * c.pieces + e] = kk[j];
      c.v[(unit * c.M + slot) * c.pieces + e] = vv[j];
    }
  }
}

int heavy_fail(int code, const char* what) {
  char msg[256];
  snprintf(msg, sizeof(msg), "heavy cache: %s", what);
  return set_error(code, msg);
}

// 16-byte pieces of a stride in 16-bit elements, or -1
int64_t pieces_of(int64_t stride) { return stride % 8 ? -1 : stride / 8; }

int check_heavy(const linattn_heavy_t* c, HeavyCacheArgs* out, int32_t* status) {
  if (!c || !c->k || !c->v || !c->mass || !c->pos || !c->seen) return heavy_fail(LINATTN_EINVAL, "NULL pointer");
  if (c->dtype != LINATTN_F16 && c->dtype != LINATTN_BF16) return heavy_fail(LINATTN_EUNSUPPORTED, "K and V are f16 or bf16");
  if (c->batch < 1 || c->n_kv_heads < 1 || c->budget < 1) return heavy_fail(LINATTN_EINVAL, "batch, n_kv_heads and budget must be > 0");
  if (c->batch > 65535 || c->n_kv_heads > 65535 || c->budget > (1 << 24))
    return heavy_fail(LINATTN_EUNSUPPORTED, "at most 65535 sequences and kv heads, and 2^24 slots");
  if (c->head_dim != 64 && c->head_dim != 128) return heavy_fail(LINATTN_EUNSUPPORTED, "head_dim must be 64 or 128");
  if (c->sinks < 0 || c->recent < 1 || static_cast<int64_t>(c->sinks) + c->recent > c->budget)
    return heavy_fail(LINATTN_EINVAL, "sinks >= 0, recent >= 1 and sinks + recent <= budget");
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | reinterpret_cast<uintptr_t>(c->mass) |
       reinterpret_cast<uintptr_t>(c->pos)) % 16)
    return heavy_fail(LINATTN_EINVAL, "the cache's arrays must be 16-byte aligned");
  out->k = static_cast<uint4*>(c->k);
  out->v = static_cast<uint4*>(c->v);
  out->mass = c->mass;
  out->pos = c->pos;
  out->seen = c->seen;
  out->B = c->batch;
  out->H = c->n_kv_heads;
  out->M = c->budget;
  out->pieces = c->head_dim / 8;
  out->sinks = c->sinks;
  out->recent = c->recent;
  out->status = status;
  return LINATTN_OK;
}

int cuda_result(cudaError_t e) { return e == cudaSuccess ? LINATTN_OK : heavy_fail(LINATTN_ECUDA, cudaGetErrorString(e)); }

}  // namespace

}  // namespace linattn

using namespace linattn;

extern "C" int linattn_heavy_append(const linattn_heavy_t* cache, const void* k_new, const void* v_new,
                                    const int64_t* k_strides, const int64_t* v_strides, int64_t T_new, int32_t* ticket,
                                    int32_t* status, void* stream) {
  HeavyCacheArgs c;
  if (const int rc = check_heavy(cache, &c, status)) return rc;
  if (T_new < 0 || T_new > (1 << 20)) return heavy_fail(LINATTN_EINVAL, "append: 0 .. 2^20 new tokens");
  if (T_new == 0) return LINATTN_OK;  // a tensor of no elements has no address
  if (!k_new || !v_new || !k_strides || !v_strides || !ticket) return heavy_fail(LINATTN_EINVAL, "append: NULL pointer");
  int64_t ks[3], vs[3];
  for (int i = 0; i < 3; ++i) {
    ks[i] = pieces_of(k_strides[i]);
    vs[i] = pieces_of(v_strides[i]);
    if (ks[i] < 0 || vs[i] < 0) return heavy_fail(LINATTN_EINVAL, "append: strides must be multiples of 16 bytes");
  }
  if ((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) % 16)
    return heavy_fail(LINATTN_EINVAL, "append: rows must be 16-byte aligned");
  return cuda_result(launch_ahead(heavy_append_kernel, dim3(c.H, c.B), APPEND_THREADS, 0, static_cast<cudaStream_t>(stream), c,
                                  static_cast<const uint4*>(k_new), static_cast<const uint4*>(v_new), ks[0], ks[1], ks[2], vs[0],
                                  vs[1], vs[2], static_cast<int>(T_new), ticket));
}

extern "C" int linattn_heavy_load(const linattn_heavy_t* cache, const void* k, const void* v, const int64_t* k_strides,
                                  const int64_t* v_strides, int64_t N, const float* mass, int64_t mass_stride,
                                  const int32_t* cu, const int32_t* rows, int64_t S, int32_t* status, void* stream) {
  HeavyCacheArgs c;
  if (const int rc = check_heavy(cache, &c, status)) return rc;
  if (S < 0 || N < 0 || N >= (int64_t(1) << 31)) return heavy_fail(LINATTN_EINVAL, "load: bad number of tokens or sequences");
  if (S == 0) return LINATTN_OK;
  if (!cu || (N > 0 && (!k || !v || !mass)) || !k_strides || !v_strides) return heavy_fail(LINATTN_EINVAL, "load: NULL pointer");
  if (!rows && S > c.B) return heavy_fail(LINATTN_EINVAL, "load: more sequences than cache rows");
  if (S > 65535) return heavy_fail(LINATTN_EUNSUPPORTED, "load: at most 65535 sequences");
  int64_t ks[2], vs[2];
  for (int i = 0; i < 2; ++i) {
    ks[i] = pieces_of(k_strides[i]);
    vs[i] = pieces_of(v_strides[i]);
    if (ks[i] < 0 || vs[i] < 0) return heavy_fail(LINATTN_EINVAL, "load: strides must be multiples of 16 bytes");
  }
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16)
    return heavy_fail(LINATTN_EINVAL, "load: rows must be 16-byte aligned");
  HeavyLoadArgs a;
  a.mass = mass;
  a.mass_stride = mass_stride;
  a.cu = cu;
  a.rows = rows;
  a.N = N;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  // CTAs for the whole GPU where the units alone are too few, each with 1024 tokens or more.
  // (The cluster that selects moving the rows too: 19.9 against 17.5 us for 32768 tokens and 8
  // heads, whose 64 CTAs are too few for the copies.)
  const int64_t units = S * c.H;
  unsigned cl = 1;
  while (cl < 8 && units * cl < sm_count() && N / S > 1024 * static_cast<int64_t>(cl)) cl *= 2;
  cfg.gridDim = dim3(static_cast<unsigned>(S) * c.H * cl);
  cfg.blockDim = dim3(SEL_THREADS);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, heavy_select_kernel, c, a);
  if (e != cudaSuccess) return cuda_result(e);
  const int per = GATHER_THREADS / c.pieces * GATHER_ROWS;
  const unsigned gx = static_cast<unsigned>((lmin(c.M, N) + per - 1) / per);
  if (gx == 0) return LINATTN_OK;
  // set up while the selection runs; the positions are read after its end
  return cuda_result(launch_ahead(heavy_gather_kernel, dim3(gx, c.H, static_cast<unsigned>(S)), GATHER_THREADS, 0, st, c, a,
                                  static_cast<const uint4*>(k), ks[0], ks[1], static_cast<const uint4*>(v), vs[0], vs[1]));
}
