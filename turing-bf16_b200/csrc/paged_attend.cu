// Attention of the newest tokens over a paged key/value cache (decoding): tbf16_paged_attend.
#include <cuda_fp8.h>

#include <algorithm>

#include "paged.cuh"

namespace {
using namespace tbf16;

// For a query row r of a key/value head (T new tokens x the head's group of query heads)
//   s_j = (q_r . k_j) scale,  out_r = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j
// over the visible positions j. Every cached element is used by 2 T group flops, 2..64 in practice, where the
// tensor cores could do hundreds: the time is the cache's bytes over the HBM rate, as long as enough bytes are in
// flight on every SM, however few or uneven the sequences, and no warp computes longer than its bytes take.
//
// Work split. The keys of a (sequence, head, query rows) item are cut into blocks of BK keys; the blocks of all
// items, laid end to end, are shared out evenly over the CTAs (one per SM), from the lengths on the device:
// ragged batches and one long sequence keep all SMs equally busy, and a captured graph follows the lengths. A
// CTA's blocks go round-robin to its teams, of one warp each unless an item has more query rows than a warp's
// registers hold outputs for: then the warps of a team read the same blocks, each for its own rows. A team is a
// pipeline of its own: it issues the TMA loads of its blocks into its own ring of stages, waits for them, and its
// warps keep their running maximum, sum and output in registers, so teams never wait for one another inside an
// item. At its end they are added up through shared memory. An item that spans CTAs leaves one partial (output,
// maximum, sum) per CTA in the workspace; the CTA that arrives last adds them in a fixed order, so results do not
// depend on which one that is.
//
// Tiles. mma.sync m16n8k16 with the cache as the 16-row operand and eight query rows as columns: S^T = K Q^T,
// O^T = V^T P^T. With the usual group of up to eight query rows no product is wasted on empty rows (a 16-row
// query tile would waste half of them, tcgen05's 128 rows fifteen sixteenths), a lane holds four weights per 16
// keys, and P^T gets from accumulator to operand layout by one 8x8 transpose per 8 keys.
// Bytes of all stages of an SM. More in flight makes the queues in front of the memory longer, not the rate higher, and
// the SMs' rates more uneven, so the last one ends later (131071 tokens, all SMs with equal shares: they end after 72
// to 82 us with 128 KB and after 65 to 92 with 192; in all 97 us and 101, 104 with 64).
constexpr int kStageBytes = 128 * 1024;
// Partials that a thread has in flight when it adds them up (24 partials of 16 rows: 21.5 us with four, 19.5 with eight).
constexpr int kPartLoads = 8;

template <int D_, bool E4M3_, int NQ_, int S_>
struct Tile {
  static constexpr int D = D_;
  static constexpr bool E4M3 = E4M3_;
  static constexpr int W = 8;                                // warps
  static constexpr int NQ = NQ_;                             // column tiles of eight query rows of a warp
  static constexpr int S = S_;                               // warps of a team: they share its blocks, each with its own rows
  static constexpr int TEAMS = W / S;
  static constexpr int R = 8 * NQ * S;                       // query rows of an item
  static constexpr int RB = D * (E4M3 ? 1 : 2);              // bytes of a cached row
  static constexpr int AW = RB < 128 ? RB : 128;             // swizzle span: 64 or 128 bytes
  static constexpr int BK = RB <= 64 ? 64 : RB <= 128 ? 32 : 16;  // keys of a block
  static constexpr int NG = BK / 16;                         // groups of 16 keys, worked on one after another
  static constexpr int GB = 16 * RB;                         // bytes of a group: [RB / AW][16 keys][AW]
  static constexpr int KB = NG * GB;                         // bytes of a block's keys (or values): 4 KB, 8 for 512-byte rows
  static constexpr int SC = E4M3 ? 2 * BK * 4 : 0;           // bytes of a block's scales
  static constexpr int MAX_STAGES = kStageBytes / (TEAMS * 2 * KB);
  static constexpr int MP = D + 4;                           // floats between rows of the merge area (no bank twice)
  static constexpr int MERGE = W * 8 * NQ * MP;              // floats of it; a join's thread groups take W * 32 * 4
};

struct AttendParams {
  PagedView c;
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh, q_st;
  __nv_bfloat16* out;
  int64_t o_sb, o_sh, o_st;
  const int* counts;
  int T, group, rows, chunks, window;  // rows = T * group query rows of a head, in chunks of R
  unsigned group_inv;                  // ceil(2^32 / group): row / group = umulhi(row, group_inv) below 2^16
  float scale_log2;
  int stages;
  int box_shift;    // log2 of the keys that one TMA load brings: min(BK, page size); rows of one span when over 16
  int nr;           // rows of an item that can be real: min(rows, R)
  unsigned* sync;   // arrivals of each item, zero between calls
  float* part;      // [2 * CTAs][partial_floats(nr, D)]: partial outputs, (maximum, sum) pairs
  float* logits;    // weights wanted: [batch * heads][rows][cap], base-2 logits
  float* lse;       // and [batch * heads][rows]: log2 of each row's sum
};

// Floats of a partial: nr rows of outputs, then of (maximum, sum) pairs, to a multiple of 16 bytes.
__host__ __device__ constexpr int partial_floats(int nr, int D) { return (nr * (D + 2) + 3) / 4 * 4; }

// In the order of all blocks each item is followed by kPad places that hold none: what an item costs a CTA beyond its
// blocks (loading its queries, waiting for its last warp, adding the warps up), so that CTAs with many short items get
// fewer keys. One number for all tiles: 64 ragged sequences up to 3000 tokens, 16 query heads on 4, with 8 / 24 / 48 take
// bf16 35 / 30 / 31 us (D 64), 48 / 43 / 43 (128), 77 / 73 / 75 (256), e4m3 33 / 31 / 34, 46 / 40 / 40, 64 / 59 / 55.
constexpr int kPad = 24;

// What a CTA knows of a sequence: the first of its blocks, and of its rounds, among all; cached and new tokens.
struct SeqInfo {
  int cum, rounds, len, count;
};

// First block that a sequence's window reaches, and the blocks of one of its items (none without new tokens).
template <class C>
__device__ __forceinline__ int first_block(const AttendParams& p, int len, int count) {
  return p.window ? max(0, len - count + 1 - p.window) / C::BK : 0;
}
template <class C>
__device__ __forceinline__ int item_blocks(const AttendParams& p, int len, int count) {
  return count ? (len + C::BK - 1) / C::BK - first_block<C>(p, len, count) : 0;
}
__device__ __forceinline__ int token_of(const AttendParams& p, int row) {
  return p.group == 1 ? row : (int)__umulhi((unsigned)row, p.group_inv);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same from a zero accumulator.
template <bool F16>
__device__ __forceinline__ void mma16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Four e4m3 values as two packed fp16 pairs, exactly.
__device__ __forceinline__ void e4m3_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}
// Packed e4m3 or bf16 values with infinities and NaNs replaced by zeros.
template <bool E4M3>
__device__ __forceinline__ void finite_only(uint32_t (&r)[4]) {
#pragma unroll
  for (uint32_t& w : r) {
    if (E4M3) w &= ~__vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
    else w &= ~__vcmpeq2(w & 0x7f807f80u, 0x7f807f80u);
  }
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2, int c3,
                                            int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
__device__ __forceinline__ unsigned count_up(unsigned* word) {
  unsigned n;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(word) : "memory");
  return n;
}
// Over the eight lanes that hold one column of an accumulator.
__device__ __forceinline__ float column_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float column_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The transpose of an 8x8 matrix of 16-bit values held two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Byte offset of 16-byte chunk `chunk` of key `row` inside a group, as TMA's swizzle places it.
template <class C>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
  if (C::AW == 128) return (chunk >> 3) * 2048 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
  return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}
// The address of chunk `even + odd` from that of chunk `odd` (odd = 0 or 1, even a constant): the swizzle is an
// exclusive or, and a group starts on a multiple of its span.
template <class C>
__device__ __forceinline__ uint32_t chunk_from(uint32_t at_odd, int even) {
  return C::AW == 128 ? (at_odd ^ ((even & 7) << 4)) + (even >> 3) * 2048 : at_odd ^ (even << 4);
}

// Where a team's next block lies: t in the order of all blocks, the item it belongs to, block of that item.
struct Cursor {
  int t, b, h, blk, blocks, j0, len;  // j0: its first key; len: cached tokens, 0 past the end of the team's blocks
  int page;                           // this lane's page of the block, loaded ahead
};

template <class C>
struct Loader {
  static constexpr bool E4M3 = C::E4M3;

  // Starts loading the page numbers that the cursor's block needs, lane i that of its i-th box.
  static __device__ __forceinline__ void fetch_pages(Cursor& u, const AttendParams& p, int lane) {
    const int j = u.j0 + (lane << p.box_shift);
    u.page = j < min(u.len, u.j0 + C::BK) ? p.c.table[u.b * p.c.table_ld + (j >> p.c.page_shift)] : 0;
  }

  // Moves the cursor to the team's first block at or after position t with anything to load.
  static __device__ __forceinline__ void seek(Cursor& u, int t, int end, const SeqInfo* info, const AttendParams& p, int lane) {
    for (;; t += C::TEAMS) {
      u.t = t;
      u.len = 0;
      if (t >= end) return;
      while (t >= info[u.b + 1].cum) ++u.b;
      const SeqInfo s = info[u.b];
      u.blocks = item_blocks<C>(p, s.len, s.count);
      const unsigned rem = t - s.cum, item = rem / (unsigned)(u.blocks + kPad);
      u.h = p.chunks == 1 ? (int)item : (int)(item / (unsigned)p.chunks);
      u.blk = (int)(rem - item * (u.blocks + kPad));
      if (u.blk >= u.blocks) continue;
      u.j0 = (first_block<C>(p, s.len, s.count) + u.blk) * C::BK;
      u.len = s.len;
      break;
    }
    fetch_pages(u, p, lane);
  }
  static __device__ __forceinline__ void next(Cursor& u, int end, const SeqInfo* info, const AttendParams& p, int lane) {
    if (u.blk + C::TEAMS < u.blocks && u.t + C::TEAMS < end) {
      u.t += C::TEAMS;
      u.blk += C::TEAMS;
      u.j0 += C::TEAMS * C::BK;
      fetch_pages(u, p, lane);
    } else {
      seek(u, u.t + C::TEAMS, end, info, p, lane);
    }
  }

  // Loads the cursor's block into a stage: up to NG boxes of keys and of values, and their scales.
  static __device__ __forceinline__ void load(const Cursor& u, uint8_t* stage, float* scales, uint64_t* bar,
                                              const CUtensorMap* km, const CUtensorMap* vm, const AttendParams& p) {
    const int box = 1 << p.box_shift, boxes = (min(C::BK, u.len - u.j0) + box - 1) >> p.box_shift;
    if (u.page < 0 || u.page >= p.c.pages) atomicOr(p.c.err, kErrPage);
    const int mine = u.page < 0 || u.page >= p.c.pages ? 0 : u.page;  // a bad number is read as page 0
    const bool one = elect_one();
    if (one) mbar_arrive_expect_tx(bar, boxes * box * (2 * C::RB + (E4M3 ? 8 : 0)));
#pragma unroll 1
    for (int i = 0; i < boxes; ++i) {
      const int page = __shfl_sync(0xffffffffu, mine, i), slot = paged_slot(p.c, u.j0 + i * box);
      if (one) {
        tma_load_5d(stage + i * box * C::RB, km, bar, 0, slot, 0, u.h, page);
        tma_load_5d(stage + C::KB + i * box * C::RB, vm, bar, 0, slot, 0, u.h, page);
        if (E4M3) {
          bulk_load(scales + i * box, p.c.k_scale + page * p.c.ks_sp + u.h * p.c.ks_sh + slot, box * 4, bar);
          bulk_load(scales + C::BK + i * box, p.c.v_scale + page * p.c.vs_sp + u.h * p.c.vs_sh + slot, box * 4, bar);
        }
      }
    }
  }
};

// A weight grows to at most 2^kSlack before a new maximum is taken: the running maximum then changes, and the
// output is rescaled, a few times per item and not with every block, and no lane has to ask the others for it.
constexpr float kSlack = 8.f;
constexpr float kNoMax = -3.4028234e38f;  // of a row that has seen nothing: every logit is far above it
// e4m3: the weights that multiply the values carry the value row's scale over the query row's `vtop`, times 2^7: at most
// 2^15 in fp16 (2^kSlack 2^7) while scales stay within vtop, and rounded to 11 bits down to 2^-14. vtop follows the
// scales, four times the largest so far, but not further than 2^kRange times the largest weighted scale that the row
// has met at a change of its maximum: else one key with a large value row, of no weight, would push the weights that
// count into fp16's subnormals. So the largest weighted scale stays at 2^(7 - kRange) or more, and what fp16's smallest
// step loses below 2^-20 of it. Groups with scales beyond vtop are looked at key by key.
constexpr int kWeightShift = 7;
constexpr float kRange = 2048.f;

// Shared memory: [rings][scales][merge][info].
template <class C>
__global__ void __launch_bounds__(C::W * 32, 1)
    attend_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm, const AttendParams p) {
  constexpr int D = C::D, W = C::W, NQ = C::NQ, S = C::S, TEAMS = C::TEAMS, R = C::R, NG = C::NG, KS = D / 16;
  constexpr int NTHREADS = W * 32, MP = C::MP, V = kPartLoads;
  constexpr bool E4M3 = C::E4M3;
  using L = Loader<C>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  float* scale_ring = reinterpret_cast<float*>(ring + (size_t)TEAMS * p.stages * 2 * C::KB);
  float* merge = scale_ring + (size_t)TEAMS * p.stages * (C::SC / 4);
  SeqInfo* info = reinterpret_cast<SeqInfo*>(merge + C::MERGE);
  __shared__ uint64_t full[TEAMS * C::MAX_STAGES], empty[TEAMS * C::MAX_STAGES];
  __shared__ float2 s_ms[TEAMS * R];   // each warp's (maximum, sum) of a row
  __shared__ float2 s_group[NTHREADS]; // that of a row in each thread group of a join
  __shared__ int s_scan[W], s_work[W], s_long[W], s_abort, s_todo;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, team = warp / S, tile = warp % S;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (tid == 0) atomicOr(p.c.err, kErrSmemAlign);
    return;
  }
  if (tid == 0) {
    tma_prefetch_desc(&km);
    tma_prefetch_desc(&vm);
    s_abort = 0;
  }
  if (tid < TEAMS * p.stages) {
    mbar_init(&full[tid], 1);
    mbar_init(&empty[tid], S > 1 ? S - 1 : 1);
  }
  fence_barrier_init();
  pdl_launch_dependents();
  pdl_wait();

  // Every sequence's places and rounds (a round: a block for each team) and their running totals.
  int total = 0, work = 0, longest = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += NTHREADS) {
    const int b = b0 + tid;
    SeqInfo s{0, 0, 0, 0};
    int x = 0, y = 0, blocks = 0;
    if (b < p.c.batch) {
      s.len = paged_len(p.c, b);
      s.count = paged_count(p.c, p.counts, b, p.T, s.len);
      blocks = item_blocks<C>(p, s.len, s.count);
      x = blocks ? (blocks + kPad) * p.c.heads * p.chunks : 0;
      y = (blocks + TEAMS - 1) / TEAMS * p.c.heads * p.chunks;
    }
    const int my_x = x, my_y = y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int dx = __shfl_up_sync(0xffffffffu, x, o), dy = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) x += dx, y += dy;
    }
    blocks = __reduce_max_sync(0xffffffffu, blocks);
    if (lane == 31) {
      s_scan[warp] = x;
      s_work[warp] = y;
      s_long[warp] = blocks;
    }
    __syncthreads();
    x += total - my_x;
    y += work - my_y;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i < warp) x += s_scan[i], y += s_work[i];
      total += s_scan[i];
      work += s_work[i];
      longest = max(longest, s_long[i]);
    }
    s.cum = x;
    s.rounds = y;
    if (b < p.c.batch) info[b] = s;
    if (b == p.c.batch - 1) info[b + 1] = SeqInfo{x + my_x, y + my_y, 0, 0};
    __syncthreads();
  }
  // Few rounds: a CTA takes one, so no item waits for another. Else CTA i takes places [share(i), share(i + 1)): `each`
  // of them, the first `more` CTAs one more.
  // Sequences of one length with fewer items than SMs: as many CTAs for each item, so that none has the end of one and
  // the start of the next to add up and join (128 items of 8000 tokens: 92 us with all SMs, 84 with 128). Leaving SMs
  // out pays while the others' loads fill the memory's queues: down to four fifths of them, or three where a CTA's bf16
  // part is up to 2 MB, start and end a large part of its time. bf16 items of 0.5 / 1 / 2 / 8 MB, all SMs: 80 of them
  // 18.1 / 25.3 / 37.1 / 108 us, 96 21.9 / 29.3 / 43.1 / 128, 112 24.4 / 32.2 / 47.9 / 146, 128 25.8 / 35.0 / 52.8 / 165;
  // whole CTAs: 80 17.5 / 25.5 / 41.1 / 133, 96 18.4 / 26.7 / 42.3 / 134, 112 19.5 / 28.4 / 45.0 / 144, 128 20.4 / 30.4 /
  // 48.8 / 159. e4m3 items, bound by instructions, of 4 MB: 96 of them 77 and 98, 128 97 and 99 (below 1 MB whole CTAs
  // would win there too, down to 80 items: 0.25 MB 18.7 and 15.9).
  const bool by_round = work <= (int)gridDim.x;
  const int items = p.c.batch * p.c.heads * p.chunks, per_item = items <= (int)gridDim.x ? gridDim.x / items : 0;
  const bool small = !E4M3 && longest <= per_item * ((2 << 20) / (2 * C::KB));
  const bool even = !by_round && per_item * items * 5 >= (int)gridDim.x * (small ? 3 : 4) && (longest + kPad) * items == total;
  const int ctas = by_round ? work : even ? per_item * items : (int)gridDim.x;
  // sequences without new tokens: zeros
  for (int b = blockIdx.x; b < p.c.batch; b += gridDim.x) {
    if (info[b].count) continue;
    const int heads = p.c.heads * p.group;
    for (int64_t i = tid; i < (int64_t)heads * p.T * (D / 8); i += NTHREADS) {
      const int row = (int)(i / (D / 8)), t = row / heads;
      *reinterpret_cast<uint4*>(p.out + b * p.o_sb + (int64_t)(row - t * heads) * p.o_sh + t * p.o_st + i % (D / 8) * 8) =
          make_uint4(0, 0, 0, 0);
    }
  }
  if ((int)blockIdx.x >= ctas) return;
  const int each = (even ? longest : total) / (even ? per_item : ctas), more = (even ? longest : total) - each * (even ? per_item : ctas);
  auto share = [&](int i) { return each * i + min(i, more); };
  int c0, c1, first_b = 0;
  if (even) {
    const int item = blockIdx.x / per_item, r = blockIdx.x - item * per_item;
    c0 = item * (longest + kPad) + share(r);
    c1 = item * (longest + kPad) + share(r + 1);
  } else {
    c0 = share(blockIdx.x);
    c1 = share(blockIdx.x + 1);
  }
  for (int hi = p.c.batch; hi - first_b > 1;) {
    const int mid = (first_b + hi) >> 1;
    if (by_round ? info[mid].rounds <= (int)blockIdx.x : info[mid].cum <= c0) first_b = mid;
    else hi = mid;
  }
  if (by_round) {
    const SeqInfo s = info[first_b];
    const int blocks = item_blocks<C>(p, s.len, s.count), rounds = (blocks + TEAMS - 1) / TEAMS, x = blockIdx.x - s.rounds;
    const int item = x / rounds, r = x - item * rounds;
    c0 = s.cum + item * (blocks + kPad) + r * TEAMS;
    c1 = s.cum + item * (blocks + kPad) + min(blocks, (r + 1) * TEAMS);
  }

  // The team's ring. Its first warp loads; every warp of it waits for a block and reads it.
  uint8_t* my_ring = ring + (size_t)team * p.stages * 2 * C::KB;
  float* my_scales = scale_ring + (size_t)team * p.stages * (C::SC / 4);
  uint64_t* my_full = full + team * p.stages;
  uint64_t* my_empty = empty + team * p.stages;
  Cursor u;
  u.b = first_b;
  u.len = 0;
  int issued = 0, waiting = 0;  // stage of the next load; blocks loaded and not used yet
  auto issue = [&]() {
    L::load(u, my_ring + (size_t)issued * 2 * C::KB, my_scales + issued * (C::SC / 4), &my_full[issued], &km, &vm, p);
    issued = issued + 1 == p.stages ? 0 : issued + 1;
    ++waiting;
    L::next(u, c1, info, p, lane);
  };
  if (tile == 0) {
    L::seek(u, c0 + team, c1, info, p, lane);
#pragma unroll 1
    while (waiting < p.stages && u.len) issue();
  }
  int stage = 0, phase = 0;
  bool dead = false;  // a wait gave up: nothing more is loaded or computed, every barrier is still reached

  const int g4 = lane >> 2, c4 = lane & 3;
  // this lane's addresses in the ldmatrix of keys and of values, for the first chunks of a group
  const uint32_t k_lane = chunk_at<C>(lane & 15, lane >> 4);
  const uint32_t v_lane = E4M3 ? k_lane : chunk_at<C>(((lane >> 4) & 1) * 8 + (lane & 7), (lane >> 3) & 1);

  // The item that holds place t.
  struct Item {
    SeqInfo s;
    int start, blocks, b, h, row0, nrow;
  };
  auto item_at = [&](int t, int from) {
    Item it;
    it.b = from;
    while (t >= info[it.b + 1].cum) ++it.b;
    it.s = info[it.b];
    it.blocks = item_blocks<C>(p, it.s.len, it.s.count);
    const int i = (int)((unsigned)(t - it.s.cum) / (unsigned)(it.blocks + kPad));
    it.start = it.s.cum + i * (it.blocks + kPad);
    it.h = p.chunks == 1 ? i : i / p.chunks;
    it.row0 = (i - it.h * p.chunks) * R;
    it.nrow = min(R, p.rows - it.row0);
    return it;
  };
  const size_t part_ld = partial_floats(p.nr, D);
  auto owner = [&](int x) {  // the CTA that has place x
    const int big = more * (each + 1);
    return x < big ? x / (each + 1) : more + (x - big) / each;
  };
  // The partials the CTA leaves, of its first item (slot 0) and its last (1): a block of the item, the first of
  // the CTAs that hold a partial of it and their number, and the word where they are counted.
  int open0 = -1, open1 = -1, at0 = 0, at1 = 0, parts0 = 0, parts1 = 0, word0 = 0, word1 = 0;
  int todo = -1;  // joins that are this CTA's (bit 0, 1), once its own items are done

  // One pass for each item of the CTA, then one for each join. Both share the code that adds up partials: the
  // instructions of a short call run once, and fetching them is a good part of its time.
#pragma unroll 1
  for (int t = c0;;) {
    const bool join = t >= c1;
    if (join) {
      if (todo < 0) {
        if (open0 < 0 && open1 < 0) break;
        // Only now the CTA says that its partials are out, so that no item of its own waited for a join. The last
        // of an item's CTAs to say so joins the item.
        if (tid == 0) {
          // acquire and release; with the barrier before, every thread's partials come before the counts
          const unsigned n0 = open0 >= 0 ? count_up(p.sync + word0) : 0, n1 = open1 >= 0 ? count_up(p.sync + word1) : 0;
          int mine = 0;
          if (open0 >= 0 && n0 == (unsigned)parts0 - 1) mine = 1, p.sync[word0] = 0;
          if (open1 >= 0 && n1 == (unsigned)parts1 - 1) mine |= 2, p.sync[word1] = 0;
          s_todo = mine;
        }
        __syncthreads();
        todo = s_todo;
      }
      if (todo == 0) break;
    }
    const Item it = item_at(!join ? t : todo & 1 ? open0 : open1, first_b);
    const SeqInfo s = it.s;
    const int start = it.start, h = it.h, row0 = it.row0, nrow = it.nrow, b = it.b;
    const int end = min(c1, start + it.blocks), n4 = nrow * (D / 4);
    if (!join && t >= end) {  // places without blocks
      t = min(c1, start + it.blocks + kPad);
      continue;
    }
    // the partials to add up: part k's outputs from src + k src_ld, its (maximum, sum) pairs from ms + k ms_ld
    const float* src = merge;
    const float2* ms = s_ms;
    size_t src_ld = R * MP, ms_ld = R, skip0 = 0;  // skip0: part 0 lies that much further on
    int pitch = MP;                                // floats between a part's rows
    int parts = TEAMS, groups = 1;
    bool split = false;
    if (join) {
      const bool first = todo & 1;
      const int i0 = first ? at0 : at1;
      todo &= first ? 2 : 0;
      parts = first ? parts0 : parts1;
      src = p.part + 2 * (size_t)i0 * part_ld;
      src_ld = 2 * part_ld;
      ms = reinterpret_cast<const float2*>(src + p.nr * D);
      ms_ld = part_ld;
      pitch = D;
      if (!by_round && !even && share(i0) < start) skip0 = part_ld;  // that CTA had another item before this one
      // groups of threads share the parts out
      groups = max(1, min((parts + V - 1) / V, NTHREADS / n4));
    } else {
      split = end - t != it.blocks;
      if (split) {
        int i0, n;
        if (by_round) {
          n = (it.blocks + TEAMS - 1) / TEAMS;
          i0 = s.rounds + (h * p.chunks + row0 / R) * n;
        } else if (even) {
          n = per_item;
          i0 = blockIdx.x / per_item * per_item;
        } else {
          i0 = owner(start);
          n = owner(start + it.blocks - 1) - i0 + 1;
        }
        const int word = (b * p.c.heads + h) * p.chunks + row0 / R;
        if (t == c0) open0 = t, at0 = i0, parts0 = n, word0 = word;
        else open1 = t, at1 = i0, parts1 = n, word1 = word;
      }
      const int lo = first_block<C>(p, s.len, s.count);
      const int tile0 = tile * NQ * 8;        // the warp's first row of the item
      const bool rows_here = tile0 < nrow;    // else this warp only frees the team's stages
      // B fragments of the warp's query rows (a lane loads row g4 of each tile), and what this lane has to know of the
      // rows in its accumulator columns, 2 c4 and 2 c4 + 1 of each tile
      uint32_t qf[NQ][KS][2];
      float mul[NQ][2];
      int at[NQ][2];  // position of the row's token; -1: the row is not there
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int r = row0 + tile0 + q * 8 + g4, tok = token_of(p, r);
        const bool there = r < p.rows && tok < s.count;
        const __nv_bfloat16* x = p.q + b * p.q_sb + (int64_t)(h * p.group + r - tok * p.group) * p.q_sh + tok * p.q_st;
        if (E4M3) {
          // fp16 rows: the largest magnitude to [2^14, 2^15) by a power of two, undone in the logits' factor. In
          // column 16 k + 4 c of a k16 step sit the two pairs the byte order of a cached row puts there.
          uint2 y[KS];
          unsigned m = 0;
#pragma unroll
          for (int k = 0; k < KS; ++k) y[k] = there ? *reinterpret_cast<const uint2*>(x + k * 16 + c4 * 4) : make_uint2(0, 0);
#pragma unroll
          for (int k = 0; k < KS; ++k)
            m = max(m, max(max((y[k].x << 16) & 0x7fffffffu, y[k].x & 0x7fff0000u),
                           max((y[k].y << 16) & 0x7fffffffu, y[k].y & 0x7fff0000u)));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const int e = m == 0 || m >= 0x7f800000u ? 15 : max(frexp_exp(__uint_as_float(m)), -110);
          const float f = exp2i(15 - e), undo = p.scale_log2 * exp2i(e - 15);
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            qf[q][k][0] = pack_f16(bf16lo(y[k].x) * f, bf16hi(y[k].x) * f);
            qf[q][k][1] = pack_f16(bf16lo(y[k].y) * f, bf16hi(y[k].y) * f);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) mul[q][i] = __shfl_sync(0xffffffffu, undo, (2 * c4 + i) * 4);
        } else {
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            qf[q][k][0] = there ? *reinterpret_cast<const uint32_t*>(x + k * 16 + c4 * 2) : 0u;
            qf[q][k][1] = there ? *reinterpret_cast<const uint32_t*>(x + k * 16 + 8 + c4 * 2) : 0u;
          }
          mul[q][0] = mul[q][1] = p.scale_log2;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r2 = row0 + tile0 + q * 8 + 2 * c4 + e, tok2 = token_of(p, r2);
          at[q][e] = r2 < p.rows && tok2 < s.count ? s.len - s.count + tok2 : -1;
        }
      }
      float o[NQ][KS][4] = {};  // O^T: 16 columns of the values x 8 query rows a tile
      float m[NQ][2], l[NQ][2];
#pragma unroll
      for (int q = 0; q < NQ; ++q) m[q][0] = m[q][1] = kNoMax, l[q][0] = l[q][1] = 0.f;
      // e4m3, of each row: vtop, 2^kWeightShift over it, the largest weighted scale that is known; the lane's smallest vtop
      float vtop[NQ][2], vmul[NQ][2], heavy[NQ][2], vlow = 0.f;
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) vtop[q][e] = heavy[q][e] = 0.f, vmul[q][e] = 1.f;
      const int pos_min = s.len - s.count, pos_max = s.len - 1;

      const int first = t + (team - (t - c0) % TEAMS + TEAMS) % TEAMS;
#pragma unroll 1
      for (int x = first; x < end; x += TEAMS) {
        // every lane looks once; only a wait in earnest is left to one lane and its limit
        if (!__all_sync(0xffffffffu, !dead && mbar_try_wait(&my_full[stage], phase)) &&
            (dead || !mbar_wait_warp(&my_full[stage], phase, &s_abort, p.c.err))) {
          dead = true;
          break;
        }
        const uint32_t kb = smem_u32(my_ring) + stage * (2 * C::KB);
        const float* ksc = my_scales + stage * (C::SC / 4) + g4;
        const int j0 = (lo + x - start) * C::BK;
        const int groups16 = rows_here ? min(NG, (s.len - j0 + 15) >> 4) : 0;
#pragma unroll 1
        for (int g = 0; g < groups16; ++g) {
          // S^T of 16 keys (rows g4, g4 + 8) x the query rows; for a single tile two accumulators shorten the chain of
          // dependent products. Fragments come in batches of four loads, so that a load's latency is met once a batch.
          const uint32_t ka = kb + g * C::GB + k_lane;
          constexpr int CH = NQ == 1 ? 2 : 1;
          float acc[NQ * CH][4];
          constexpr int KI = E4M3 ? KS / 2 : KS, KB4 = KI < 4 ? KI : 4;
#pragma unroll
          for (int k0 = 0; k0 < KI; k0 += KB4) {
            uint32_t r[KB4][4];
#pragma unroll
            for (int k = 0; k < KB4; ++k) ldsm4(r[k], chunk_from<C>(ka, 2 * (k0 + k)));
#pragma unroll
            for (int kk = 0; kk < KB4; ++kk)
#pragma unroll
              for (int half = 0; half < (E4M3 ? 2 : 1); ++half) {
                // bf16: a register is eight keys' chunk half; e4m3: eight keys' chunk, two k16 steps in the four
                const int k = E4M3 ? 2 * (k0 + kk) + half : k0 + kk;
                uint32_t a[4];
                if (E4M3) {
                  e4m3_f16(r[kk][2 * half], a[0], a[2]);
                  e4m3_f16(r[kk][2 * half + 1], a[1], a[3]);
                } else {
#pragma unroll
                  for (int i = 0; i < 4; ++i) a[i] = r[kk][i];
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                  float(&d)[4] = acc[q * CH + k % CH];
                  if (k < CH) mma16_first<E4M3>(d, a, qf[q][k][0], qf[q][k][1]);
                  else mma16<E4M3>(d, a, qf[q][k][0], qf[q][k][1]);
                }
              }
          }
          const int jg = j0 + g * 16;
          const bool whole = jg + 15 <= pos_min && (!p.window || jg > pos_max - p.window);
          float ks[2] = {1.f, 1.f}, vs[2];  // e4m3: scales of this lane's two keys
          if (E4M3) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              ks[i] = ksc[g * 16 + i * 8];
              vs[i] = ksc[C::BK + g * 16 + i * 8];
            }
          }
          // logits in units of log 2
          float sc[NQ][4];
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = CH == 2 ? acc[q * CH][e] + acc[q * CH + CH - 1][e] : acc[q][e];
              sc[q][e] = y * (E4M3 ? mul[q][e & 1] * ks[e >> 1] : mul[q][e & 1]);
            }
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int j = jg + g4 + i * 8;
              // the scale of a row that nobody sees may be anything
              if (E4M3 && (j > pos_max || (p.window && j <= pos_min - p.window))) vs[i] = 0.f;
#pragma unroll
              for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const bool see = j <= at[q][e] && (!p.window || j > at[q][e] - p.window);
                  if (!see) sc[q][2 * i + e] = -INFINITY;
                }
            }
          }
          if (p.logits) {
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (at[q][e & 1] >= 0)
                  p.logits[((int64_t)(b * p.c.heads + h) * p.rows + row0 + tile0 + q * 8 + 2 * c4 + (e & 1)) * p.c.cap + jg +
                           g4 + (e >> 1) * 8] = sc[q][e];
          }
          bool grew = false;
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) grew |= fmaxf(sc[q][e], sc[q][2 + e]) - m[q][e] > kSlack;
          if (E4M3) grew |= fmaxf(fabsf(vs[0]), fabsf(vs[1])) > vlow;
          if (__any_sync(0xffffffffu, grew)) {
            float top = 0.f;  // e4m3: the largest scale, infinities aside
            if (E4M3) {
              // rows of zeros have a scale too (append gives them 1): they count for nothing
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t any = 0;
#pragma unroll 1
                for (int k = c4; k < C::RB / 16; k += 4) {
                  uint32_t w[4];
                  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                               : "r"(kb + C::KB + g * C::GB + chunk_at<C>(g4 + i * 8, k)));
                  any |= (w[0] | w[1] | w[2] | w[3]) & 0x7f7f7f7fu;
                }
                any |= __shfl_xor_sync(0xffffffffu, any, 1);
                any |= __shfl_xor_sync(0xffffffffu, any, 2);
                if (fabsf(vs[i]) < INFINITY) {
                  if (any == 0) vs[i] = 0.f;
                  top = fmaxf(top, fabsf(vs[i]));
                }
              }
              top = column_max(top);
            }
            vlow = INFINITY;
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
              float fac[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float was = m[q][e];
                m[q][e] = fmaxf(was, column_max(fmaxf(sc[q][e], sc[q][2 + e])));
                fac[e] = ex2(was - m[q][e]);
                l[q][e] *= fac[e];
                if (E4M3) {
                  float y = 0.f;
#pragma unroll
                  for (int i = 0; i < 2; ++i)
                    if (fabsf(vs[i]) < INFINITY) y = fmaxf(y, ex2(sc[q][2 * i + e] - m[q][e]) * fabsf(vs[i]));
                  heavy[q][e] = fmaxf(heavy[q][e] * fac[e], column_max(y));
                  const float v = vtop[q][e];
                  float now = top > v ? top * 4.f : v;  // two bits of room, so that the next ones rarely come here
                  if (heavy[q][e] > 0.f) now = fminf(now, heavy[q][e] * kRange);
                  now = fminf(fmaxf(now, 0x1p-110f), 0x1p126f);
                  now = fmaxf(now, fac[e] * v * 0x1p-40f);  // what the row has summed up stays in fp32's range
                  fac[e] = fac[e] * v / now;
                  vtop[q][e] = now;
                  vmul[q][e] = (float)(1 << kWeightShift) / now;
                  vlow = fminf(vlow, now);
                }
              }
#pragma unroll
              for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[q][k][e] *= fac[e & 1];
            }
          }
          float pw[NQ][4];  // weights for the output
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = ex2(sc[q][e] - m[q][e & 1]);
              l[q][e & 1] += w;
              // the scale first: over a vtop that is far below, it could pass fp32's range where the product does not
              pw[q][e] = E4M3 ? w * vs[e >> 1] * vmul[q][e & 1] : w;
            }
          const uint32_t vg = kb + C::KB + g * C::GB, va = vg + v_lane;
          bool odd = false;
          if (!whole) {
            // A masked weight is 0, but 0 x NaN is not: if the values of a partly masked group hold infinities or
            // NaNs (stale slots, a later token's), those are added here, to the rows that see them, and are zeros in
            // the products below; all other bits of the result stay what they are without them.
#pragma unroll 1
            for (int i = lane; i < C::GB / 16; i += 32) {
              uint32_t w[4];
              asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vg + i * 16));
#pragma unroll
              for (int k = 0; k < 4; ++k)
                odd |= (E4M3 ? __vcmpeq4(w[k] & 0x7f7f7f7fu, 0x7f7f7f7fu) : __vcmpeq2(w[k] & 0x7f807f80u, 0x7f807f80u)) != 0;
            }
            odd = __any_sync(0xffffffffu, odd);
            if (E4M3) {  // a scale may be NaN too
#pragma unroll
              for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (sc[q][e] == -INFINITY) pw[q][e] = 0.f;
            }
            if (odd) {
#pragma unroll 1
              for (int k = 0; k < 16; ++k) {
                const int j = jg + k;
                float w[NQ][2];
                bool see[NQ][2];
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const float w0 = __shfl_sync(0xffffffffu, pw[q][e], (k & 7) * 4 + c4);
                    const float w1 = __shfl_sync(0xffffffffu, pw[q][2 + e], (k & 7) * 4 + c4);
                    w[q][e] = k < 8 ? w0 : w1;
                    see[q][e] = j <= at[q][e] && (!p.window || j > at[q][e] - p.window);
                  }
#pragma unroll
                for (int n = 0; n < KS; ++n) {
                  // this lane's two output rows of tile n: bf16 columns g4 and g4 + 8, e4m3 columns 2 g4 and 2 g4 + 1
                  float y[2];
                  if (E4M3) {
                    unsigned short v;
                    asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(vg + chunk_at<C>(k, n) + g4 * 2));
                    uint32_t lo2, hi2;
                    e4m3_f16(v, lo2, hi2);
                    y[0] = f16lo(lo2);
                    y[1] = f16hi(lo2);
                  } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                      unsigned short v;
                      asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(vg + chunk_at<C>(k, 2 * n + i) + g4 * 2));
                      y[i] = bf16lo(v);
                    }
                  }
#pragma unroll
                  for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                      if (see[q][e & 1] && !isfinite(y[e >> 1])) o[q][n][e] += w[q][e & 1] * y[e >> 1];
                }
              }
            }
          }
          // P^T as the products' B operand. e4m3: fp16, 11 bits, on values that are exact in fp16. bf16: in two parts
          // (16 bits of them): one part would add its 2^-9 to the output's own rounding. The first is cut
          // off, not rounded, and the second more than 0, so that an infinite value makes both products infinite, of
          // one sign; a weight of 0 has two zeros
          uint32_t hi[NQ][2], lw[NQ][2];
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float y = pw[q][2 * i], z = pw[q][2 * i + 1];
              const uint32_t w = E4M3 ? pack_f16(y, z) : __byte_perm(__float_as_uint(y), __float_as_uint(z), 0x7632);
              hi[q][i] = transpose8(w);
              if (!E4M3)
                lw[q][i] = transpose8(pack_bf16(fmaxf(y - bf16hi(__float_as_uint(y)), fminf(y, 0x1p-126f)),
                                                fmaxf(z - bf16hi(__float_as_uint(z)), fminf(z, 0x1p-126f))));
            }
          constexpr int VI = E4M3 ? KS / 2 : KS, VB4 = VI < 4 ? VI : 4;
#pragma unroll
          for (int k0 = 0; k0 < VI; k0 += VB4) {
            uint32_t r[VB4][4];
#pragma unroll
            for (int k = 0; k < VB4; ++k) {
              ldsm4t(r[k], chunk_from<C>(va, 2 * (k0 + k)));
              if (odd) finite_only<E4M3>(r[k]);
            }
#pragma unroll
            for (int kk = 0; kk < VB4; ++kk) {
              if (E4M3) {
                // a register holds columns 2 n, 2 n + 1 of keys 2 c, 2 c + 1: paired by keys, the even columns of a
                // chunk are the tile's rows 0-7 and the odd ones its rows 8-15
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  uint32_t a[4];
                  e4m3_f16(__byte_perm(r[kk][2 * i], 0, 0x3120), a[0], a[1]);
                  e4m3_f16(__byte_perm(r[kk][2 * i + 1], 0, 0x3120), a[2], a[3]);
#pragma unroll
                  for (int q = 0; q < NQ; ++q) mma16<true>(o[q][2 * (k0 + kk) + i], a, hi[q][0], hi[q][1]);
                }
              } else {
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                  mma16<false>(o[q][k0 + kk], r[kk], hi[q][0], hi[q][1]);
                  mma16<false>(o[q][k0 + kk], r[kk], lw[q][0], lw[q][1]);
                }
              }
            }
          }
        }
        __syncwarp();  // this warp has read the stage
        bool freed = true;
        if (S > 1 && tile > 0) {
          if (lane == 0) mbar_arrive(&my_empty[stage]);
        } else if (u.len) {
          // the team's other warps run on the same block, so they are about done with it too
          if (S > 1) freed = mbar_wait_warp(&my_empty[stage], phase, &s_abort, p.c.err);
        }
        --waiting;
        stage = stage + 1 == p.stages ? 0 : stage + 1;
        phase ^= stage == 0;
        if (!freed) {
          dead = true;
          break;
        }
        if (tile == 0 && u.len) issue();
      }

      // the warps' parts of the item
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = tile0 + q * 8 + 2 * c4 + e;  // row of the item
          const float f = E4M3 ? vtop[q][e] * (1.f / (1 << kWeightShift)) : 1.f;
          l[q][e] = column_sum(l[q][e]);
          if (g4 == 0) s_ms[team * R + r] = make_float2(m[q][e], l[q][e]);
          if (r >= nrow) continue;
          float* dst = merge + (size_t)(team * R + r) * MP;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            if (E4M3) {
              *reinterpret_cast<float2*>(dst + k * 16 + g4 * 2) = make_float2(o[q][k][e] * f, o[q][k][2 + e] * f);
            } else {
              dst[k * 16 + g4] = o[q][k][e];
              dst[k * 16 + 8 + g4] = o[q][k][2 + e];
            }
          }
        }
      __syncthreads();
    }
    float* part = p.part + (2 * (size_t)blockIdx.x + (t == c0 ? 0 : 1)) * part_ld;
#pragma unroll 1
    for (bool again = false;; again = true) {  // again: the thread groups' sums of a join
      const int group = groups == 1 ? 0 : tid / n4;
#pragma unroll 1
      for (int i = tid - group * n4; i < n4 && group < groups; i += NTHREADS) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        const float* x = src + (again ? i * 4 : r * pitch + d);
        const float2* y = ms + (again ? i : r);
        float a = kNoMax, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int k0 = group; k0 < parts; k0 += V * groups) {
          float2 z[V];
          float4 w[V];
          float top = a;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int k = k0 + j * groups;
            const size_t off = k ? 0 : skip0;
            z[j] = make_float2(kNoMax, 0.f);
            w[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < parts) {
              z[j] = y[k * ms_ld + off / 2];
              w[j] = *reinterpret_cast<const float4*>(x + k * src_ld + off);
            }
          }
#pragma unroll
          for (int j = 0; j < V; ++j) top = fmaxf(top, z[j].x);
          float f = ex2(a - top);
          a = top;
          sum *= f;
          v.x *= f; v.y *= f; v.z *= f; v.w *= f;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            f = ex2(z[j].x - top);
            sum += z[j].y * f;
            v.x += w[j].x * f; v.y += w[j].y * f; v.z += w[j].z * f; v.w += w[j].w * f;
          }
        }
        if (groups > 1) {
          *reinterpret_cast<float4*>(merge + tid * 4) = v;
          s_group[tid] = make_float2(a, sum);
        } else if (split) {
          *reinterpret_cast<float4*>(part + r * D + d) = v;
          if (d == 0) *reinterpret_cast<float2*>(part + p.nr * D + 2 * r) = make_float2(a, sum);
        } else {
          // v / sum as bf16; zeros for rows that see nothing
          const int row = row0 + r, tok = token_of(p, row);
          const float g = sum == 0.f || tok >= s.count ? 0.f : __fdividef(1.f, sum);
          if (g == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<uint2*>(p.out + b * p.o_sb + (int64_t)(h * p.group + row - tok * p.group) * p.o_sh +
                                    tok * p.o_st + d) = make_uint2(pack_bf16(v.x * g, v.y * g), pack_bf16(v.z * g, v.w * g));
          if (p.lse && d == 0) p.lse[(int64_t)(b * p.c.heads + h) * p.rows + row] = a + log2f(sum);
        }
      }
      if (groups == 1) break;
      __syncthreads();
      src = merge;
      src_ld = n4 * 4;
      ms = s_group;
      ms_ld = n4;
      skip0 = 0;
      parts = groups;
      groups = 1;
    }
    __syncthreads();  // the merge area is free
    if (!join) t = min(c1, start + it.blocks + kPad);
  }
  if (dead && tile == 0) {  // see the team's copies in flight through, again with a limit, before leaving
    for (int i = 0; lane == 0 && i < waiting; ++i) {
      volatile int never = 0;
      mbar_wait(&my_full[stage], phase, &never, p.c.err);
      stage = stage + 1 == p.stages ? 0 : stage + 1;
      phase ^= stage == 0;
    }
    __syncwarp();
  }
}

// weights[b, h, j] += sum_r e^(s_rj - log-sum_r) over the head's query rows, from the logits the attention left
// (fp32, 4 rows bytes a position, where the cache has 2 D to 4 D) and its row sums. Two positions a thread, eight rows
// in flight: with few sequences there are few threads, and each has all rows to go through.
constexpr int kWeightThreads = 128;
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(const AttendParams p, float* weights, int64_t w_sb, int64_t w_sh,
                                                                 int block_keys) {
  constexpr int SPAN = kWeightThreads * 2, V = 8;
  pdl_launch_dependents();
  pdl_wait();
  const int per = (p.c.cap + SPAN - 1) / SPAN;
  for (int64_t x = blockIdx.x; x < (int64_t)p.c.batch * p.c.heads * per; x += gridDim.x) {
    const int bh = (int)(x / per), b = bh / p.c.heads, h = bh - b * p.c.heads;
    const int len = paged_len(p.c, b), n = paged_count(p.c, p.counts, b, p.T, len);
    const int lo = p.window ? max(0, len - n + 1 - p.window) / block_keys * block_keys : 0;
    const int j = (int)(x - (int64_t)bh * per) * SPAN + threadIdx.x * 2;
    if (n == 0 || j + 1 < lo || j >= len) continue;
    const float* logits = p.logits + (int64_t)bh * p.rows * p.c.cap + j;
    const float* lse = p.lse + (int64_t)bh * p.rows;
    float* w = weights + b * w_sb + h * w_sh + j;
    const float old[2] = {w[0], j + 1 < len ? w[1] : 0.f};
    float a[2] = {};
    const int rows = n * p.group;
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += V) {
      float2 v[V];
      float z[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        z[k] = r0 + k < rows ? lse[r0 + k] : -INFINITY;
        if (r0 + k < rows) v[k] = *reinterpret_cast<const float2*>(logits + (int64_t)(r0 + k) * p.c.cap);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (z[k] == -INFINITY) continue;  // past the rows, or a row that sees nothing
        if (z[k] != z[k]) {  // a row of NaN weights: only what it sees
          const int at = len - n + token_of(p, r0 + k), from = p.window ? at - p.window + 1 : 0;
          if (j >= from && j <= at) a[0] = z[k];
          if (j + 1 >= from && j + 1 <= at) a[1] = z[k];
          continue;
        }
        a[0] += ex2(v[k].x - z[k]);
        a[1] += ex2(v[k].y - z[k]);
      }
    }
    if (j >= lo) w[0] = old[0] + a[0];
    if (j + 1 >= lo && j + 1 < len) w[1] = old[1] + a[1];
  }
}

// ------------------------------------------------------------------ host

int tile_map(CUtensorMap* map, void* base, const tbf16_paged_cache* c, int64_t sp, int64_t sh, int64_t ss, int box) {
  const int item = c->dtype == TBF16_E4M3 ? 1 : 2, span = (int)std::min<int64_t>(c->D * item, 128);
  return tbf16_host::make_tmap_pages(map, base, item, c->D, span, c->page_size, c->heads, c->pages, ss, sh, sp, box);
}

constexpr int kSmemMax = 227 * 1024;

template <class C>
int attend_smem(const AttendParams& p) {
  return C::TEAMS * p.stages * (2 * C::KB + C::SC) + C::MERGE * 4 + (p.c.batch + 1) * (int)sizeof(SeqInfo);
}
// Static shared memory of the kernel, rounded up.
constexpr int kSmemStatic = 4 * 1024;

template <class C>
int launch_attend(const tbf16_paged_cache* cache, AttendParams& p, const tbf16_host::DeviceInfo* dev, cudaStream_t st) {
  CUtensorMap km, vm;
  const int box = (int)std::min<int64_t>(C::BK, cache->page_size);
  p.box_shift = 0;
  while ((1 << p.box_shift) < box) ++p.box_shift;
  if (int s = tile_map(&km, cache->k, cache, cache->k_sp, cache->k_sh, cache->k_ss, box)) return s;
  if (int s = tile_map(&vm, cache->v, cache, cache->v_sp, cache->v_sh, cache->v_ss, box)) return s;
  static_assert(C::MERGE >= C::W * 32 * 4, "room for a join's thread groups");
  p.stages = C::MAX_STAGES;
  const int smem = attend_smem<C>(p);  // a batch of 1024 with 256-wide bf16 rows takes 216 KB
  if (smem + kSmemStatic > kSmemMax) return TBF16_ERR_UNSUPPORTED;
  static bool attr_done[64] = {false};
  if (!attr_done[dev->device & 63]) {
    if (cudaFuncSetAttribute(attend_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - kSmemStatic) !=
        cudaSuccess) {
      cudaGetLastError();
      return TBF16_ERR_LAUNCH;
    }
    attr_done[dev->device & 63] = true;
  }
  return tbf16_host::launch_pdl(attend_kernel<C>, dev->sms, C::W * 32, smem, 1, st, km, vm, p);
}

// Query rows of an item. Heads with more than 32 make several items of the same keys,
// which run at the same time and find most of them in L2.
int item_rows(int64_t rows) { return rows <= 8 ? 8 : rows <= 16 ? 16 : 32; }

struct Workspace {
  int64_t rows, chunks, nr, part, lse, logits;  // sizes in floats, in this order
  Workspace(const tbf16_paged_cache* c, int64_t Hq, int64_t T, bool weights, int sms) {
    rows = T * (Hq / c->heads);
    const int R = item_rows(rows);
    chunks = (rows + R - 1) / R;
    nr = std::min<int64_t>(rows, R);
    part = 2 * (int64_t)sms * partial_floats((int)nr, (int)c->D);
    lse = weights ? (c->batch * c->heads * rows + 3) / 4 * 4 : 0;
    logits = weights ? c->batch * c->heads * rows * c->max_pages * c->page_size : 0;
  }
  int64_t bytes() const { return (part + lse + logits) * 4; }
};

template <int D, bool E4M3>
int launch_rows(const tbf16_paged_cache* cache, AttendParams& p, const tbf16_host::DeviceInfo* dev, cudaStream_t st) {
  // Up to 16 rows in one warp: a cached fragment is read from shared memory and converted once for both tiles. 256-wide
  // outputs of two tiles would not fit a warp's registers; there, and for 32 rows, two or four warps share a block
  // (16 query heads on one of 128, 8 sequences of 32768 tokens: two tiles 36 us, two warps 51; on one of 256: 80 and 64).
  constexpr bool WIDE = D == 256;
  const int R = item_rows(p.rows);
  if (R == 8) return launch_attend<Tile<D, E4M3, 1, 1>>(cache, p, dev, st);
  if (R == 16) return launch_attend<Tile<D, E4M3, WIDE ? 1 : 2, WIDE ? 2 : 1>>(cache, p, dev, st);
  return launch_attend<Tile<D, E4M3, WIDE ? 1 : 2, WIDE ? 4 : 2>>(cache, p, dev, st);
}

bool attend_sizes_ok(const tbf16_paged_cache* c, int64_t Hq, int64_t T) {
  return c && c->batch >= 0 && c->heads >= 1 && Hq >= 1 && Hq <= 65536 && Hq % c->heads == 0 && T >= 0 && T <= 4096 &&
         T * (Hq / c->heads) <= 65536;
}

}  // namespace

extern "C" int64_t tbf16_paged_attend_ws_size(const tbf16_paged_cache* cache, int64_t Hq, int64_t T, int with_weights) {
  const tbf16_host::DeviceInfo* dev = tbf16_host::device_info();
  if (!dev || !attend_sizes_ok(cache, Hq, T)) return 0;
  return Workspace(cache, Hq, T, with_weights != 0, dev->sms).bytes();
}

extern "C" int64_t tbf16_paged_attend_sync_size(const tbf16_paged_cache* cache, int64_t Hq, int64_t T) {
  if (!attend_sizes_ok(cache, Hq, T)) return 0;
  return cache->batch * cache->heads * Workspace(cache, Hq, T, false, 0).chunks * 4;
}

extern "C" int tbf16_paged_attend(const tbf16_paged_cache* cache, const void* q, int64_t q_sb, int64_t q_sh,
                                  int64_t q_st, int64_t Hq, int64_t T, const int32_t* counts, float scale,
                                  int64_t window, void* out, int64_t out_sb, int64_t out_sh, int64_t out_st,
                                  float* weights, int64_t w_sb, int64_t w_sh, void* sync, void* ws, int64_t ws_bytes,
                                  void* stream) {
  if (int st = tbf16_host::require_sm100()) return st;
  AttendParams p;
  if (int st = tbf16_host::paged_view(cache, &p.c)) return st;
  if (T == 0 || cache->batch == 0) return TBF16_OK;
  if (!q || !out || !attend_sizes_ok(cache, Hq, T) || window < 0 || !(scale == scale)) return TBF16_ERR_INVALID;
  for (int64_t s : {q_sb, q_sh, q_st, out_sb, out_sh, out_st}) {
    if (s < 0) return TBF16_ERR_INVALID;
    if (s % 8) return TBF16_ERR_ALIGN;
  }
  if (!tbf16_host::aligned16(q) || !tbf16_host::aligned16(out) || !tbf16_host::aligned16(ws)) return TBF16_ERR_ALIGN;
  const tbf16_host::DeviceInfo* dev = tbf16_host::device_info();
  const Workspace need(cache, Hq, T, weights != nullptr, dev->sms);
  if (!sync || !ws || ws_bytes < need.bytes()) return TBF16_ERR_INVALID;
  // blocks are counted in 32 bits, 16 keys at the least in each
  if (cache->batch * cache->heads * need.chunks > INT32_MAX / (p.c.cap / 16 + 1 + kPad)) return TBF16_ERR_INVALID;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_sb; p.q_sh = q_sh; p.q_st = q_st;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_sb = out_sb; p.o_sh = out_sh; p.o_st = out_st;
  p.counts = counts;
  p.T = (int)T;
  p.group = (int)(Hq / cache->heads);
  p.group_inv = (unsigned)(((UINT64_C(1) << 32) + p.group - 1) / p.group);
  p.rows = (int)need.rows;
  p.chunks = (int)need.chunks;
  p.nr = (int)need.nr;
  p.window = (int)(window > p.c.cap ? 0 : window);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.sync = static_cast<unsigned*>(sync);
  p.part = static_cast<float*>(ws);
  p.lse = weights ? p.part + need.part : nullptr;
  p.logits = weights ? p.lse + need.lse : nullptr;
  const bool e4m3 = cache->dtype == TBF16_E4M3;
  auto st = static_cast<cudaStream_t>(stream);
  int rc;
  if (cache->D == 64) rc = e4m3 ? launch_rows<64, true>(cache, p, dev, st) : launch_rows<64, false>(cache, p, dev, st);
  else if (cache->D == 128) rc = e4m3 ? launch_rows<128, true>(cache, p, dev, st) : launch_rows<128, false>(cache, p, dev, st);
  else rc = e4m3 ? launch_rows<256, true>(cache, p, dev, st) : launch_rows<256, false>(cache, p, dev, st);
  if (rc != TBF16_OK || !weights) return rc;
  const int block_keys = cache->D * (e4m3 ? 1 : 2) <= 64 ? 64 : cache->D * (e4m3 ? 1 : 2) <= 128 ? 32 : 16;
  const int span = kWeightThreads * 2;
  const int64_t blocks = cache->batch * cache->heads * ((p.c.cap + span - 1) / span);
  return tbf16_host::launch_pdl(weights_kernel, (unsigned)std::min<int64_t>(blocks, (int64_t)dev->sms * 16), kWeightThreads, 0, 1, st, p, weights, w_sb,
                    w_sh, block_keys);
}
