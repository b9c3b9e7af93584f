// Attention of new tokens over a paged KV cache (see paged.cuh), grouped-query aware.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the keys j <= p of the token's sequence, p its position.
//
// A CTA works on one KV head and a block of new tokens of one sequence, over all keys or a part of them. The G = Hq / Hkv query heads of the KV head
// are packed with the tokens into the 128 rows of a tile (row = token * G + head), so that keys and values are read once for all of them
// whatever G is. The dataflow is that of attn_fwd3.cu: S = Q K^T in tensor memory, a softmax thread to a row, P back into tensor memory as the
// A operand of O += P V, the output rescaled only when a row's maximum has grown by 2^8; tiles of 128 keys, assembled by TMA from the
// sequence's pages (one box for a page's rows, or a part of a longer page) into the same swizzled layout. What is different:
//
//  * Two tiles to a CTA. With more than 128 rows they are two tiles of rows that share the keys; with 128 or less (single tokens, short
//    chunks) they are the same rows at every other 128 keys, added up at the end: one tile alone would wait for its own softmax.
//  * Work is dealt out on the device, from the lengths as they are at that time: a warp of every CTA scans them. Where the blocks do not fill the
//    machine, the keys of every block are cut into pieces whose results a second kernel joins (see paged_plan).
//  * Rows behind a sequence's last key may hold anything. Scores there are set to -inf, but a product takes 0 * V too, so an idle warp clears those
//    rows of V in shared memory before the tile is handed on. Pages that are not there, and those behind the last, are zeros from TMA (a
//    coordinate outside of the pool).
//
// Scores, maxima, sums and outputs are fp32; P is rounded to bf16 for its product (an operand has no more bits), while the sum that divides the
// result is of P before that: a result is 0.0020 to 0.0023 of its norm off, of which its own rounding to bf16 is 0.0017. (The decode kernel, which
// memory bounds, takes P in two terms.)
//
// What bounds it. Whole prompts: a step of 256 rows takes 1.9 us, 0.8 of the tensor rate (exponentials share it, as in attn_fwd3.cu), and every CTA some 7 us
// beside its steps (first scores after 5.2 us, results 5.3 us behind the last step), which nothing covers: a CTA has its SM to itself. 15712 steps of
// 1344 blocks on 148 SMs are 202 us without the second and 271 with it, measured 269. us, dense / pages of 64 / 16: [1, 4096] with 32 / 8 heads of 128 133 / 135 /
// 136 (1000 TFLOP/s), [4, 2987] with 32 / 32 heads 325 / 327 / 327, [8, 1024] with 12 / 12 heads of 64 44 / 49 / 49 (8 steps of a CTA at most).
// The next 512 tokens over 7681 keys, 32 / 8 heads: 71 us (870 TFLOP/s), two pieces of 64 blocks on 128 of 148 SMs, 60 of it in steps. A block of one tile takes half as long and is cut into half as many pieces: 284
// tokens over 5983 keys, 25 / 25 heads of 64, 40 us, with as many as the others 53. Few rows: keys come at 6 TB/s while steps run, and the ends of it, 5 us
// in front and 6 behind with the second kernel, are what is left: 5 tokens over 30000 keys 35 us (3.5 TB/s), 16 over 2000 12.
#include "paged.cuh"

namespace gf {

constexpr int PG_TILE = 128;      // rows of a tile, keys of a step
constexpr int PG_THREADS = 384;   // warpgroup 0: TMA warp, MMA warp, warp that clears rows, an idle one; warpgroups 1 and 2: softmax of tile 0 / 1
constexpr int PG_REGS_CTRL = 104; // 128 x 104 + 256 x 200 = 64512, the block's own at launch (384 x 168)
constexpr int PG_REGS_SOFTMAX = 200;
constexpr int PG_PARTS = 2;       // P V of a tile is issued in this many parts of the keys
constexpr float PG_RESCALE = 8.0f;  // log2 units

struct PagedAttn {
  PagedBatch seqs;
  int Hq, Hkv, G, tq, tb;        // G = Hq / Hkv, tq = 128 / G tokens of a tile, tb of a block: tq or two times that
  int slots;                     // CTAs that run at a time; 0: no block is cut
  int skip_ones;                 // sequences of one new token are not this kernel's
  float scale;
  __nv_bfloat16* out;            // [T, Hq, D], rows ldo apart
  long long ldo;
  int* cut;                      // how many blocks were cut into pieces (all, or 0)
  int4* where;                   // for each of them, what the kernel that joins pieces wants to know (see there)
  float* part;                   // [item][rows][D], then [item][rows][maximum, sum]
  float* part_ml;
  int rows, items, blocks;       // rows of an item in `part`, items and blocks (of all KV heads) at most
};

constexpr int PG_WHOLE = 1 << 30;   // no block is cut
struct PgShape {                 // what a sequence is cut into
  int n, len, keys, blocks, steps;
  bool short_end;                // its last block has rows for one tile alone (see `alternate` below), and takes half as long
  // pieces of a block, none longer than U steps of two tiles
  __device__ __forceinline__ int pieces(bool end, int U) const {
    if (U == PG_WHOLE) return 1;
    if (end && short_end) U *= 2;
    return (unsigned)(steps + U - 1) / (unsigned)U;
  }
  __device__ __forceinline__ int items(int U) const { return blocks == 0 ? 0 : (blocks - 1) * pieces(false, U) + pieces(true, U); }
  __device__ __forceinline__ int longest() const { return blocks == 0 ? 0 : blocks == 1 && short_end ? (steps + 1) / 2 : steps; }     // block, uncut
};
__device__ __forceinline__ PgShape pg_shape(const PagedAttn& p, int b) {
  PgShape s;
  s.n = max(0, p.seqs.end(b) - p.seqs.first(b));
  if (p.skip_ones && s.n == 1) s.n = 0;
  s.len = p.seqs.lens[b];
  s.keys = (int)min((long long)max(s.len, 0), p.seqs.capacity());
  s.blocks = (s.n + p.tb - 1) / p.tb;
  s.steps = max(1, (s.keys + PG_TILE - 1) / PG_TILE);
  s.short_end = s.n - (s.blocks - 1) * p.tb <= p.tq;
  return s;
}

// Whole warp: steps of a piece. All blocks uncut where they fill the machine; else the shortest pieces that run at one time, or, of cuts in 2, 3
// and 4, the one whose waves of CTAs take the least (a piece costs about 3 steps of its own). `own`: the lane's sequence of the first 32.
__device__ __forceinline__ int paged_plan(const PagedAttn& p, const PgShape& own, int& whole) {
  constexpr int OWN = 3;
  if (p.slots == 0) return PG_WHOLE;
  const int lane = threadIdx.x & 31;
  auto sum = [&](auto f) {
    int n = f(own);
    for (int b = lane + 32; b < p.seqs.B; b += 32) n += f(pg_shape(p, b));
    return __reduce_add_sync(0xffffffffu, n) * p.Hkv;
  };
  auto items = [&](int U) { return sum([&](const PgShape& s) { return s.items(U); }); };
  whole = sum([](const PgShape& s) { return s.blocks; });
  if (whole == 0) return PG_WHOLE;
  if (2 * whole <= p.slots) {
    int U = max(1, (sum([](const PgShape& s) { return max(0, s.blocks - 1) * s.steps + (s.blocks == 0 ? 0 : s.short_end ? (s.steps + 1) / 2 : s.steps); }) + p.slots - 1) / p.slots);
#pragma unroll 1
    while (items(U) > p.slots) U += 1 + U / 16;    // ends: with whole blocks there are no more than half of them
    return U;
  }
  int most = own.longest();
  for (int b = lane + 32; b < p.seqs.B; b += 32) most = max(most, pg_shape(p, b).longest());
  most = __reduce_max_sync(0xffffffffu, most);
  int best = PG_WHOLE, cost = (whole + p.slots - 1) / p.slots * (most + OWN);
#pragma unroll 1
  for (int k = 2; k <= 4 && most > 0; ++k) {
    const int U = (most + k - 1) / k, n = items(U);
    const int c = (n + p.slots - 1) / p.slots * (U + OWN);
    if (n <= 2 * p.slots && c < cost) {
      cost = c;
      best = U;
    }
  }
  return best;
}

// A block of a sequence, and the keys of a piece of it.
struct PgItem {
  int b, hk, token, tokens, pos, len, keys, pieces, j0, j1;     // first token (row of q), how many, position of the first; steps j0 .. j1 - 1
  int piece, block;              // which one, of which block
  __device__ __forceinline__ int visible(int upto) const {   // keys that the last of the first `upto` tokens sees
    return max(0, min(pos + min(upto, tokens), keys));
  }
  __device__ __forceinline__ int steps(int upto) const { return (visible(upto) + PG_TILE - 1) / PG_TILE; }
};
__device__ __forceinline__ void pg_block(const PagedAttn& p, PgItem& it, const PgShape& s, int b, int blk) {
  it.b = b;
  it.token = p.seqs.first(b) + blk * p.tb;
  it.tokens = min(p.tb, s.n - blk * p.tb);
  it.pos = s.len - s.n + blk * p.tb;
  it.len = s.len;
  it.keys = s.keys;
}

// Whole warp: item x; false behind the last one. Inside a sequence the last block (the most keys) comes first, its heads and pieces
// next to each other.
__device__ __forceinline__ bool pg_find(const PagedAttn& p, const PgShape& own, int x, int U, PgItem& it) {
  const int lane = threadIdx.x & 31;
  const bool cuts = p.slots != 0;
  const int mask = cuts ? 0xffff : -1;
#pragma unroll 1
  for (int base = 0, before = 0; base < p.seqs.B; base += 32) {
    PgShape s = base == 0 ? own : base + lane < p.seqs.B ? pg_shape(p, base + lane) : PgShape{};
    int each = s.pieces(false, U), at_end = s.pieces(true, U);
    const int n = s.blocks == 0 ? 0 : ((s.blocks - 1) * each + at_end) * p.Hkv;
    const int both = cuts ? n | (s.blocks * p.Hkv) << 16 : n;          // items, and blocks: both are less than 2^16 where any may be cut
    int incl = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, ((before + incl) & mask) > x);
    if (hit) {
      const int l = __ffs(hit) - 1, front = before + __shfl_sync(0xffffffffu, incl - both, l), rem = x - (front & mask);
      s.n = __shfl_sync(0xffffffffu, s.n, l);
      s.len = __shfl_sync(0xffffffffu, s.len, l);
      s.keys = __shfl_sync(0xffffffffu, s.keys, l);
      s.blocks = __shfl_sync(0xffffffffu, s.blocks, l);
      each = __shfl_sync(0xffffffffu, each, l);
      at_end = __shfl_sync(0xffffffffu, at_end, l);
      const int behind = rem - at_end * p.Hkv;               // the items of the last block
      int blk = s.blocks - 1, in = rem;
      it.pieces = at_end;
      if (behind >= 0) {
        const int q = behind / (each * p.Hkv);
        in = behind - q * each * p.Hkv;
        blk -= 1 + q;
        it.pieces = each;
      }
      pg_block(p, it, s, base + l, blk);
      const int steps = it.steps(p.tb);
      it.hk = in;
      it.piece = it.j0 = 0;
      it.j1 = steps;
      if (it.pieces > 1) {                                   // steps piece / pieces and steps (piece + 1) / pieces, in 32 bits
        const unsigned pieces = it.pieces, piece = in % pieces, part = steps / pieces, rest = steps - part * pieces;
        it.hk = in / pieces;
        it.piece = piece;
        it.j0 = piece * part + piece * rest / pieces;
        it.j1 = (piece + 1) * part + (piece + 1) * rest / pieces;
      }
      it.block = (front >> 16) + (s.blocks - 1 - blk) * p.Hkv + it.hk;       // (where blocks may be cut)
      return it.pieces == 1 || x < p.items;                  // (no more pieces are made than there is room for)
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

template <int HD>
struct PgCfg {
  static constexpr int CH = HD / 64;
  static constexpr int TILE_BYTES = PG_TILE * HD * 2;
  static constexpr int OFF_Q = 0;                                   // 2 tiles
  static constexpr int OFF_K = OFF_Q + 2 * TILE_BYTES;              // 2 stages; at the end the sums of tile 1's keys
  static constexpr int OFF_V = OFF_K + 2 * TILE_BYTES;              // 2 stages
  static constexpr int OFF_BAR = OFF_V + 2 * TILE_BYTES;
  static constexpr int OFF_ML = OFF_BAR + 256;                      // maxima and sums of tile 1's keys
  static constexpr int SMEM_BYTES = OFF_ML + 2 * PG_TILE * 4 + 1024;
  static constexpr int TM_S = 0;      // + t * 128; P (bf16 pairs) occupies the first 64 columns of the same region
  static constexpr int TM_O = 256;    // + t * 128
  static constexpr int TMEM_COLS = 512;
  static_assert(PG_TILE * HD * 4 <= 2 * TILE_BYTES, "sums fit in the stages of K");
};

__device__ __forceinline__ float pg_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 4-D tile load global -> shared
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

template <int HD>
__global__ void __launch_bounds__(PG_THREADS, 1)
paged_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedAttn p) {
  using Cfg = PgCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem + Cfg::OFF_Q;
  uint8_t* sK = smem + Cfg::OFF_K;
  uint8_t* sV = smem + Cfg::OFF_V;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;    // [2]
  uint64_t* k_empty = bars + 3;   // [2]
  uint64_t* v_full = bars + 5;    // [2]
  uint64_t* v_empty = bars + 7;   // [2]
  uint64_t* s_full = bars + 9;    // [2] per tile
  uint64_t* o_done = bars + 11;   // [2] per tile
  uint64_t* v_tail = bars + 13;   // the last V tile before its rows behind the sequence are cleared
  uint64_t* p_full = bars + 14;   // [2][PG_PARTS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14 + 2 * PG_PARTS);
  __shared__ PgItem shared_item;
  __shared__ int shared_there, shared_failed;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  auto fail = [&](int code) {                      // a wait that ran out
    if (p.seqs.status) atomicCAS(p.seqs.status, 0, code);
    shared_failed = 1;
  };
  PgItem it{};
  bool there = false, alternate, clears;
  int n_j, tail, box;
  auto derive = [&](const PgItem& o) {
    alternate = o.tokens <= p.tq;
    n_j = o.j1 - o.j0;
    // the last step's V has rows behind the sequence inside a page
    box = min(PG_TILE, 1 << p.seqs.page_shift);
    tail = o.keys - (o.j1 - 1) * PG_TILE;                            // rows of the last step that are keys
    clears = n_j > 0 && tail < PG_TILE && (tail & (box - 1)) != 0;
  };
  // A CTA of few steps is mostly this: the queries are on their way before the other warps have started. (Keys and values too was slower: the
  // producer's code then stands twice, and the softmax warps spill.)
  if (warp == 0) {
    PgShape own{};
    if (lane < p.seqs.B) own = pg_shape(p, lane);
    if (lane == 0) {
      mbar_init(q_full, 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&k_full[i], 1);
        mbar_init(&k_empty[i], 1);
        mbar_init(&v_full[i], 1);
        mbar_init(&v_empty[i], 1);
        mbar_init(&s_full[i], 1);
        for (int c = 0; c < PG_PARTS; ++c) mbar_init(&p_full[i * PG_PARTS + c], 4);
        mbar_init(&o_done[i], 1);
      }
      mbar_init(v_tail, 1);
      mbar_fence_init();
      shared_failed = 0;
    }
    int whole = 0;                 // blocks
    const int U = paged_plan(p, own, whole);
    there = pg_find(p, own, blockIdx.x, U, it);
    if (lane == 0) {
      shared_there = there;
      if (there) shared_item = it;
      if (p.slots && blockIdx.x == 0) *p.cut = U == PG_WHOLE || !there ? 0 : whole;
      if (U != PG_WHOLE && there && it.piece == 0 && it.block < p.blocks) {
        p.where[2 * it.block] = make_int4(blockIdx.x, it.pieces, it.steps(p.tb), it.token);
        p.where[2 * it.block + 1] = make_int4(it.tokens, it.hk, 0, 0);
      }
    }
    if (there) {
      derive(it);
      if (lane == 0) {
        const int qtiles = alternate ? 1 : 2;
        mbar_expect_tx(q_full, qtiles * p.tq * p.G * HD * 2);
        for (int t = 0; t < qtiles; ++t)
#pragma unroll
          for (int c = 0; c < Cfg::CH; ++c)
            tma_load_3d(sQ + t * Cfg::TILE_BYTES + c * (PG_TILE * 128), &tmQ, q_full, c * 64, it.hk * p.G, it.token + t * p.tq);
        if (it.keys != it.len) p.seqs.bad();
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  } else if (threadIdx.x == 64) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  if (!shared_there) {
    if (warp == 1) tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    return;
  }
  const PgItem& item = shared_item;                // read where it is needed: the softmax warps have no registers to keep it in
  if (warp != 0) derive(item);
  // steps of each tile: one behind the other over its own keys (two tiles of rows), or every other (one)
  int cnt[2];
  cnt[0] = alternate ? (n_j + 1) >> 1 : max(0, min(item.j1, item.steps(p.tq)) - item.j0);
  cnt[1] = alternate ? n_j >> 1 : n_j;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PG_REGS_CTRL));
  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer: a lane has one box of a step
    auto page_of = [&](int j) {
      const int key = j * PG_TILE + lane * box;
      if (lane * box >= PG_TILE || j >= it.j1 || key >= it.keys) return p.seqs.pages;       // zeros
      const int page = p.seqs.table[(long long)it.b * p.seqs.ld + (key >> p.seqs.page_shift)];
      if (page >= 0 && page < p.seqs.pages) return page;
      p.seqs.bad();
      return p.seqs.pages;
    };
    auto boxes_to = [&](uint8_t* dst, const CUtensorMap* m, uint64_t* bar, int j, int page) {
      if (lane == 0) mbar_expect_tx(bar, Cfg::TILE_BYTES);
      __syncwarp();
      if (lane * box < PG_TILE) {
        const int y = (j * PG_TILE + lane * box) & ((1 << p.seqs.page_shift) - 1);
  #pragma unroll
        for (int c = 0; c < Cfg::CH; ++c)
          tma_load_4d(dst + c * (PG_TILE * 128) + lane * box * 128, m, bar, c * 64, y, it.hk, page);
      }
      __syncwarp();
    };
    int next = page_of(it.j0);
    for (int i = 0; i < n_j; ++i) {
      const int j = it.j0 + i, st = i & 1, page = next;
      const uint32_t ph = (i >> 1) & 1;
      next = page_of(j + 1);
      if (!mbar_wait_warp(&k_empty[st], ph ^ 1)) {
        if (lane == 0) fail(GF_ERR_WAIT_EMPTY);
        break;
      }
      boxes_to(sK + st * Cfg::TILE_BYTES, &tmK, &k_full[st], j, page);
      if (!mbar_wait_warp(&v_empty[st], ph ^ 1)) {
        if (lane == 0) fail(GF_ERR_WAIT_EMPTY);
        break;
      }
      boxes_to(sV + st * Cfg::TILE_BYTES, &tmV, clears && i == n_j - 1 ? v_tail : &v_full[st], j, page);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    const bool leader = elect_one();
    constexpr uint32_t idesc_qk = umma_idesc_bf16(PG_TILE, PG_TILE, 0, 0);
    constexpr uint32_t idesc_pv = umma_idesc_bf16(PG_TILE, HD, 0, 1);
    const uint64_t dq0 = umma_desc_sw128(smem_u32(sQ), 16, 1024);
    const uint64_t dk0 = umma_desc_sw128(smem_u32(sK), 16, 1024);
    const uint64_t dv0 = umma_desc_sw128(smem_u32(sV), PG_TILE * 128, 1024);
    constexpr uint64_t TILE_D = Cfg::TILE_BYTES >> 4;
    bool ok = mbar_wait_warp_tight(q_full, 0);
    if (!ok && leader) fail(GF_ERR_WAIT_FULL);
    const uint64_t second = alternate ? 0 : TILE_D;        // Q of tile 1
    // S_t = Q_t K(stage)^T, announced on s_full[t]
    auto issue_qk = [&](int t, int st) {
      const uint64_t qa = dq0 + (t ? second : 0), ka = dk0 + (st ? TILE_D : 0);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const uint64_t off = ((kk >> 2) * (PG_TILE * 128) + (kk & 3) * 32) >> 4;
        umma_bf16_ss_u(leader, tmem_base + Cfg::TM_S + t * 128, qa + off, ka + off, idesc_qk, kk > 0 ? 1u : 0u);
      }
      umma_commit_u(leader, &s_full[t]);
    };
    // O_t += P_t V(stage), n-th of the tile
    auto issue_pv = [&](int t, int st, int n) {
      const uint64_t va = dv0 + (st ? TILE_D : 0);
#pragma unroll
      for (int c = 0; c < PG_PARTS; ++c) {
        if (ok && !mbar_wait_warp_tight(&p_full[t * PG_PARTS + c], n & 1)) {
          if (leader) fail(GF_ERR_WAIT_SOFTMAX);
          ok = false;
        }
        if (ok) {
          tc_fence_after();
#pragma unroll
          for (int kk = c * (PG_TILE / 16 / PG_PARTS); kk < (c + 1) * (PG_TILE / 16 / PG_PARTS); ++kk)
            umma_bf16_ts_u(leader, tmem_base + Cfg::TM_O + t * 128, tmem_base + Cfg::TM_S + t * 128 + kk * 8,
                           va + ((kk * 2048) >> 4), idesc_pv, (n > 0 || kk > 0) ? 1u : 0u);
        }
      }
      if (ok && n == (t ? cnt[1] : cnt[0]) - 1) umma_commit_u(leader, &o_done[t]);
    };
    auto full = [&](uint64_t* bar, int i) {
      if (ok && !mbar_wait_warp_tight(&bar[i & 1], (i >> 1) & 1)) {
        if (leader) fail(GF_ERR_WAIT_FULL);
        ok = false;
      }
    };
    if (alternate) {
      // step i belongs to tile i % 2 and lies in stage i % 2
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i < n_j) full(k_full, i);
        if (ok && i < n_j) {
          tc_fence_after();
          issue_qk(i, i);
          umma_commit_u(leader, &k_empty[i]);
        }
      }
      for (int i = 0; i < n_j && ok; ++i) {
        const int t = i & 1;
        full(v_full, i);
        if (!ok) break;
        issue_pv(t, t, i >> 1);
        if (!ok) break;
        umma_commit_u(leader, &v_empty[t]);
        if (i + 2 < n_j) {
          full(k_full, i + 2);
          if (!ok) break;
          tc_fence_after();
          issue_qk(t, t);
          umma_commit_u(leader, &k_empty[t]);
        }
      }
    } else {
      if (n_j > 0) full(k_full, 0);
      if (ok && n_j > 0) {
        tc_fence_after();
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (cnt[t] > 0) issue_qk(t, 0);
        umma_commit_u(leader, &k_empty[0]);
      }
      for (int i = 0; i < n_j && ok; ++i) {
        full(v_full, i);
        if (i + 1 < n_j) full(k_full, i + 1);
        if (!ok) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (ok && i < cnt[t]) issue_pv(t, i & 1, i);
          if (ok && i + 1 < cnt[t]) issue_qk(t, (i + 1) & 1);
        }
        if (!ok) break;
        umma_commit_u(leader, &v_empty[i & 1]);
        if (i + 1 < n_j) umma_commit_u(leader, &k_empty[(i + 1) & 1]);
      }
    }
  } else if (warp == 2 && clears) {
    // ---------------------------------------------------------------- rows of the last V behind the sequence: zeros
    if (!mbar_wait_warp(v_tail, 0)) {
      if (lane == 0) fail(GF_ERR_WAIT_FULL);
    } else {
      const int st = (n_j - 1) & 1, end = (tail + box - 1) & ~(box - 1);       // what lies behind `end` came as zeros
      for (int c = 0; c < Cfg::CH; ++c) {
        uint4* rows = reinterpret_cast<uint4*>(sV + st * Cfg::TILE_BYTES + c * (PG_TILE * 128));
        for (int i = tail * 8 + lane; i < end * 8; i += 32) rows[i] = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[st]);
    }
  }
  } else {
    // ---------------------------------------------------------------- softmax warps: tile t = warp / 4 - 1
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PG_REGS_SOFTMAX));
    const int t = (warp >> 2) - 1;
    const int lane_grp = warp & 3;
    const int r = lane_grp * 32 + lane;
    const int tile_token = alternate ? 0 : t * p.tq;                   // first token of the tile in the block
    const int tile_rows = max(0, min(p.tq, item.tokens - tile_token)) * p.G;
    const int tok = tile_token + r / p.G, head = item.hk * p.G + r % p.G;
    const bool mine = r < tile_rows;                                   // the row is a token's
    const bool idle = lane_grp * 32 >= tile_rows;                      // no row of the warp is
    const int lim = mine ? min(item.pos + tok, item.keys - 1) : -1;        // last key that the row sees
    const int tile_lim = min(item.pos + tile_token, item.keys - 1);        // ... that all of them see
    const uint32_t tlane = (uint32_t)(lane_grp * 32) << 16;
    const uint32_t ts = tmem_base + Cfg::TM_S + t * 128 + tlane;
    const uint32_t to = tmem_base + Cfg::TM_O + t * 128 + tlane;
    const float sl2 = p.scale * 1.4426950408889634f;
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    const int my_n = t ? cnt[1] : cnt[0];
    for (int j = 0; j < my_n && ok; ++j) {
      if (!mbar_wait_warp_tight(&s_full[t], j & 1)) {
        fail(GF_ERR_WAIT_TMEM_FULL);
        ok = false;
        break;
      }
      if (idle) {
        if (lane == 0)
          for (int c = 0; c < PG_PARTS; ++c) mbar_arrive(&p_full[t * PG_PARTS + c]);
        continue;
      }
      tc_fence_after();
      const int kv0 = (item.j0 + (alternate ? 2 * j + t : j)) * PG_TILE;
      const bool need_mask = kv0 + PG_TILE - 1 > tile_lim;
      // ---- row maximum, 64 scores at a time (the exponential pass reads them from tensor memory again)
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        uint32_t sa[32], sb[32];
        tmem_ld32(ts + c2 * 64, sa);
        tmem_ld32(ts + c2 * 64 + 32, sb);
        tmem_ld_wait();
        if (need_mask) {
          const int last = lim - kv0 - c2 * 64;                          // last visible column here
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i > last) sa[i] = 0xff800000u;  // -inf
            if (32 + i > last) sb[i] = 0xff800000u;
          }
          tmem_st32(ts + c2 * 64, sa);
          tmem_st32(ts + c2 * 64 + 32, sb);
          tmem_st_wait();
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) mx4[e] = pg_max3(mx4[e], __uint_as_float(sa[i + e]), __uint_as_float(sb[i + e]));
        }
      }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      // ---- reference maximum: moved (and O, l rescaled) only when the row's maximum grew a lot. The commit behind s_full also covered
      // the last P V, so O is quiescent here.
      if (j == 0) {
        m_ref = mx;
      } else {
        const bool grow = (mx - m_ref) * sl2 > PG_RESCALE;
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? ex2_approx((m_ref - mx) * sl2) : 1.f;
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t rr[32];
            tmem_ld32(to + c * 32, rr);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) rr[i] = __float_as_uint(__uint_as_float(rr[i]) * alpha);
            tmem_st32(to + c * 32, rr);
          }
          l *= alpha;
          if (grow) m_ref = mx;
        }
      }
      const float mref_use = (m_ref == -INFINITY) ? 0.f : m_ref;  // row with no visible key yet
      const float mneg = -mref_use * sl2;
      const uint64_t sl2x = pk2f(sl2, sl2), mnegx = pk2f(mneg, mneg);
      uint64_t rsa = 0, rsb = 0;
      uint32_t sa[32], sb[32];
      auto chunk = [&](const uint32_t (&sv)[32], uint32_t dst) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const uint64_t x = f2_fma(pk2(sv[i], sv[i + 1]), sl2x, mnegx);
          const float p0 = ex2_approx(lo2(x)), p1 = ex2_approx(hi2(x));
          if (i & 2) rsa = f2_add(rsa, pk2f(p0, p1)); else rsb = f2_add(rsb, pk2f(p0, p1));
          pk[i >> 1] = pack_bf16x2(p0, p1);
        }
        tmem_st16(dst, pk);
      };
      tmem_ld32(ts, sa);
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        tmem_ld_wait();
        tmem_ld32(ts + c2 * 64 + 32, sb);
        chunk(sa, ts + c2 * 32);
        tmem_ld_wait();
        if (c2 == 0) tmem_ld32(ts + 64, sa);
        chunk(sb, ts + c2 * 32 + 16);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t * PG_PARTS + c2]);
      }
      const uint64_t rs = f2_add(rsa, rsb);
      l += lo2(rs) + hi2(rs);
    }
    // ---- end: all products into O have been done
    auto done = [&](int tile) {
      if (ok && (tile ? cnt[1] : cnt[0]) > 0 && !mbar_wait_warp_tight(&o_done[tile], 0)) {
        fail(GF_ERR_WAIT_TMEM_FULL);
        ok = false;
      }
    };
    done(t);
    if (alternate) {
      // both tiles have sums of the same rows: tile 1 leaves its own in shared memory, column by column
      float* sums = reinterpret_cast<float*>(sK);
      float* ml = reinterpret_cast<float*>(smem + Cfg::OFF_ML);
      done(0);
      if (t == 1 && !idle) {
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t rr[32];
          tmem_ld32(to + c * 32, rr);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) sums[(c * 32 + i) * PG_TILE + r] = my_n > 0 ? __uint_as_float(rr[i]) : 0.f;
        }
        ml[r] = m_ref;
        ml[PG_TILE + r] = l;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    if (ok && !idle && !(alternate && t == 1)) {
      tc_fence_after();
      float a0 = 1.f, a1 = 0.f;
      const float* sums = reinterpret_cast<const float*>(sK);
      if (alternate) {
        const float* ml = reinterpret_cast<const float*>(smem + Cfg::OFF_ML);
        const float m1 = ml[r], mm = fmaxf(m_ref, m1), use = mm == -INFINITY ? 0.f : mm;
        a0 = ex2_approx((m_ref - use) * sl2);
        a1 = ex2_approx((m1 - use) * sl2);
        l = l * a0 + ml[PG_TILE + r] * a1;
        m_ref = mm;
      }
      const bool whole = item.pieces == 1;
      const float inv = !whole ? 1.f : l > 0.f ? 1.f / l : 0.f;
      a0 *= inv;
      a1 *= inv;
      __nv_bfloat16* orow = p.out + (long long)(item.token + tok) * p.ldo + head * HD;
      const long long row = (long long)blockIdx.x * p.rows + (alternate ? r : t * PG_TILE + r);
      // left for the other kernel four columns of 32 rows at a time: a warp's rows lie next to each other
      float* prow = p.part + (row - lane) * HD + lane * 4;
      // rolled up: code that runs once is waited for
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t rr[32];
        tmem_ld32(to + c * 32, rr);
        tmem_ld_wait();
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          o[i] = my_n > 0 ? __uint_as_float(rr[i]) * a0 : 0.f;       // tensor memory that nothing wrote may hold anything
          if (alternate) o[i] += sums[(c * 32 + i) * PG_TILE + r] * a1;
        }
        if (!mine) continue;
        if (whole) {
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            uint4 u;
            uint32_t* pu = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
            for (int e = 0; e < 4; ++e) pu[e] = pack_bf16x2(o[q4 * 8 + e * 2], o[q4 * 8 + e * 2 + 1]);
            *reinterpret_cast<uint4*>(orow + c * 32 + q4 * 8) = u;
          }
        } else if (n_j > 0) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(prow + (c * 32 + i) * 32) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
      if (mine && !whole && n_j > 0) *reinterpret_cast<float2*>(p.part_ml + 2 * row) = make_float2(m_ref * sl2, l);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (shared_failed) error_drain_pause();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

constexpr int PG_COLS = 8, PG_AHEAD = 4;
// Adds up the pieces of blocks that were cut: a CTA has 8 columns of one block, a warp 32 of its rows, a lane one of them. Where a block's pieces are is
// left in memory by the CTA that has the first: most CTAs here begin when the first kernel's registers are free, at its end, so that what they do to
// find out would be waited for. Two or three pieces of many rows want warps on an SM, many pieces of few rows loads of a warp on
// their way together: the whole call, us, with 2 / 4 (64 registers) / 8 pieces at a time, 512 new tokens over 7681 keys, 2 pieces 72 / 72 to 75 / 76, 5 over
// 30000, 17 pieces 39.2 / 37.6 / 37.0, 16 over 2000, 16 pieces 14.2 / 12.5 / 12.3.
template <int HD>
__global__ void __launch_bounds__(256, 4) paged_join_kernel(const __grid_constant__ PagedAttn p) {
  constexpr int GROUPS = HD / PG_COLS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = (blockIdx.x % GROUPS) * PG_COLS;
  const int block = blockIdx.x / GROUPS, t = warp >> 2, r = (warp & 3) * 32 + lane;       // block, tile and row in it
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cut = *p.cut;
  const int4 a = p.where[2 * block], b = p.where[2 * block + 1];     // items of the block from a.x on, how many, its steps of keys, its first token; tokens, KV head
  const int pieces = a.y, steps = a.z, rows = max(0, min(p.tq, b.x - t * p.tq)) * p.G;         // rows of the tile
  const long long item = a.x;
  if (block >= cut || pieces == 1 || item + pieces > p.items || r >= rows) return;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + item * p.rows + t * PG_TILE + r;
  const float* part = p.part + (item * p.rows + t * PG_TILE + r - lane) * HD + col * 32 + lane * 4;
  // a piece that has no keys was not run; there are such where a block has fewer steps than pieces
  auto run = [&](int k) { return steps >= pieces || steps * k / pieces < steps * (k + 1) / pieces; };
  float m = -INFINITY, l = 0.f, o[PG_COLS];
#pragma unroll
  for (int e = 0; e < PG_COLS; ++e) o[e] = 0.f;
#pragma unroll 1
  for (int k0 = 0; k0 < pieces; k0 += PG_AHEAD) {           // what PG_AHEAD pieces left is on its way together
    float2 x[PG_AHEAD];
    float4 v[PG_AHEAD][PG_COLS / 4];
#pragma unroll
    for (int i = 0; i < PG_AHEAD; ++i) {
      const int k = k0 + i;
      x[i] = make_float2(-INFINITY, 0.f);
      if (k >= pieces || !run(k)) continue;
      x[i] = ml[(long long)k * p.rows];
#pragma unroll
      for (int e = 0; e < PG_COLS / 4; ++e) v[i][e] = *reinterpret_cast<const float4*>(part + (long long)k * p.rows * HD + e * 128);
    }
    float mm = m;
#pragma unroll
    for (int i = 0; i < PG_AHEAD; ++i) mm = fmaxf(mm, x[i].x);
    const float use = mm == -INFINITY ? 0.f : mm, old = ex2_approx(m - use);
    m = mm;
    l *= old;
#pragma unroll
    for (int e = 0; e < PG_COLS; ++e) o[e] *= old;
#pragma unroll
    for (int i = 0; i < PG_AHEAD; ++i) {
      if (x[i].y == 0.f) continue;                         // 0 times what may be anything
      const float w = ex2_approx(x[i].x - use);
      l += x[i].y * w;
#pragma unroll
      for (int e = 0; e < PG_COLS / 4; ++e) {
        o[4 * e] += v[i][e].x * w;
        o[4 * e + 1] += v[i][e].y * w;
        o[4 * e + 2] += v[i][e].z * w;
        o[4 * e + 3] += v[i][e].w * w;
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint4 u;
  u.x = pack_bf16x2(o[0] * inv, o[1] * inv); u.y = pack_bf16x2(o[2] * inv, o[3] * inv);
  u.z = pack_bf16x2(o[4] * inv, o[5] * inv); u.w = pack_bf16x2(o[6] * inv, o[7] * inv);
  *reinterpret_cast<uint4*>(p.out + (long long)(a.w + t * p.tq + r / p.G) * p.ldo + (b.y * p.G + r % p.G) * HD + col) = u;
}

static int pg_map(CUtensorMap* out, const void* base, int rank, const cuuint64_t* dims, const long long* strides, const cuuint32_t* box) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return GFH_TMAP;
  cuuint64_t bytes[3];
  for (int i = 0; i < rank - 1; ++i) bytes[i] = dims[i + 1] > 1 ? (cuuint64_t)strides[i] * 2 : dims[0] * 2;   // a stride that nothing goes by
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, bytes, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? GFH_OK : GFH_TMAP;
}

template <int HD>
static int launch_paged(PagedAttn& p, const void* q, long long ldq, const void* kp, const void* vp, const long long* strides, int items,
                        cudaStream_t st) {
  using Cfg = PgCfg<HD>;
  static gf::DeviceOnce configured;
  auto kern = paged_attn_kernel<HD>;
  if (configured.todo()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES) != cudaSuccess) return GFH_CUDA;
    configured.mark();
  }
  const PagedBatch& S = p.seqs;
  CUtensorMap tq, tk, tv;
  const cuuint64_t qdims[3] = {HD, (cuuint64_t)p.Hq, (cuuint64_t)S.T};
  const long long qstrides[2] = {HD, ldq};
  const cuuint32_t qbox[3] = {64, (cuuint32_t)p.G, (cuuint32_t)p.tq};
  const int page = 1 << S.page_shift;
  const cuuint64_t dims[4] = {HD, (cuuint64_t)page, (cuuint64_t)p.Hkv, (cuuint64_t)S.pages};
  const cuuint32_t box[4] = {64, (cuuint32_t)(page < PG_TILE ? page : PG_TILE), 1, 1};
  const long long ks[3] = {strides[1], strides[2], strides[0]}, vs[3] = {strides[4], strides[5], strides[3]};
  int rc = pg_map(&tq, q, 3, qdims, qstrides, qbox);
  if (!rc) rc = pg_map(&tk, kp, 4, dims, ks, box);
  if (!rc) rc = pg_map(&tv, vp, 4, dims, vs, box);
  if (rc) return rc;
  kern<<<items, PG_THREADS, Cfg::SMEM_BYTES, st>>>(tq, tk, tv, p);
  return cudaGetLastError() == cudaSuccess ? GFH_OK : GFH_CUDA;
}

template <int HD>
static int launch_join(const PagedAttn& p, cudaStream_t st) {
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.blocks * (HD / PG_COLS)));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, paged_join_kernel<HD>, p) != cudaSuccess) return GFH_CUDA;
  note_extra_launches(1);
  return GFH_OK;
}

// Items of a call at most, rows of one that are tokens' at most, and whether blocks may be cut: what decides the grid and the workspace. They are
// not where there are two for every SM, nor where no sequence has more than four steps of keys (those four take 6 us, as long as one and the
// second kernel), nor beside the decode kernel (`ones`) when that has more to do: a step of keys of all KV heads of all sequences takes it as long
// as a step takes here, 2 us, with 1.25 of them for every SM. 31 sequences of up to 2048 keys with one token and one with 4 / 30 / 481, 32 / 8 heads, cut / not: 60
// / 46, 62 / 47, 56 / 56 us.
//
// Over those few steps blocks have one tile's rows where as many run at one time, half of the SMs' beside the decode kernel: each takes half as long. us, two
// tiles / one: 61 tokens over 414 keys, 32 / 8 heads of 128 16.7 / 12.0, a prompt of 469, 16 / 1 heads 16.4 / 12.7, of 200, 32 / 8 heads 12.6 / 10.1.
//
// `keys` is what the page table has room for: the host knows no lengths. A table that is wider than its sequences (a captured step's) gives up the
// last two rules: a prompt of 200, 32 / 8 heads, its own table / one for 4096 keys 16.4 / 22.5, four of them 20.5 / 26.6 (L2 flushed). Every sequence counts
// as if it had part of a block, those of one token too, which have none beside the decode kernel: the CTAs without a block leave.
struct PgCall {
  int items, rows, slots, blocks, tb;
  long long ws;
};
static bool pg_call(PgCall& c, int B, int T, bool one_each, bool ones, long long keys, int Hq, int Hkv, int D, int sms) {
  const int tq = PG_TILE / (Hq / Hkv);
  auto blocks_of = [&](int tb) { return one_each ? (long long)B : min((long long)T, ((long long)T + (long long)B * (tb - 1)) / tb); };
  c.tb = keys <= 4 * PG_TILE && blocks_of(tq) * Hkv <= (ones ? sms / 2 : sms) ? tq : 2 * tq;
  const long long items = blocks_of(c.tb) * Hkv;
  if (items > 0x7fffffffll) return false;
  const bool beside = ones && 4ll * B * Hkv >= 5ll * sms;
  c.slots = items < 2 * sms && keys > 4 * PG_TILE && !beside ? sms : 0;
  c.blocks = (int)items;
  c.items = c.slots ? 2 * sms : (int)items;
  c.rows = one_each || T <= tq ? PG_TILE : 2 * PG_TILE;       // blocks of one tile, or of two
  c.ws = c.slots ? 256 + 32ll * c.blocks + 4ll * c.items * c.rows * (D + 2) : 0;
  return true;
}

}  // namespace gf

using namespace gf;

static bool paged_sizes(int B, int T, int Hq, int Hkv, int D) {
  return B > 0 && T > 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= PG_TILE && (D == 64 || D == 128) && Hkv <= 65535;
}

// Bytes of workspace of a call, -1 for sizes that are not taken. one_each: there is no `cu`; ones: as for gf_paged_attn; keys: width * page.
GF_API long long gf_paged_attn_workspace(int B, int T, int one_each, int ones, long long keys, int Hq, int Hkv, int D) {
  gf::bind();
  PgCall c;
  if (!paged_sizes(B, T, Hq, Hkv, D) || !pg_call(c, B, T, one_each != 0, ones != 0, keys, Hq, Hkv, D, sm_count())) return -1;
  return c.ws;
}

// x [T, Hq, D] and y alike; ws: as many bytes as gf_paged_attn_workspace says, on a 16-byte boundary. scale > 0. ones != 0: sequences of one new
// token go to the decode kernel, with that many splits and its scratch (see gf_paged_attn_one), while this one's CTAs run out. Each kernel is
// launched while the one in front of it runs, and none ends before that one has.
GF_API int gf_paged_attn(const PagedCall* c, float scale, void* ws, long long ws_bytes, int ones, float* ones_scratch, void* stream) {
  PagedAttn p{};
  if (!c || !paged_batch(p.seqs, *c) || c->pages == 0 || c->H > 0x7fffffff || c->Hk > 65535) return GFH_BAD_ARG;
  const int B = p.seqs.B, T = p.seqs.T, Hq = (int)c->H, Hkv = (int)c->Hk, D = (int)c->D;
  if (!paged_sizes(B, T, Hq, Hkv, D) || !(scale > 0.f) || (reinterpret_cast<uintptr_t>(ws) & 15)) return GFH_BAD_ARG;
  if (ones && !attn_paged_one_ok(*c, ones, ones_scratch)) return GFH_BAD_ARG;
  gf::bind();
  PgCall n;
  if (!pg_call(n, B, T, !p.seqs.cu, ones != 0, p.seqs.capacity(), Hq, Hkv, D, sm_count())) return GFH_TOO_LARGE;
  if (ws_bytes < n.ws || (n.ws && !ws)) return GFH_BAD_ARG;
  gf::enter();
  p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.tq = PG_TILE / p.G; p.tb = n.tb;
  p.slots = n.slots; p.scale = scale; p.rows = n.rows; p.items = n.items; p.blocks = n.blocks;
  p.skip_ones = ones != 0;
  p.out = (__nv_bfloat16*)c->y; p.ldo = c->ldy;
  if (n.slots) {
    p.cut = (int*)ws;
    p.where = (int4*)((char*)ws + 256);
    p.part = (float*)((char*)ws + 256 + 32ll * n.blocks);
    p.part_ml = p.part + (long long)n.items * n.rows * D;
  }
  cudaStream_t st = (cudaStream_t)stream;
  int rc = D == 128 ? launch_paged<128>(p, c->x, c->ldx, c->kpages, c->vpages, c->strides, n.items, st)
                    : launch_paged<64>(p, c->x, c->ldx, c->kpages, c->vpages, c->strides, n.items, st);
  if (!rc && ones) {
    note_extra_launches(1);
    rc = attn_paged_one(*c, scale, ones, ones_scratch, 1, st);
  }
  if (!rc && n.slots) rc = D == 128 ? launch_join<128>(p, st) : launch_join<64>(p, st);
  return rc;
}
