// tree_attention_tc.cuh - tcgen05 kernel of the tree attention (bf16, head_dim 64 or 128);
// included by tree_attention.cu.
//
// A segment is one (sequence, key/value head, block of query rows): its keys are the cached
// tiles of 128 positions, the last of them partly filled, and the drafted tokens, which go into
// what is left of that last tile if they are few, else into a tile of their own. The
// lengths are known on the GPU only, so the blocks share the work out there: all segments'
// tiles, and kExtra more for what a segment costs besides, form one row, of which block c takes
// [c X, (c + 1) X). A segment that is cut leaves (max, sum, O) per piece in the workspace, and
// tree_join_kernel joins the pieces in order. Cuts near a segment's end move there, and short
// segments are not cut.
//
// Query rows of a tile: `tt` tokens times the G query heads of the key/value head (tt G <=
// 128), fetched by one TMA box per 64 columns, so row r is token r / G, head r % G.
//   warps 0-3, 4-7  softmax groups 0 and 1, one thread per row: scores from TMEM, mask, running
//                   maximum and sum, exponentials rounded to bf16 back into TMEM over the scores
//   warps 8, 10     TMA: queries and keys, values, each through a ring of tiles; the lanes look
//                   up the pages, a box of rows of one page each
//   warp 11         mends tiles that hold more or less than cached rows: drafted tokens put behind
//                   the last cached row, rows past the end cleared
//   warp 9          tcgen05.mma, both products: S = Q K^T, O += P V (P from TMEM)
//   TMEM            S / P of group 0, 1 [0, 128), [128, 256); O of group 0, 1 after them
// NQ = 1 (rows fit one tile): the groups take the tiles of keys in turn, each with a maximum,
// sum and O of its own, joined at the end of the segment's piece. NQ = 2: each group has its own
// tile of rows, and both meet the same keys, which so cross shared memory's boundary once for
// 256 rows. P of a tile is handed over in two halves of 64 keys, so that the first half's product
// with V runs while the second half is exponentiated.
//
// The running maximum may lag behind by up to 2^8: O is rescaled only when a row's maximum
// grows by more than that. P is then up to 2^8 instead of 1, with the same relative rounding.
//
// Measured, GPU time with the join (bf16; 6.5 TB/s is what a copy of memory reaches):
//   1 token, 203 positions, 32 heads over 8 of 128              9.6 us
//   16 tokens, 4 sequences of up to 4096, 32 heads of 128      42 us (158 MB: 24 us by bytes)
//   1 token, 65536 positions, 32 heads over 8 of 128           58.5 us (268 MB: 41 us by bytes)
//   1 token, 64 sequences of about 700, 32 heads over 8       64.6 us (183 MB: 28 us by bytes)
//   64 tokens, 2 sequences of up to 65536, 32 heads over 8    126 us (427 MB, 109 GFLOP: 67 us either way)
// What bounds them: the first is one chain of dependent steps, lengths -> table -> tile ->
// softmax -> product -> store. In the second a block has some 15 tiles; starting (6 us), the
// pieces' beginnings and ends (about four tiles' time each) and the join (5 us) are not
// overlapped by enough of them. In the last, a tile's chain is what is left: scores -> exponentials
// -> product with V -> the next scores into the same columns; without the exponentials it would
// take 92 us, with one eighth of Q K^T 108 us, so neither unit bounds it alone.
//
// Against the kernel of tree_attention.cu on the same bf16 calls: 1 token, 1000 positions 16.0 and
// 17.6 us; 64 sequences of about 700 64 and 128 us; 4 of up to 4096 42 and 105 us; 64 tokens, 65536
// positions 126 and 3250 us. NQ = 2 against NQ = 1 with the keys read by two blocks, 256 rows: up
// to 65536 positions 126 and 149 us, about 5000 79 and 78 us, 240 rows of 64 over up to 5809
// positions 19.5 and 18.5 us: it gains where rows are long and costs little where they are not.
#pragma once

namespace {

using namespace sm100;

__device__ unsigned int g_tree_dev_error = 0;

constexpr int kTile = 128;
constexpr int kTcThreads = 384;
constexpr int kKeyWarp = 8, kMmaWarp = 9, kValueWarp = 10, kMendWarp = 11;
constexpr int kFewDrafts = 16;   // so many drafted tokens can share the last cached tile
constexpr int kWhole = 4;        // segments of up to so many tiles are not cut: a cut costs kExtra
constexpr int kMaxPieces = 192;  // of one segment: at most one for each block and one more
// Least share of a block and what a segment's beginning and end count for, in tiles. With 5 and 3
// instead of 2 and 4: 4 sequences of up to 5809 positions 24 us instead of 19, one of 1000 18 instead of
// 14; with nothing counted for the ends 4 sequences of 4096 56 us instead of 41.
constexpr int kLeast = 2, kExtra = 4;
// Sequences of up to so many cached positions have P in two bf16 parts, P V in two products: a
// row that sees few keys does not average the roundings of P out (one part: up to 2^-8 of a
// weight). On short rows the second product costs little (64 sequences of about 700: 64.8 us, with
// one part 61.5), on long ones it would cost more (2 of up to 65536: 140 us instead of 126).
constexpr int kFine = 1024;
constexpr float kLag = 8.f;      // log2 of how far the running maximum may lag

struct TcArgs {
  const int *tables, *lens, *parents;
  const bf16 *k_new, *v_new;
  int64_t n_b, n_t, n_h;  // its strides
  bf16* out;
  int4* ws_start;  // [block]: where it starts, for the join: sequence, head and row block, tile
  float* ws_ml;    // [slot][NQ][2][128]
  float4* ws_o;    // [slot][NQ][d / 4][128]
  int batch, tokens, heads, kv_heads, group, pages, page, max_pages;
  int capacity;    // positions that a row of the tables holds
  int tt;          // tokens per query tile
  int row_blocks;  // blocks of NQ query tiles
  int box;         // rows of a page fetched by one TMA box
  int log_bpt;     // log2 of the boxes of a tile
  int boxes_per_page, log_bpp;  // log_bpp < 0: no power of two
  unsigned long long bpp_magic;  // ceil(2^36 / boxes_per_page)
  float scale_log2;
};

__device__ __forceinline__ int tree_len(const TcArgs& a, int b) {
  return min(max(a.lens[b], 0), a.capacity);
}
// Whether the drafted tokens share the last cached tile of a sequence of this length.
__device__ __forceinline__ bool tree_shares(const TcArgs& a, int len) {
  const int rest = len % kTile;
  return rest != 0 && a.tokens <= kFewDrafts && rest + a.tokens <= kTile;
}
__device__ __forceinline__ int tree_tiles(const TcArgs& a, int b) {
  const int len = tree_len(a, b);
  return (len + kTile - 1) / kTile + (tree_shares(a, len) ? 0 : 1);
}

// Where a cut goes that falls `off` into a segment of n tiles (and kExtra before them): to a
// tile, or to 0 or n when that is near or the segment is short.
__device__ __forceinline__ int cut_at(int off, int n, int share) {
  off = max(off - kExtra, 0);
  if (n <= kWhole) return 2 * off >= n ? n : 0;
  const int near = min(max(share / 4, 1), 4);
  if (off < near) return 0;
  if (n - off < near) return n;
  return off;
}

// One block's walk over its pieces of segments: the place it has come to and its end.
struct Walk {
  int b, hm, t, tiles, end_b, end_hm, end_t;
};
struct Piece {
  int b, kvh, mb, t0, n, tiles, len;
  bool shares;  // the drafted tokens are in the last cached tile
};

template <int D, int NQ>
struct TreeSmem {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kRingK = D == 128 ? 3 : 5;
  static constexpr int kRingV = (D == 128 ? 4 : 6) - NQ;
  uint8_t q[NQ][kTileBytes];
  uint8_t k[kRingK][kTileBytes];
  uint8_t v[kRingV][kTileBytes];
  uint64_t q_full, q_empty;
  uint64_t k_full[kRingK], k_empty[kRingK], k_land[kRingK];  // land: the copies of a tile that is mended before it is full
  uint64_t v_full[kRingV], v_empty[kRingV], v_land[kRingV];
  uint64_t s_full[2], p_full[2][2], o_done[2][2];  // [group][half of the tile]
  uint64_t o_free[2];
  uint64_t x_full;
  uint64_t mma_done;
  float xm[2][kTile], xl[2][kTile];  // NQ = 1: the groups' maxima and sums
  // Drafted tokens whose v holds infinities or NaN, of the last pieces: products wait for the
  // end of the piece before, so the mending warp is at most kRingV pieces ahead of a reader.
  uint32_t bad[8][4];
  uint32_t tmem_base;
  int abort;
};
template <int D, int NQ>
constexpr bool tiles_aligned() {
  using S = TreeSmem<D, NQ>;
  return offsetof(S, k) % 1024 == 0 && offsetof(S, v) % 1024 == 0;
}
static_assert(tiles_aligned<128, 1>() && tiles_aligned<128, 2>() && tiles_aligned<64, 1>() && tiles_aligned<64, 2>(),
              "swizzled tiles are 1024-byte aligned");

__device__ __forceinline__ bool tree_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  int ok = 1;
  if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, abort, &g_tree_dev_error, code) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

__device__ __forceinline__ bool next_piece(const TcArgs& a, Walk& w, Piece& p) {
  const bool last = w.b == w.end_b && w.hm == w.end_hm;
  if (last ? w.t >= w.end_t : w.b >= w.end_b && (w.b > w.end_b || w.hm > w.end_hm)) return false;
  p.b = w.b;
  p.kvh = a.row_blocks == 1 ? w.hm : w.hm / a.row_blocks;
  p.mb = w.hm - p.kvh * a.row_blocks;
  p.t0 = w.t;
  p.tiles = w.tiles;
  p.n = (last ? w.end_t : w.tiles) - w.t;
  p.len = tree_len(a, w.b);
  p.shares = tree_shares(a, p.len);
  w.t = 0;
  if (last) {
    w.t = w.end_t;
  } else if (++w.hm == a.kv_heads * a.row_blocks) {
    w.hm = 0;
    if (++w.b < a.batch) w.tiles = tree_tiles(a, w.b);
  }
  return true;
}

// This block's walk, computed by each warp for itself (a lane takes consecutive sequences).
__device__ __forceinline__ Walk tree_plan(const TcArgs& a) {
  const int lane = threadIdx.x & 31, hms = a.kv_heads * a.row_blocks;
  const int per = (a.batch + 31) >> 5, b0 = min(lane * per, a.batch), b1 = min(b0 + per, a.batch);
  int sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int t = tree_tiles(a, b) + kExtra;
    sum += t;
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  const int total = __shfl_sync(0xffffffffu, inc, 31) * hms;
  const int share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, kLeast);
  // Where this block's range begins (even lanes) and ends (odd lanes): the lane whose sequences
  // hold the place, the sequence among them, the segment of the sequence, the tile of the segment.
  const int from = (int)blockIdx.x * share, at = from + (lane & 1) * share;
  const unsigned beyond0 = __ballot_sync(0xffffffffu, inc * hms > from);
  const unsigned beyond1 = __ballot_sync(0xffffffffu, inc * hms > from + share);
  const unsigned beyond = (lane & 1) ? beyond1 : beyond0;
  const int src = beyond ? __ffs(beyond) - 1 : 0;
  int lo = __shfl_sync(0xffffffffu, inc - sum, src) * hms;
  int b = a.batch, hm = 0, t = 0, n = 0;
  if (beyond) {
    for (b = src * per;; ++b) {
      n = tree_tiles(a, b);
      if (at < lo + (n + kExtra) * hms) break;
      lo += (n + kExtra) * hms;
    }
    hm = (at - lo) / (n + kExtra);
    t = cut_at(at - lo - hm * (n + kExtra), n, share);
    if (t == n) {
      t = 0;
      if (++hm == hms) {
        hm = 0;
        if (++b < a.batch) n = tree_tiles(a, b);
      }
    }
  }
  Walk w;
  w.b = __shfl_sync(0xffffffffu, b, 0);
  w.hm = __shfl_sync(0xffffffffu, hm, 0);
  w.t = __shfl_sync(0xffffffffu, t, 0);
  w.tiles = __shfl_sync(0xffffffffu, n, 0);
  w.end_b = __shfl_sync(0xffffffffu, b, 1);
  w.end_hm = __shfl_sync(0xffffffffu, hm, 1);
  w.end_t = __shfl_sync(0xffffffffu, t, 1);
  return w;
}

template <int D, int NQ>
__global__ void __launch_bounds__(kTcThreads, 1)
tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kn,
                         const __grid_constant__ CUtensorMap map_vn, const __grid_constant__ CUtensorMap map_kc,
                         const __grid_constant__ CUtensorMap map_vc, const __grid_constant__ TcArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (smem_u32(smem_raw) & 1023u) {  // the swizzled tiles need a 1024-byte-aligned base
    if (threadIdx.x == 0) atomicCAS(&g_tree_dev_error, 0u, 40u);
    return;
  }
  pdl_launch_dependents();
  using Smem = TreeSmem<D, NQ>;
  Smem& s = *reinterpret_cast<Smem*>(smem_raw);
  constexpr int kRingK = Smem::kRingK, kRingV = Smem::kRingV;
  constexpr uint32_t kTileBytes = Smem::kTileBytes;
  constexpr uint32_t kTmemCols = 512;
  constexpr uint32_t kOCol = 2 * kTile;  // O of group g at kOCol + g * D
  constexpr uint32_t kIdescS = idesc_bf16_f32(kTile, kTile, false, false);
  constexpr uint32_t kIdescPV = idesc_bf16_f32(kTile, D, false, true);
  constexpr int kSub = D / 64;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&s.q_full, 1);
    mbar_init(&s.q_empty, 1);
    for (int i = 0; i < kRingK; ++i) {
      mbar_init(&s.k_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
      mbar_init(&s.k_land[i], 1);
    }
    for (int i = 0; i < kRingV; ++i) {
      mbar_init(&s.v_full[i], 1);
      mbar_init(&s.v_empty[i], 1);
      mbar_init(&s.v_land[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&s.p_full[i][h], kTile);
        mbar_init(&s.o_done[i][h], 1);
      }
      mbar_init(&s.o_free[i], NQ == 1 ? 2 * kTile : kTile);
    }
    mbar_init(&s.x_full, 2 * kTile);
    mbar_init(&s.mma_done, 1);
    s.abort = 0;
    fence_barrier_init();
  }
  if (warp == kKeyWarp && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_kc);
    tma_prefetch_desc(&map_kn);
  }
  if (warp == kValueWarp && lane == 0) {
    tma_prefetch_desc(&map_vc);
    tma_prefetch_desc(&map_vn);
  }
  if (warp == kMmaWarp) tmem_alloc(&s.tmem_base, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  pdl_wait();
  Walk w = tree_plan(a);
  if (a.ws_start && threadIdx.x == 0) a.ws_start[blockIdx.x] = make_int4(w.b, w.hm, w.t, 0);

  if (warp == kKeyWarp || warp == kValueWarp) {
    // ------------------------------------------------ TMA
    const bool keys = warp == kKeyWarp;
    const CUtensorMap* const cached = keys ? &map_kc : &map_vc;
    const CUtensorMap* const drafted = keys ? &map_kn : &map_vn;
    uint8_t* const ring = keys ? s.k[0] : s.v[0];
    uint64_t* const full = keys ? s.k_full : s.v_full;
    uint64_t* const empty = keys ? s.k_empty : s.v_empty;
    uint64_t* const land = keys ? s.k_land : s.v_land;
    const uint32_t depth = keys ? kRingK : kRingV;
    const int per_tile = 1 << a.log_bpt;
    uint32_t st = 0, par = 0, uc = 0;
    uint32_t used = 0u, landed = 0u, land_par = 0u;  // per ring place: loaded, last load to be mended, parity of `land`
    bool ok = true;
    Piece p = {};
    // page and first row in it of a box of the piece's sequence
    auto look_up = [&](int box, int& page, int& slot) {
      page = slot = 0;
      if (box * a.box < p.len) {
        const int pi = a.log_bpp >= 0 ? box >> a.log_bpp : (int)(((uint32_t)box * a.bpp_magic) >> 36);
        slot = (box - pi * a.boxes_per_page) * a.box;
        page = a.tables[(int64_t)p.b * a.max_pages + pi];
        if ((uint32_t)page >= (uint32_t)a.pages) page = a.pages;  // outside: read as zeros
      }
    };
    while (ok && next_piece(a, w, p)) {
      // 32 boxes in a row, one to a lane, and the 32 after them
      int first = p.t0 * per_tile, page, slot, next_page, next_slot;
      look_up(first + lane, page, slot);
      if (keys) {
        if (!tree_wait(&s.q_empty, (uc & 1u) ^ 1u, &s.abort, 10)) { ok = false; break; }
        if (lane == 0) {
          mbar_arrive_expect_tx(&s.q_full, (uint32_t)(NQ * D * 2 * a.tt * a.group));
#pragma unroll
          for (int i = 0; i < NQ * kSub; ++i)
            tma_load_4d(s.q[i / kSub] + (i % kSub) * (kTile * 128), &map_q, &s.q_full, (i % kSub) * 64,
                        p.kvh * a.group, (p.mb * NQ + i / kSub) * a.tt, p.b);
        }
        __syncwarp();
      }
      ++uc;
      look_up(first + 32 + lane, next_page, next_slot);
      for (int t = p.t0; t < p.t0 + p.n; ++t) {
        const bool old = t * kTile < p.len;
        const int boxes = old ? (min(kTile, p.len - t * kTile) + a.box - 1) / a.box : 0;
        const int at = t * per_tile - first;
        if (!tree_wait(&empty[st], par ^ 1u, &s.abort, 11)) { ok = false; break; }
        const bool mend = keys ? p.shares && t == p.tiles - 1 : (t + 1) * kTile > p.len;
        uint64_t* const bar = mend ? &land[st] : &full[st];
        used |= 1u << st;
        landed = mend ? landed | 1u << st : landed & ~(1u << st);
        land_par ^= mend ? 1u << st : 0u;
        if (lane == 0) mbar_arrive_expect_tx(bar, old ? (uint32_t)(boxes * a.box * D * 2) : kTileBytes);
        uint8_t* const to = ring + st * kTileBytes;
        if (old) {
          for (int i = 0; i < boxes; ++i) {
            const int pg = __shfl_sync(0xffffffffu, page, at + i), sl = __shfl_sync(0xffffffffu, slot, at + i);
            if (lane == 0) {
#pragma unroll
              for (int c = 0; c < kSub; ++c)
                tma_load_4d(to + c * (kTile * 128) + i * a.box * 128, cached, bar, c * 64, sl, p.kvh, pg);
            }
          }
        } else if (lane == 0) {
#pragma unroll
          for (int c = 0; c < kSub; ++c)
            tma_load_4d(to + c * (kTile * 128), drafted, bar, c * 64, 0, p.kvh, p.b);
        }
        __syncwarp();
        if (at + per_tile == 32) {
          first += 32;
          page = next_page;
          slot = next_slot;
          look_up(first + 32 + lane, next_page, next_slot);
        }
        if (++st == depth) { st = 0; par ^= 1u; }
      }
    }
    if (!ok && lane == 0) {  // let issued copies land before shared memory is released
      const uint64_t begin = globaltimer();
      if (keys && uc > 0)
        while (!mbar_try_wait(&s.q_full, (uc - 1) & 1u) && globaltimer() - begin < kWaitTimeoutNs) {}
      for (uint32_t i = 0; i < depth; ++i) {  // the last load of each place: this round's below st, the last round's from st on
        if (!((used >> i) & 1u)) continue;
        uint64_t* const bar = (landed >> i) & 1u ? &land[i] : &full[i];
        const uint32_t phase = (landed >> i) & 1u ? ((land_par >> i) & 1u) ^ 1u : i < st ? par : par ^ 1u;
        while (!mbar_try_wait(bar, phase) && globaltimer() - begin < kWaitTimeoutNs) {}
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------ MMA
    if (elect_one()) {
      uint32_t uc = 0, gt = 0;
      uint32_t kt = 0, k_par = 0, vt = 0, v_par = 0;  // the rings' next places
      bool ok = true;
      Piece p = {};
      constexpr uint32_t kStep = kTileBytes >> 4;  // from one place of a ring to the next, in a descriptor
      const uint64_t q_desc = smem_desc_sw128(smem_u32(s.q[0]), 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(smem_u32(s.k[0]), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_u32(s.v[0]), kTile * 128, 1024);
      auto wait_k = [&]() {
        const bool y = mbar_wait(&s.k_full[kt], k_par, &s.abort, &g_tree_dev_error, 21);
        tc_fence_after();
        return y;
      };
      auto free_k = [&]() {
        mma_commit(&s.k_empty[kt]);
        if (++kt == kRingK) { kt = 0; k_par ^= 1u; }
      };
      auto free_v = [&]() {
        mma_commit(&s.v_empty[vt]);
        if (++vt == kRingV) { vt = 0; v_par ^= 1u; }
      };
      auto issue_s = [&](int g, int qi) {  // scores of group g: Q tile qi, the next key tile
        const uint64_t qd = q_desc + (uint32_t)qi * kStep, kd = k_desc + kt * kStep;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (uint32_t)(((kk >> 2) * (kTile * 128) + (kk & 3) * 32) >> 4);
          mma_bf16_ss(tmem + (uint32_t)(g * kTile), qd + off, kd + off, kIdescS, kk > 0 ? 1u : 0u);
        }
        mma_commit(&s.s_full[g]);
      };
      // O of group g (+)= P V over half h of the next value tile: the exponentials of 32 keys
      // take 16 of the 32 columns that their scores had, their second parts the other 16.
      auto issue_pv = [&](int g, int h, bool add, bool two) {
        const uint64_t vd = v_desc + vt * kStep + (uint32_t)(h * (kTile / 2 * 128) >> 4);
        const uint32_t o = tmem + kOCol + (uint32_t)(g * D), pc = tmem + (uint32_t)(g * kTile + h * (kTile / 2));
        if (two) {
#pragma unroll
          for (int kk = 0; kk < kTile / 32; ++kk)
            mma_bf16_ts(o, pc + (uint32_t)((kk >> 1) * 32 + 16 + (kk & 1) * 8), vd + (uint32_t)(kk * 128), kIdescPV,
                        (add || kk > 0) ? 1u : 0u);
          add = true;
        }
#pragma unroll
        for (int kk = 0; kk < kTile / 32; ++kk)
          mma_bf16_ts(o, pc + (uint32_t)((kk >> 1) * 32 + (kk & 1) * 8), vd + (uint32_t)(kk * 128), kIdescPV,
                      (add || kk > 0) ? 1u : 0u);
        mma_commit(&s.o_done[g][h]);
      };
      while (ok && next_piece(a, w, p)) {
        const int n = p.n;
        const bool two = p.len <= kFine;
        if (!mbar_wait(&s.q_full, uc & 1u, &s.abort, &g_tree_dev_error, 20)) { ok = false; break; }
        tc_fence_after();
        // t = -2 .. n - 1 (NQ = 1), -1 .. n - 1 (NQ = 2): P V of tile t, and the scores of the tile
        // whose place that frees
        constexpr int kAhead = NQ == 1 ? 2 : 1;
#pragma unroll 1
        for (int t = -kAhead; ok && t < n; ++t) {
          const bool more = t + kAhead < n;
          if (t >= 0 && !(ok = mbar_wait(&s.v_full[vt], v_par, &s.abort, &g_tree_dev_error, 22))) break;
#pragma unroll 1
          for (int i = 0; i < NQ; ++i) {
            const uint32_t G = gt + (uint32_t)t;
            const int g = NQ == 1 ? (int)(G & 1u) : i;
            const uint32_t use = NQ == 1 ? G >> 1 : G;
            if (t == 0 &&
                !(ok = mbar_wait(&s.o_free[i], (uc & 1u) ^ 1u, &s.abort, &g_tree_dev_error, 23)))
              break;
            for (int h = 0; t >= 0 && h < 2; ++h) {
              if (!(ok = mbar_wait(&s.p_full[g][h], use & 1u, &s.abort, &g_tree_dev_error, 24))) break;
              tc_fence_after();
              issue_pv(g, h, t >= kAhead || h > 0, two);
              if (NQ == 2 && t == 0 && i == 0 && h == 0) {
                // The second group starts half a tile behind the first, and stays there: the groups
                // take turns at the special function unit and the tensor core.
                issue_s(1, 1);
                free_k();
                if (n == 1) mma_commit(&s.q_empty);
              }
            }
            if (!ok) break;
            if (more && !(NQ == 2 && t < 0 && i == 1)) {
              if (i == 0 && !(ok = wait_k())) break;
              issue_s(g, NQ == 1 ? 0 : i);
            }
          }
          if (!ok) break;
          if (t >= 0) free_v();
          if (more && !(NQ == 2 && t < 0)) {
            free_k();
            if (t + kAhead == n - 1) mma_commit(&s.q_empty);
          }
        }
        if (!ok) break;
        gt += (uint32_t)n;
        ++uc;
      }
      // Every MMA issued by this thread has completed once mma_done flips.
      mma_commit(&s.mma_done);
      const uint64_t begin = globaltimer();
      while (!mbar_try_wait(&s.mma_done, 0) && globaltimer() - begin < kWaitTimeoutNs) {}
    }
    __syncwarp();
  } else if (warp == kMendWarp) {
    // ------------------------------------------------ tiles that are not 128 cached rows
    uint32_t gt = 0, uc = 0, k_par = 0u, v_par = 0u;  // per ring place: parity of `land`
    bool ok = true;
    Piece p;
    auto chunk = [&](uint8_t* tile, int row, int c) {  // 16 bytes of a row, where the swizzle puts them
      return reinterpret_cast<uint4*>(tile + (c / 8) * (kTile * 128) + row * 128 + ((c ^ row) & 7) * 16);
    };
    // An exponent of all ones among the 8 values: its half's top bit comes out set.
    auto not_finite = [](const uint4& y) {
      return (((y.x & 0x7f807f80u) + 0x00800080u) | ((y.y & 0x7f807f80u) + 0x00800080u) |
              ((y.z & 0x7f807f80u) + 0x00800080u) | ((y.w & 0x7f807f80u) + 0x00800080u)) & 0x80008000u;
    };
    auto clear_not_finite = [](uint32_t& x) {
      const uint32_t hit = ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
      if (hit & 0x8000u) x &= 0xffff0000u;
      if (hit & 0x80000000u) x &= 0x0000ffffu;
    };
    while (ok && next_piece(a, w, p)) {
      const int* const parents = a.parents ? a.parents + (int64_t)p.b * a.tokens : nullptr;
      for (int tile = max(p.t0, p.len / kTile); tile < p.t0 + p.n; ++tile) {  // the last one or two of the segment
        const uint32_t G = gt + (uint32_t)(tile - p.t0);
        const int rest = p.len - tile * kTile;  // cached rows; none: the drafted tokens' own tile
        const int ki = G % kRingK, vi = G % kRingV;
        uint8_t* const kt = s.k[ki];
        uint8_t* const vt = s.v[vi];
        const uint32_t v_phase = (v_par >> vi) & 1u;
        v_par ^= 1u << vi;
        const bool drafts = tile == p.tiles - 1;
        uint32_t gone[4] = {0u, 0u, 0u, 0u};  // absent tokens
        if (drafts && parents)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            gone[k] = __ballot_sync(0xffffffffu, 32 * k + lane < a.tokens && parents[32 * k + lane] < -1);
        // The products with P = 0 have to leave no trace of a drafted token's v, whatever it
        // holds: absent tokens' rows are cleared, and infinities and NaN of the others are
        // cleared and put back at the end for the rows that see them.
        uint32_t bad[4] = {0u, 0u, 0u, 0u};
        constexpr int kPer = kFewDrafts * (D / 8) / 32;
        if (drafts && p.shares) {
          uint4 kx[kPer], vx[kPer];
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int x = i * 32 + lane, row = x / (D / 8);
            kx[i] = vx[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row < a.tokens) {
              const int64_t at = p.b * a.n_b + row * a.n_t + p.kvh * a.n_h + (x % (D / 8)) * 8;
              kx[i] = *reinterpret_cast<const uint4*>(a.k_new + at);
              vx[i] = *reinterpret_cast<const uint4*>(a.v_new + at);
            }
          }
          if (!tree_wait(&s.k_land[ki], (k_par >> ki) & 1u, &s.abort, 41)) { ok = false; break; }
          k_par ^= 1u << ki;
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int x = i * 32 + lane, row = x / (D / 8);
            if (row < a.tokens) *chunk(kt, rest + row, x % (D / 8)) = kx[i];
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.k_full[ki]);
          if (!tree_wait(&s.v_land[vi], v_phase, &s.abort, 42)) { ok = false; break; }
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int x = i * 32 + lane, row = x / (D / 8);
            if (row < a.tokens) {
              if ((gone[0] >> row) & 1u) vx[i] = make_uint4(0u, 0u, 0u, 0u);
              if (not_finite(vx[i])) {
                bad[0] |= 1u << row;
                clear_not_finite(vx[i].x);
                clear_not_finite(vx[i].y);
                clear_not_finite(vx[i].z);
                clear_not_finite(vx[i].w);
              }
              *chunk(vt, rest + row, x % (D / 8)) = vx[i];
            }
          }
          bad[0] = __reduce_or_sync(0xffffffffu, bad[0]);
        } else {
          if (!tree_wait(&s.v_land[vi], v_phase, &s.abort, 43)) { ok = false; break; }
          if (drafts) {
            uint32_t any_bad = 0u;
#pragma unroll 4
            for (int x = lane; x < a.tokens * (D / 8); x += 32) {
              const int row = x / (D / 8);
              const uint32_t g4 = row < 32 ? gone[0] : row < 64 ? gone[1] : row < 96 ? gone[2] : gone[3];
              uint4* const at = chunk(vt, row, x % (D / 8));
              if ((g4 >> (row & 31)) & 1u) *at = make_uint4(0u, 0u, 0u, 0u);
              else any_bad |= not_finite(*at);
            }
            __syncwarp();
            if (__any_sync(0xffffffffu, any_bad != 0u)) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                bool mine = false;
#pragma unroll 1
                for (int c = 0; c < D / 8; ++c) {
                  uint4* const at = chunk(vt, 32 * k + lane, c);
                  uint4 y = *at;
                  if (!not_finite(y)) continue;
                  mine = true;
                  clear_not_finite(y.x);
                  clear_not_finite(y.y);
                  clear_not_finite(y.z);
                  clear_not_finite(y.w);
                  *at = y;
                }
                bad[k] = __ballot_sync(0xffffffffu, mine);
              }
            }
          }
        }
        if (rest > 0) {  // rows past the end hold whatever the page or the ring held before
#pragma unroll 4
          for (int x = (rest + (drafts ? a.tokens : 0)) * 8 + lane; x < kTile * 8; x += 32)
#pragma unroll
            for (int c = 0; c < kSub; ++c)
              *reinterpret_cast<uint4*>(vt + c * (kTile * 128) + x * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        if (drafts && lane < 4) s.bad[uc & 7][lane] = lane == 0 ? bad[0] : lane == 1 ? bad[1] : lane == 2 ? bad[2] : bad[3];
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.v_full[vi]);
      }
      gt += (uint32_t)p.n;
      ++uc;
    }
  } else {
    // ------------------------------------------------ softmax groups
    const int g = warp >> 2, qd = warp & 3;
    const int r = qd * 32 + lane;  // row of the query tile == TMEM lane
    const uint32_t lane_off = (uint32_t)(qd * 32) << 16;
    const uint32_t s_addr = tmem + lane_off + (uint32_t)(g * kTile);
    const uint32_t o_addr = tmem + lane_off + kOCol;
    uint32_t gt = 0, uc = 0;
    bool ok = true;
    Piece p;
    while (ok && next_piece(a, w, p)) {
      const int n = p.n;
      const int tok0 = (p.mb * NQ + (NQ == 1 ? 0 : g)) * a.tt;
      const int rows = max(min(a.tt, a.tokens - tok0), 0) * a.group;
      const bool busy = qd * 32 < rows;  // a warp without query rows only keeps the barriers going
      const int token = tok0 + r / a.group;
      uint32_t seen[4] = {0u, 0u, 0u, 0u};
      float m = -INFINITY, l = 0.f;
      bool any = false;  // this group has had a tile of this piece
      for (int t = 0; t < n; ++t) {
        const uint32_t G = gt + (uint32_t)t;
        if (NQ == 1 && (int)(G & 1u) != g) continue;
        const uint32_t use = NQ == 1 ? G >> 1 : G;  // how often the group's buffers were used before
        const int tile = p.t0 + t;
        const int rest = p.len - tile * kTile;  // cached keys of the tile
        const bool drafts = tile == p.tiles - 1;
        if (drafts && r < rows) ancestor_bits(a.parents ? a.parents + (int64_t)p.b * a.tokens : nullptr, token, seen);
        if (!tree_wait(&s.s_full[g], use & 1u, &s.abort, 31)) { ok = false; break; }
        tc_fence_after();
        // A loop and not straight code for the halves: the code's first pass is fetched from L2,
        // and that is what a short call waits for.
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (busy) {
            const uint32_t half = s_addr + (uint32_t)(h * (kTile / 2));
            uint32_t v[64];
            tmem_ld32(half, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
            tmem_ld32(half + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
            tmem_wait_ld();
            reg_fence<64>(v);
            const int left = rest - 64 * h;  // cached keys of this half
            if (left < 64) {
              uint32_t keep[2];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const int x = left - 32 * c;
                keep[c] = x >= 32 ? 0xffffffffu : x > 0 ? (1u << x) - 1u : 0u;
                if (rest <= 0) keep[c] = h == 0 ? seen[c] : seen[2 + c];
                else if (x < 32 && x > -32) keep[c] |= x >= 0 ? seen[0] << x : seen[0] >> -x;
              }
#pragma unroll
              for (int k = 0; k < 64; ++k) v[k] = (keep[k >> 5] >> (k & 31)) & 1u ? v[k] : 0xff800000u;
            }
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 64; k += 8)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                x[j] = max3f(x[j], __uint_as_float(v[k + 2 * j]), __uint_as_float(v[k + 2 * j + 1]));
            const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * a.scale_log2;
            float factor = 1.f;
            if (m == -INFINITY) {
              m = mx;  // nothing seen before: O and l are zero
            } else if (mx > m + kLag) {
              factor = fast_exp2(m - mx);
              m = mx;
            }
            const float neg_m = m == -INFINITY ? 0.f : -m;
            f32x2 rs[2];
            if (p.len <= kFine) {
              uint32_t y[2][32];  // of 32 keys each: 16 words of first parts, 16 of second ones
              f32x2 r2[2];
              exp_pack_two<32, 2>(v, y[0], y[0] + 16, a.scale_log2, neg_m, rs);
              exp_pack_two<32, 2>(v + 32, y[1], y[1] + 16, a.scale_log2, neg_m, r2);
              rs[0] = f2_add(rs[0], r2[0]);
              rs[1] = f2_add(rs[1], r2[1]);
              tmem_st32(half, y[0]);
              tmem_st32(half + 32, y[1]);
            } else {
              exp_pack_rounded<64, 2>(v, a.scale_log2, neg_m, rs);
              tmem_st16(half, *reinterpret_cast<const uint32_t(*)[16]>(&v[0]));
              tmem_st16(half + 32, *reinterpret_cast<const uint32_t(*)[16]>(&v[16]));
            }
            l = l * factor + ((f2_lo(rs[0]) + f2_hi(rs[0])) + (f2_lo(rs[1]) + f2_hi(rs[1])));
            if ((any || h > 0) && __any_sync(0xffffffffu, factor != 1.f)) {
              // O *= factor; it must hold every product before this one
              if (!tree_wait(&s.o_done[g][h ^ 1], (h ? use : use - 1) & 1u, &s.abort, 32)) { ok = false; break; }
              tc_fence_after();
              tmem_wait_st();
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_ld32(o_addr + (uint32_t)(g * D + c), o);
                tmem_wait_ld();
                reg_fence<32>(o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
                tmem_st32(o_addr + (uint32_t)(g * D + c), o);
              }
            }
            tmem_wait_st();
          }
          tc_fence_before();
          mbar_arrive(&s.p_full[g][h]);
        }
        if (!ok) break;
        any = true;
      }
      if (!ok) break;
      // ---------------- end of the piece: O / l, or the piece's (max, sum, O)
      const bool cut = !(p.t0 == 0 && n == p.tiles);
      const int slot = 2 * (int)blockIdx.x + (p.t0 == 0 ? 1 : 0);
      if (NQ == 1 && p.t0 + n == p.tiles && r < rows && (int)((gt + (uint32_t)n - 1) & 1u) != g)
        ancestor_bits(a.parents ? a.parents + (int64_t)p.b * a.tokens : nullptr, token, seen);  // the other group had the drafted tile
      const bool here = (seen[0] | seen[1] | seen[2] | seen[3]) != 0u;
      const uint32_t last = gt + (uint32_t)n - 1;
      const int64_t row_at =
          (((int64_t)p.b * a.tokens + token) * a.heads + p.kvh * a.group + r % a.group) * D;
      float w0 = 1.f, w1 = 0.f;
      bool use0 = true, use1 = false;
      int c0 = 0, c1 = D;
      if constexpr (NQ == 1) {
        // both groups' results: this one writes half of the columns
        if (uc > 0 && !tree_wait(&s.o_free[0], (uc - 1) & 1u, &s.abort, 34)) { ok = false; break; }
        s.xm[g][r] = m;
        s.xl[g][r] = l;
        mbar_arrive(&s.x_full);
        // This group's last product first: with it all products before it are complete, so the
        // other group's barrier is at most one phase short of the one waited for (a parity says
        // nothing about a phase two ahead).
        const uint32_t own = (last & 1u) == (uint32_t)g ? last : last - 1;
        const uint32_t other = own == last ? last - 1 : last;
        if ((n > 1 || own == last) && !tree_wait(&s.o_done[g][1], (own >> 1) & 1u, &s.abort, 35)) { ok = false; break; }
        if ((n > 1 || other == last) && !tree_wait(&s.o_done[g ^ 1][1], (other >> 1) & 1u, &s.abort, 36)) { ok = false; break; }
        if (!tree_wait(&s.x_full, uc & 1u, &s.abort, 37)) { ok = false; break; }
        use0 = n > 1 || (last & 1u) == 0u;
        use1 = n > 1 || (last & 1u) == 1u;
        const float m0 = use0 ? s.xm[0][r] : -INFINITY, m1 = use1 ? s.xm[1][r] : -INFINITY;
        m = fmaxf(m0, m1);
        w0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - m);
        w1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - m);
        l = (use0 ? s.xl[0][r] * w0 : 0.f) + (use1 ? s.xl[1][r] * w1 : 0.f);
        c0 = g * (D / 2);
        c1 = c0 + D / 2;
      } else {
        if (!tree_wait(&s.o_done[g][1], last & 1u, &s.abort, 35)) { ok = false; break; }
      }
      tc_fence_after();
      const float inv = cut ? 1.f : here ? 1.f / l : 0.f;
      uint32_t sees_bad[4] = {0u, 0u, 0u, 0u};  // drafted tokens that bring infinities or NaN to this row
      if (p.t0 + n == p.tiles) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sees_bad[k] = r < rows ? seen[k] & s.bad[uc & 7][k] : 0u;
      }
      if (busy) {
        const int ti = NQ == 1 ? 0 : g;
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
          uint32_t o[32];
          if constexpr (NQ == 1) {
            uint32_t x[32];
            tmem_ld32(o_addr + (uint32_t)c, o);
            tmem_ld32(o_addr + (uint32_t)(D + c), x);
            tmem_wait_ld();
            reg_fence<32>(o);
            reg_fence<32>(x);
#pragma unroll
            for (int k = 0; k < 32; ++k) {  // an unused group's O is not read as a number
              const float y0 = use0 ? __uint_as_float(o[k]) * w0 : 0.f;
              const float y1 = use1 ? __uint_as_float(x[k]) * w1 : 0.f;
              o[k] = __float_as_uint((y0 + y1) * inv);
            }
          } else {
            tmem_ld32(o_addr + (uint32_t)(g * D + c), o);
            tmem_wait_ld();
            reg_fence<32>(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * inv);
          }
          if ((sees_bad[0] | sees_bad[1] | sees_bad[2] | sees_bad[3]) != 0u) {
            for (int j = 0; j < a.tokens; ++j) {
              const uint32_t bits = j < 32 ? sees_bad[0] : j < 64 ? sees_bad[1] : j < 96 ? sees_bad[2] : sees_bad[3];
              if (!((bits >> (j & 31)) & 1u)) continue;
              const bf16* vj = a.v_new + p.b * a.n_b + j * a.n_t + p.kvh * a.n_h + c;
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                const float x = __bfloat162float(vj[k]);
                if (!(fabsf(x) < INFINITY)) o[k] = __float_as_uint(__uint_as_float(o[k]) + x);
              }
            }
          }
          if (r < rows) {
            if (cut) {
              float4* to = a.ws_o + ((int64_t)(slot * NQ + ti) * (D / 4) + c / 4) * kTile + r;
#pragma unroll
              for (int k = 0; k < 8; ++k)
                to[k * kTile] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                            __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint4 packed = pack16<bf16>(reinterpret_cast<const float*>(o) + 8 * k);
                if (!here) packed = make_uint4(0u, 0u, 0u, 0u);
                *reinterpret_cast<uint4*>(a.out + row_at + c + 8 * k) = packed;
              }
            }
          }
        }
        if (cut && r < rows && (NQ == 2 || g == 0)) {
          float* to = a.ws_ml + (int64_t)(slot * NQ + ti) * 2 * kTile + r;
          to[0] = m;
          to[kTile] = l;
        }
      }
      tc_fence_before();
      mbar_arrive(&s.o_free[NQ == 1 ? 0 : g]);
      gt += (uint32_t)n;
      ++uc;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the pieces of the segments that were cut: out = sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p,
// in order of the pieces. blockIdx.y: a block of the attention kernel that begins inside a
// segment, the first one that does; blockIdx.x: 8 rows of the segment, a thread 4 columns of one row.
template <int D, int NQ>
__global__ void __launch_bounds__(2 * D) tree_join_kernel(const __grid_constant__ TcArgs a, int blocks) {
  __shared__ int stop;  // the first later block that does not begin inside the segment
  pdl_enter();
  const int c = blockIdx.y + 1;
  if (threadIdx.x == 0) stop = blocks;
  const int4 at = a.ws_start[c], before = a.ws_start[c - 1];
  __syncthreads();
  if (at.z == 0 || (before.x == at.x && before.y == at.y && before.z > 0)) return;
  for (int i = c + 1 + threadIdx.x; i < blocks; i += 2 * D) {
    const int4 x = a.ws_start[i];
    if (x.x != at.x || x.y != at.y || x.z == 0) atomicMin(&stop, i);
  }
  __syncthreads();
  const int b = at.x, hm = at.y, lo = c;
  const int kvh = a.row_blocks == 1 ? hm : hm / a.row_blocks, mb = hm - kvh * a.row_blocks;
  const int pieces = stop - c + 1;  // piece 0 is the end of block c - 1, piece i the beginning of block c - 1 + i
  const int x0 = blockIdx.x * 8;    // the block's rows, all of one query tile
  const int ti = x0 / kTile, r0 = x0 - ti * kTile;
  auto slot = [&](int i) { return (int64_t)((i == 0 ? 2 * (lo - 1) + 1 : 2 * (lo - 1 + i)) * NQ + ti); };
  // The pieces' weights 2^(m_p - m) for the 8 rows, and 1 / sum_p 2^(m_p - m) l_p.
  __shared__ float weight[kMaxPieces][8];
  __shared__ float inverse[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int y = warp; y < 8; y += 2 * D / 32) {
    const int r = r0 + y;
    float m = -INFINITY, l = 0.f, mi[kMaxPieces / 32], li[kMaxPieces / 32];
#pragma unroll
    for (int k = 0; k < kMaxPieces / 32; ++k) {
      const int i = k * 32 + lane;
      const float* const ml = a.ws_ml + slot(i) * 2 * kTile + r;
      mi[k] = i < pieces ? __ldcg(ml) : -INFINITY;
      li[k] = i < pieces ? __ldcg(ml + kTile) : 0.f;
      m = fmaxf(m, mi[k]);
    }
    m = warp_max(m);
#pragma unroll
    for (int k = 0; k < kMaxPieces / 32; ++k) {
      const int i = k * 32 + lane;
      if (i >= pieces) continue;
      // without a maximum the sum is 0, or NaN where all that is visible of the piece scores NaN
      const float wi = mi[k] == -INFINITY ? li[k] : fast_exp2(mi[k] - m);
      weight[i][y] = wi;
      l += wi == 0.f ? 0.f : wi * li[k];
    }
    l = warp_sum(l);
    if (lane == 0) inverse[y] = 1.f / l;
  }
  __syncthreads();
  const int r = r0 + (threadIdx.x & 7), c4 = threadIdx.x >> 3;
  const int token = (mb * NQ + ti) * a.tt + r / a.group;
  if (r >= a.tt * a.group || token >= a.tokens) return;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = 0; i < pieces; ++i) {
    const float4 v = __ldcg(a.ws_o + (slot(i) * (D / 4) + c4) * kTile + r);
    const float wi = weight[i][threadIdx.x & 7];
    o.x = wi == 0.f ? o.x : fmaf(wi, v.x, o.x);
    o.y = wi == 0.f ? o.y : fmaf(wi, v.y, o.y);
    o.z = wi == 0.f ? o.z : fmaf(wi, v.z, o.z);
    o.w = wi == 0.f ? o.w : fmaf(wi, v.w, o.w);
  }
  const bool here = !a.parents || a.parents[(int64_t)b * a.tokens + token] >= -1;
  const float inv = here ? inverse[threadIdx.x & 7] : 0.f;
  if (!here) o = make_float4(0.f, 0.f, 0.f, 0.f);
  store4(a.out + (((int64_t)b * a.tokens + token) * a.heads + kvh * a.group + r % a.group) * D + c4 * 4,
         make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// ------------------------------------------------------------------ host

struct TcPlan {
  bool on;          // the tensor-core kernel takes this call
  int nq, tt, row_blocks, box, grid;
  bool join;        // segments may be cut
  size_t ml_off, o_off, bytes;
};

// The call's sizes and types (not its strides and pointers) decide: bf16 whose rows make whole
// 128-byte lines goes here at every length; the file's head has both kernels' times.
TcPlan tc_plan(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t d, int64_t page,
               int64_t max_pages, int dtype) {
  TcPlan p = {};
  const int64_t group = heads / kv_heads;
  if (dtype != NKL_BFLOAT16 || (d != 64 && d != 128) || group > kTile || page % 8 != 0) return p;
  p.box = 8;
  while (p.box < kTile && page % (2 * p.box) == 0) p.box *= 2;
  if (page / p.box > 256) return p;  // the division by boxes per page is exact up to there
  p.tt = (int)(kTile / group);
  const int64_t q_tiles = (tokens + p.tt - 1) / p.tt;
  p.nq = q_tiles > 1 ? 2 : 1;
  p.row_blocks = (int)((q_tiles + p.nq - 1) / p.nq);
  const int64_t seg_tiles = (page * max_pages + kTile - 1) / kTile + 1;  // at most
  const int64_t segments = batch * kv_heads * p.row_blocks;
  if (segments * (seg_tiles + kExtra) > 0x7fffffffLL / 4 || kv_heads * p.row_blocks > 65535) return p;
  p.on = true;
  p.join = seg_tiles > kWhole;
  p.grid = (int)std::min<int64_t>(std::min(sm_count(), kMaxPieces - 1), p.join ? segments * seg_tiles : segments);
  if (p.join) {
    const size_t slots = 2 * (size_t)p.grid * p.nq;
    p.ml_off = ((size_t)p.grid * 16 + 255) & ~size_t(255);
    p.o_off = p.ml_off + slots * 2 * kTile * 4;
    p.bytes = p.o_off + slots * kTile * d * 4;
  }
  return p;
}

template <int D, int NQ>
int tc_launch(const TreeArgs& g, const TcPlan& p, unsigned char* ws, cudaStream_t st) {
  const char* op = "nkl_attention_tree";
  CUtensorMap mq, mkn, mvn, mkc, mvc;
  {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)g.heads, (uint64_t)g.tokens, (uint64_t)g.batch};
    const uint64_t strides[3] = {(uint64_t)g.q_h * 2, (uint64_t)g.q_t * 2, (uint64_t)g.q_b * 2};
    const uint32_t box[4] = {64, (uint32_t)g.group, (uint32_t)p.tt, 1};
    if (int rc = make_tensor_map_bf16(&mq, g.q, 4, dims, strides, box, op)) return rc;
  }
  {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)g.tokens, (uint64_t)g.kv_heads, (uint64_t)g.batch};
    const uint64_t strides[3] = {(uint64_t)g.n_t * 2, (uint64_t)g.n_h * 2, (uint64_t)g.n_b * 2};
    const uint32_t box[4] = {64, kTile, 1, 1};
    if (int rc = make_tensor_map_bf16(&mkn, g.k_new, 4, dims, strides, box, op)) return rc;
    if (int rc = make_tensor_map_bf16(&mvn, g.v_new, 4, dims, strides, box, op)) return rc;
  }
  {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)g.page, (uint64_t)g.kv_heads, (uint64_t)g.pages};
    const uint64_t strides[3] = {(uint64_t)g.c_s * 2, (uint64_t)g.c_h * 2, (uint64_t)g.c_p * 2};
    const uint32_t box[4] = {64, (uint32_t)p.box, 1, 1};
    if (int rc = make_tensor_map_bf16(&mkc, g.k_cache, 4, dims, strides, box, op)) return rc;
    if (int rc = make_tensor_map_bf16(&mvc, g.v_cache, 4, dims, strides, box, op)) return rc;
  }
  TcArgs a = {};
  a.tables = g.tables;
  a.lens = g.lens;
  a.parents = g.parents;
  a.k_new = static_cast<const bf16*>(g.k_new);
  a.v_new = static_cast<const bf16*>(g.v_new);
  a.n_b = g.n_b;
  a.n_t = g.n_t;
  a.n_h = g.n_h;
  a.out = static_cast<bf16*>(g.out);
  if (p.join) {
    a.ws_start = reinterpret_cast<int4*>(ws);
    a.ws_ml = reinterpret_cast<float*>(ws + p.ml_off);
    a.ws_o = reinterpret_cast<float4*>(ws + p.o_off);
  }
  a.batch = g.batch; a.tokens = g.tokens; a.heads = g.heads; a.kv_heads = g.kv_heads; a.group = g.group;
  a.pages = g.pages; a.page = g.page; a.max_pages = g.max_pages; a.capacity = g.max_pages * g.page;
  a.tt = p.tt; a.row_blocks = p.row_blocks; a.box = p.box;
  a.boxes_per_page = g.page / p.box;
  a.log_bpt = 0;
  while (p.box << a.log_bpt < kTile) ++a.log_bpt;
  a.log_bpp = -1;
  for (int i = 0; i < 9; ++i)
    if (a.boxes_per_page == 1 << i) a.log_bpp = i;
  a.bpp_magic = ((1ull << 36) + a.boxes_per_page - 1) / a.boxes_per_page;
  a.scale_log2 = g.scale * kLog2e;
  constexpr size_t smem = sizeof(TreeSmem<D, NQ>);
  static_assert(smem <= 232448, "shared memory of a block");
  static std::atomic<bool> set[64] = {};  // per device: the smem attribute is set (idempotent)
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(tree_attention_tc_kernel<D, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return fail(NKL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_release);
  }
  int rc = launch_pdl(tree_attention_tc_kernel<D, NQ>, dim3((unsigned)p.grid), dim3(kTcThreads), smem, st, op, mq, mkn,
                      mvn, mkc, mvc, a);
  if (rc || !p.join || p.grid < 2) return rc;
  const int rows = std::min<int>(NQ == 1 ? p.tt * g.group : NQ * kTile, NQ == 1 ? g.tokens * g.group : NQ * kTile);
  return launch_pdl(tree_join_kernel<D, NQ>, dim3((unsigned)((rows + 7) / 8), (unsigned)(p.grid - 1)), dim3(2 * D), 0, st,
                    op, a, p.grid);
}

}  // namespace
