// tree_attention_8bit_ring.cuh - the tree attention over a cache in 8 bits for up to 16 query rows to a key/value
// head (bf16, head_dim 64 or 128, pages of a multiple of 8): a decoding step; included by tree_attention.cu.
//
// The work is shared out as by the tcgen05 kernel (tree_plan: all segments' tiles of 128 positions in a row,
// cut into equal shares on the GPU; the drafted tokens count as a tile of their own), one block to an SM.
//   warp 8    TMA: tiles of keys and values, as bytes, through a ring of four, five or eight
//   warp 9    the powers of two of their rows
//   warp 10   the drafted tokens, while the others are at the cached ones
//   warps 0-7 16 keys of each tile: the products of tree_attention_8bit.cuh with fragments by ldmatrix (transposed
//             for the values, two entries of a key at a time, which __byte_perm pairs with the next key's), sums of
//             their own; at a piece's end the sums meet in shared memory, while the ring goes on
// Segments that are cut leave (max, sum, O) of a piece in the workspace for tree_join_kernel.
//
// Measured against the kernel of tree_attention_8bit.cuh on the same calls, GPU time with the join (32 heads over 8 of
// 128 but where it says so):
//   1 token, 203 positions                                7.2 and 11 us
//   1 token, 32 sequences of up to 8192                    85 and 150 us (60 by bytes)
//   1 token, 65536 positions                               41 and 49 us (20 by bytes)
//   1 token, 64 sequences of about 700                     37 and 35 us (10 by bytes)
//   4 tokens, 8 sequences of up to 4096                    34 and 47 us (6 by bytes)
//   16 tokens, 4 sequences of up to 4096, 32 heads of 128  50 and 70 us (12 by bytes)
// so every call that it can take goes here: only many short sequences lose by it, 2 us, and how long they are the host
// does not know. What bounds it: on long rows the products' warps, 1130 cycles to a tile of 32 KB. The conversions from
// e4m3 to f16 are 264 of them (measured alone: a scheduler takes one of 32 lanes every other cycle, the SM's four 512 to a
// tile), with the loads and products around them some 380; the rest is the chain from the scores over the weights to the
// transposed ones, with two warps to a scheduler, which issue in 43 % of the cycles. On short rows it is a piece's
// beginning and end (5000 cycles) and the start: plan, tables and the first tiles take 7000. More than eight such warps do
// not fit: their sums are 64 or 128 registers each. The drafted tokens by one of the eight warps at a piece's end instead
// of by warp 10: 32 sequences 117 us for 109, 203 positions 11.8 for 7.8 (at that time).
#pragma once

namespace {

constexpr int kRingWarps = 8, kRingThreads = 32 * (kRingWarps + 3);

template <int D, int NT>
struct RingSmem {
  static constexpr int kStages = D == 128 ? 6 - NT : 8;
  uint8_t tile[kStages][2][kTile * D];
  float o[kRingWarps + 1][8 * NT][D];
  float ml[kRingWarps + 1][8 * NT][2];
  alignas(4) uint8_t powers[kStages][2][kTile];
  uint64_t full[kStages], empty[kStages], joined, read;
  int bad, abort;
};

__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

// The drafted tokens, at most 16, of a piece that ends a segment, by one warp, as drafted_8bit has it; but the loads go
// out together, the ancestors are followed from lane to lane, and k and v stay in bf16. It is short because it runs
// cold, between the others' products: instructions that are not there yet cost it more than memory.
template <int NT, int DC>
__device__ __forceinline__ bool drafted_few(const TreeArgs& t, const Piece& p, Sums8<NT, DC>& sums) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int64_t from = p.b * t.n_b + p.kvh * t.n_h;
  const bf16* const kn = static_cast<const bf16*>(t.k_new) + from;
  const bf16* const vn = static_cast<const bf16*>(t.v_new) + from;
  const bf16* const qn = static_cast<const bf16*>(t.q) + p.b * t.q_b;
  const int up0 = lane >= t.tokens ? -2 : t.parents ? t.parents[(int64_t)p.b * t.tokens + lane] : lane - 1;  // this lane's token
  uint2 kr[4 * DC][2], qr[4 * DC][NT];
  uint32_t v[4 * DC][4];
  int token_of[NT];
#pragma unroll
  for (int y = 0; y < NT; ++y) {
    const int r = 8 * y + g, token = r / t.group;
    const bool real = r < t.tokens * t.group;
    token_of[y] = real ? token : 31;  // its `up` is -2
    const bf16* const row = qn + (real ? token * t.q_t + (p.kvh * t.group + r - token * t.group) * t.q_h : 0);
#pragma unroll
    for (int s = 0; s < 4 * DC; ++s) qr[s][y] = *reinterpret_cast<const uint2*>(row + 16 * s + 4 * t4);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const bf16* const row = kn + min(8 * k + g, t.tokens - 1) * t.n_t + 4 * t4;
#pragma unroll
    for (int s = 0; s < 4 * DC; ++s) kr[s][k] = *reinterpret_cast<const uint2*>(row + 16 * s);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bf16* const row = vn + min(2 * t4 + (i & 1) + 8 * (i >> 1), t.tokens - 1) * t.n_t + 2 * g;
#pragma unroll
    for (int j = 0; j < 4 * DC; ++j) v[j][i] = *reinterpret_cast<const uint32_t*>(row + 16 * j);
  }
  uint32_t seen = 0u;  // the tokens that this lane's sees, itself one of them
  {
    int at = lane, up = up0;
    bool on = up >= -1;
    while (__any_sync(0xffffffffu, on)) {
      if (on) seen |= 1u << at;
      on = on && up >= 0 && up < at;  // not the root, nor a parent that comes later, which is none
      if (on) at = up;
      up = __shfl_sync(0xffffffffu, up0, at);
      on = on && up >= -1;  // an absent parent ends the path
    }
  }
  float x[NT][4] = {};
#pragma unroll
  for (int y = 0; y < NT; ++y) {
    const bool real = __shfl_sync(0xffffffffu, up0, token_of[y]) >= -1;  // rows that are none, or absent, stay unread
#pragma unroll
    for (int s = 0; s < 4 * DC; ++s) {
      const uint32_t ka[4] = {kr[s][0].x, kr[s][1].x, kr[s][0].y, kr[s][1].y};
      mma_b16(x[y], ka, real ? qr[s][y].x : 0u, real ? qr[s][y].y : 0u);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * y + 2 * t4 + i;
      const uint32_t bits = __shfl_sync(0xffffffffu, seen, r < t.tokens * t.group ? r / t.group : 31);
#pragma unroll
      for (int k = 0; k < 2; ++k) x[y][2 * k + i] = (bits >> (8 * k + g)) & 1u ? x[y][2 * k + i] * (t.scale * kLog2e) : -INFINITY;
    }
  }
  const float none[2] = {0.f, 0.f};
  sums.weigh(x, none);
  uint32_t w[NT][2][2];  // the weights in two parts
#pragma unroll
  for (int y = 0; y < NT; ++y)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float a = x[y][2 * k], b = x[y][2 * k + 1];
      const __nv_bfloat162 hi = __floats2bfloat162_rn(a, b);
      const __nv_bfloat162 lo = __floats2bfloat162_rn(a - __low2float(hi), b - __high2float(hi));
      w[y][0][k] = transpose(*reinterpret_cast<const uint32_t*>(&hi));
      w[y][1][k] = transpose(*reinterpret_cast<const uint32_t*>(&lo));
    }
  // weights of 0 must meet no infinity: v that are not finite, or of absent tokens, are left out here
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool here = __shfl_sync(0xffffffffu, up0, 2 * t4 + (i & 1) + 8 * (i >> 1)) >= -1;
#pragma unroll
    for (int j = 0; j < 4 * DC; ++j) {
      if (!here) v[j][i] = 0u;
      bad |= (v[j][i] & 0x7f80u) == 0x7f80u || (v[j][i] & 0x7f800000u) == 0x7f800000u;
    }
  }
  bad = __any_sync(0xffffffffu, bad);
  if (bad)
#pragma unroll
    for (int j = 0; j < 4 * DC; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if ((v[j][i] & 0x7f80u) == 0x7f80u) v[j][i] &= 0xffff0000u;
        if ((v[j][i] & 0x7f800000u) == 0x7f800000u) v[j][i] &= 0xffffu;
      }
#pragma unroll
  for (int j = 0; j < 4 * DC; ++j) {
    const uint32_t va[4] = {__byte_perm(v[j][0], v[j][1], 0x5410), __byte_perm(v[j][0], v[j][1], 0x7632),
                            __byte_perm(v[j][2], v[j][3], 0x5410), __byte_perm(v[j][2], v[j][3], 0x7632)};
#pragma unroll
    for (int y = 0; y < NT; ++y)
#pragma unroll
      for (int z = 1; z >= 0; --z) mma_b16(sums.o[y][j], va, w[y][z][0], w[y][z][1]);
  }
  return bad;
}

// t: the call, for the drafted tokens and the queries; a: the plan's view of it, whose `tokens` says that the
// drafted tokens have a tile of their own.
template <int D, int NT>
__global__ void __launch_bounds__(kRingThreads, 1)
attention_8bit_ring_kernel(const __grid_constant__ CUtensorMap map_kc, const __grid_constant__ CUtensorMap map_vc,
                           const __grid_constant__ TcArgs a, const __grid_constant__ TreeArgs t) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (smem_u32(smem_raw) & 1023u) {  // the swizzled tiles need a 1024-byte-aligned base
    if (threadIdx.x == 0) atomicCAS(&g_tree_dev_error, 0u, 50u);
    pdl_enter();
    return;
  }
  typedef RingSmem<D, NT> Smem;
  Smem& s = *reinterpret_cast<Smem*>(smem_raw);
  constexpr int kStages = Smem::kStages, DC = D / 64;
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.full[i], 2);
      mbar_init(&s.empty[i], kRingWarps);
    }
    mbar_init(&s.joined, kRingWarps + 1);
    mbar_init(&s.read, kRingWarps);
    s.abort = 0;
    s.bad = 0;
    fence_barrier_init();
  }
  if (warp == kRingWarps && lane == 0) {
    tma_prefetch_desc(&map_kc);
    tma_prefetch_desc(&map_vc);
  }
  __syncthreads();
  pdl_wait();
  Walk w = tree_plan(a);
  if (a.ws_start && threadIdx.x == 0) a.ws_start[blockIdx.x] = make_int4(w.b, w.hm, w.t, 0);
  uint32_t st = 0, par = 0;
  bool ok = true;
  Piece p = {};
  auto cached_end = [&] { return min(p.t0 + p.n, (p.len + kTile - 1) / kTile); };  // of the piece's tiles of cached keys

  // the piece's query rows, where a row of 16 entries' products lies, and the sums' columns
  const int rows = t.tokens * t.group, g = lane >> 2, t4 = lane & 3;
  auto parents_of = [&](const Piece& p) { return t.parents ? t.parents + (int64_t)p.b * t.tokens : nullptr; };
  auto queries_of = [&](const Piece& p) {
    return [&](int r, bool& real) {
      const int token = r / t.group;
      const int* const parents = parents_of(p);
      real = r < rows && (!parents || parents[token] >= -1);
      return static_cast<const bf16*>(t.q) + p.b * t.q_b + (real ? token * t.q_t + (p.kvh * t.group + r - token * t.group) * t.q_h : 0);
    };
  };
  auto entry = [&](int x) { return 16 * x + 4 * t4; };
  auto col = [&](int j) { return 16 * j + 2 * g; };
  // a warp's sums of its piece, into shared memory once the piece before is read out of it
  uint32_t uc = 0;
  auto leave = [&](Sums8<NT, DC>& sums, int at, bool bad) {
    if (uc > 0 && !tree_wait<true>(&s.read, (uc - 1) & 1u, &s.abort, 54)) return false;
    if (at == kRingWarps && lane == 0) s.bad = bad;
#pragma unroll
    for (int y = 0; y < NT; ++y)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int z = 4; z < 32; z *= 2) sums.l[y][i] += __shfl_xor_sync(0xffffffffu, sums.l[y][i], z);
        const int r = 8 * y + 2 * t4 + i;
        if (g == 0) {
          s.ml[at][r][0] = sums.m[y][i];
          s.ml[at][r][1] = sums.l[y][i];
        }
        // O's reference becomes the sums'
        const float f = sums.mv[y][i] == -INFINITY ? 1.f : fast_exp2(sums.mv[y][i] - kRaise - sums.m[y][i]);
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
          *reinterpret_cast<float2*>(&s.o[at][r][col(j)]) = make_float2(sums.o[y][j][i] * f, sums.o[y][j][2 + i] * f);
      }
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.joined);
    return true;
  };

  if (warp == kRingWarps) {
    // ------------------------------------------------ TMA
    const int per_tile = 1 << a.log_bpt;
    uint32_t used = 0u;
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
      int first = p.t0 * per_tile, page, slot, next_page, next_slot;
      look_up(first + lane, page, slot);
      look_up(first + 32 + lane, next_page, next_slot);
      const int end = cached_end();
      for (int x = p.t0; x < end; ++x) {
        const int boxes = (min(kTile, p.len - x * kTile) + a.box - 1) / a.box;
        const int at = x * per_tile - first;
        if (!tree_wait<true>(&s.empty[st], par ^ 1u, &s.abort, 51)) { ok = false; break; }
        used |= 1u << st;
        if (lane == 0) mbar_arrive_expect_tx(&s.full[st], (uint32_t)(2 * boxes * a.box * D));
        for (int i = 0; i < boxes; ++i) {
          const int pg = __shfl_sync(0xffffffffu, page, at + i), sl = __shfl_sync(0xffffffffu, slot, at + i);
          if (lane == 0) {
            tma_load_4d(s.tile[st][0] + i * a.box * D, &map_kc, &s.full[st], 0, sl, p.kvh, pg);
            tma_load_4d(s.tile[st][1] + i * a.box * D, &map_vc, &s.full[st], 0, sl, p.kvh, pg);
          }
        }
        __syncwarp();
        if (at + per_tile == 32) {
          first += 32;
          page = next_page;
          slot = next_slot;
          look_up(first + 32 + lane, next_page, next_slot);
        }
        if (++st == (uint32_t)kStages) { st = 0; par ^= 1u; }
      }
    }
    if (!ok && lane == 0) {  // let issued copies land before shared memory is released (or the time run out)
      const uint64_t begin = globaltimer();
      for (uint32_t i = 0; i < (uint32_t)kStages; ++i)
        if ((used >> i) & 1u)
          while (!mbar_try_wait(&s.full[i], i < st ? par : par ^ 1u) && globaltimer() - begin < kWaitTimeoutNs) {}
    }
  } else if (warp == kRingWarps + 1) {
    // ------------------------------------------------ the rows' powers of two
    while (ok && next_piece(a, w, p)) {
      const int end = cached_end();
      ok = put_powers(a, p, end, [&](uint32_t k, uint32_t v) {
        if (!tree_wait<true>(&s.empty[st], par ^ 1u, &s.abort, 52)) return false;
        reinterpret_cast<uint32_t*>(s.powers[st][0])[lane] = k;
        reinterpret_cast<uint32_t*>(s.powers[st][1])[lane] = v;
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.full[st]);
        if (++st == (uint32_t)kStages) { st = 0; par ^= 1u; }
        return true;
      });
    }
  } else if (warp == kRingWarps + 2) {
    // ------------------------------------------------ the drafted tokens, at most 16, of pieces that end a segment
    while (ok && next_piece(a, w, p)) {
      Sums8<NT, DC> sums;
      sums.clear();
      bool bad = false;
      if (p.t0 + p.n == p.tiles) bad = drafted_few(t, p, sums);
      ok = leave(sums, kRingWarps, bad);
      ++uc;
    }
  } else {
    // ------------------------------------------------ products
    // what ldmatrix reads: lane l gives the address of row l % 8 of matrix l / 8; the matrices are the first and last 8
    // of the warp's 16 keys, of a chunk of 16 entries and the next one
    const int key_row = 16 * warp + (lane & 15), chunk0 = lane >> 4;
    const uint32_t row_at = (uint32_t)(key_row * D);
    const uint32_t swizzle = D == 128 ? key_row & 7 : (key_row >> 1) & 3;
    Queries8<bf16, NT, DC> q;
    Piece next = {};
    bool more = next_piece(a, w, next);
    if (more) q.fetch(t, queries_of(next), entry);
    while (ok && more) {
      p = next;
      q.turn(t);
      Sums8<NT, DC> sums;
      sums.clear();
      const int end = cached_end();
      for (int x = p.t0; x < end; ++x) {
        if (!tree_wait<true>(&s.full[st], par, &s.abort, 53)) { ok = false; break; }
        const int left = p.len - x * kTile - 16 * warp;  // cached keys among the warp's 16
        if (left > 0) {
          const uint32_t kt = smem_u32(s.tile[st][0]) + row_at, vt = smem_u32(s.tile[st][1]) + row_at;
          float c[NT][2][4] = {};  // two sums, so that the products do not all wait for one another
#pragma unroll
          for (int z = 0; z < D / 16; z += 2) {
            uint32_t words[4];
            ldmatrix(words, kt + ((((uint32_t)(z + chunk0)) ^ swizzle) << 4));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t ka[4];
              e4m3_pairs(words[2 * h], ka[0], ka[2]);
              e4m3_pairs(words[2 * h + 1], ka[1], ka[3]);
#pragma unroll
              for (int y = 0; y < NT; ++y) mma_f16(c[y][h], ka, q.hi[y][z + h][0], q.hi[y][z + h][1]);
            }
          }
          float sc[NT][4], e[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int key = 8 * k + g;
            const uint32_t kc = s.powers[st][0][16 * warp + key], vc = s.powers[st][1][16 * warp + key];
            const float ks = kc == 255u ? NAN : kc == 0u ? 5.877472e-39f : __uint_as_float(kc << 23);
            const float ve = vc == 255u ? NAN : (float)((int)vc - 127);
            e[k] = key < left ? ve : 0.f;
#pragma unroll
            for (int y = 0; y < NT; ++y)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                sc[y][2 * k + i] = key < left ? (c[y][0][2 * k + i] + c[y][1][2 * k + i]) * q.factor[y][i] * ks : -INFINITY;
          }
          sums.weigh(sc, e);
          uint32_t pw[NT][2];
#pragma unroll
          for (int y = 0; y < NT; ++y)
#pragma unroll
            for (int k = 0; k < 2; ++k) pw[y][k] = transpose(half_pair(sc[y][2 * k], sc[y][2 * k + 1]));
          uint32_t there[2] = {0xffffffffu, 0xffffffffu};  // of the pairs of keys 2 t4, 2 t4 + 1 and 8 more
          if (left < 16)
#pragma unroll
            for (int k = 0; k < 2; ++k)
              there[k] = (8 * k + 2 * t4 < left ? 0xffffu : 0u) | (8 * k + 2 * t4 + 1 < left ? 0xffff0000u : 0u);
#pragma unroll
          for (int z = 0; z < D / 16; z += 2) {
            uint32_t words[4];
            ldmatrix_trans(words, vt + ((((uint32_t)(z + chunk0)) ^ swizzle) << 4));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t va[4];
              e4m3_pairs(__byte_perm(words[2 * h] & there[0], 0u, 0x3120), va[0], va[1]);
              e4m3_pairs(__byte_perm(words[2 * h + 1] & there[1], 0u, 0x3120), va[2], va[3]);
#pragma unroll
              for (int y = 0; y < NT; ++y) mma_f16(sums.o[y][z + h], va, pw[y][0], pw[y][1]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.empty[st]);
        if (++st == (uint32_t)kStages) { st = 0; par ^= 1u; }
      }
      if (!ok) break;
      // ------------------------------------------------ the piece's end: the warps' sums, in their order
      more = next_piece(a, w, next);
      if (more) q.fetch(t, queries_of(next), entry);  // on their way while the sums meet
      if (!leave(sums, warp, false)) { ok = false; break; }
      if (!tree_wait<true>(&s.joined, uc & 1u, &s.abort, 55)) { ok = false; break; }
      const int* const parents = parents_of(p);
      const bool whole = p.t0 + p.n == p.tiles, cut = !(p.t0 == 0 && whole);
      const int slot = 2 * (int)blockIdx.x + (p.t0 == 0 ? 1 : 0);
      for (int i = threadIdx.x; i < 8 * NT * (D / 4); i += 32 * kRingWarps) {
        const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
        if (r >= rows) break;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k <= kRingWarps; ++k) top = fmaxf(top, s.ml[k][r][0]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k <= kRingWarps; ++k) {
          const float mk = s.ml[k][r][0], lk = s.ml[k][r][1];
          if (mk == -INFINITY && lk == 0.f) continue;  // nothing seen (a sum of NaN: only NaN was)
          const float f = mk == top ? 1.f : fast_exp2(mk - top);
          const float4 y = *reinterpret_cast<const float4*>(&s.o[k][r][c]);
          sum = fmaf(f, lk, sum);
          x.x = fmaf(f, y.x, x.x);
          x.y = fmaf(f, y.y, x.y);
          x.z = fmaf(f, y.z, x.z);
          x.w = fmaf(f, y.w, x.w);
        }
        const int token = r / t.group;
        const bool present = !parents || parents[token] >= -1;
        if (s.bad && whole && present) {
          uint32_t seen[4];
          ancestor_bits(parents, token, seen);
          for (int j = 0; j < t.tokens; ++j) {
            if (!((seen[0] >> j) & 1u)) continue;
            const float4 v = four_of(static_cast<const bf16*>(t.v_new) + p.b * t.n_b + j * t.n_t + p.kvh * t.n_h + c);
            x.x += fabsf(v.x) < INFINITY ? 0.f : v.x;
            x.y += fabsf(v.y) < INFINITY ? 0.f : v.y;
            x.z += fabsf(v.z) < INFINITY ? 0.f : v.z;
            x.w += fabsf(v.w) < INFINITY ? 0.f : v.w;
          }
        }
        if (cut) {
          a.ws_o[((int64_t)slot * (D / 4) + c / 4) * kTile + r] = x;
          if (c == 0) {
            float* const to = a.ws_ml + (int64_t)slot * 2 * kTile + r;
            to[0] = top;
            to[kTile] = sum;
          }
        } else {
          const float inv = 1.f / sum;
          const float4 y = present ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
          store4(a.out + (((int64_t)p.b * t.tokens + token) * t.heads + p.kvh * t.group + r % t.group) * D + c, y);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.read);
      ++uc;
    }
  }
  __syncthreads();  // every warp is through with shared memory and its barriers
}

// ------------------------------------------------------------------ host

constexpr int kRingRows = 16;  // query rows to a key/value head, at most: two tiles of 8 to a warp

template <int D, int NT>
int ring_launch(const TreeArgs& g, const TcPlan& p, unsigned char* ws, cudaStream_t st, TcScales scales) {
  const char* op = "nkl_attention_tree_8bit";
  CUtensorMap mkc, mvc;
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)g.page, (uint64_t)g.kv_heads, (uint64_t)g.pages};
  const uint64_t strides[3] = {(uint64_t)g.c_s, (uint64_t)g.c_h, (uint64_t)g.c_p};
  const uint32_t box[4] = {D, (uint32_t)p.box, 1, 1};
  if (int rc = make_tensor_map_u8(&mkc, g.k_cache, 4, dims, strides, box, op)) return rc;
  if (int rc = make_tensor_map_u8(&mvc, g.v_cache, 4, dims, strides, box, op)) return rc;
  TcArgs a = tc_args(g, p, ws);
  a.k_scales = static_cast<const uint8_t*>(scales.k);
  a.v_scales = static_cast<const uint8_t*>(scales.v);
  a.block = scales.block;
  a.per_page = g.page / scales.block;
  TcArgs plan = a;
  plan.tokens = kTile;  // the drafted tokens have a tile of their own
  constexpr size_t smem = sizeof(RingSmem<D, NT>);
  static_assert(smem <= 232448, "shared memory of a block");
  if (int rc = allow_smem<attention_8bit_ring_kernel<D, NT>>(smem, op)) return rc;
  int rc = launch_pdl(attention_8bit_ring_kernel<D, NT>, dim3((unsigned)p.grid), dim3(kRingThreads), smem, st, op, mkc, mvc,
                      plan, g);
  if (rc || !p.join || p.grid < 2) return rc;
  return launch_pdl(tree_join_kernel<D, 1>, dim3((unsigned)((g.tokens * g.group + 7) / 8), (unsigned)(p.grid - 1)), dim3(2 * D), 0,
                    st, op, a, p.grid);
}

}  // namespace
