// Attention of new tokens over the paged cache, on the matrix cores.
//
// The rows of one key head are the new tokens times the query heads that share
// it, token-major, so that one pass over a key serves all of them.  Per tile of
// keys a wave computes, for 32 rows,
//   S^T = K Q^T   (A: keys, B: rows; 32x32x16)
//   O^T += V^T P^T
// In both products' result a lane holds one row (its column), so the running
// maximum, the sum and the rescaling of O are a lane's own, one exchange between
// the halves of the wave aside, and the exponentials of S^T are P^T in the order
// in which the second product takes them: its sum over keys may run in any order
// that A and B share, and V is read from LDS transposed in that order.  K and V
// go from their pages straight to LDS, a tile ahead, 16 bytes a lane, their
// 16-byte pieces permuted within a row so that neither read meets bank conflicts.
//
// Work is cut into items of (sequence, rows, range of keys), about as many as fill
// the device, from the lengths on the device: the host knows neither how long the
// sequences are nor how they differ.  A sequence in one part is stored at once;
// parts of a longer one go to the workspace and a second kernel joins them.
#include <algorithm>

#include "layer.h"

namespace moe {

template <class T>
struct Mfma32;
template <>
struct Mfma32<Bf16> {
  static constexpr uint32_t kExp = 0x7f80u;   // all ones: not finite
  static __device__ __forceinline__ f32x16 mul(u32x4_t a, u32x4_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    bf16x2_t v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};
template <>
struct Mfma32<F16> {
  static constexpr uint32_t kExp = 0x7c00u;
  static __device__ __forceinline__ f32x16 mul(u32x4_t a, u32x4_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNoMax = -3e38f;   // a row's maximum before its first key: finite, below all scores

struct AttnPlan {
  int tpt;       // tokens a tile
  int hpt;       // heads a token in a tile
  int hchunks;   // tiles that share a key head and its tokens
  int target;    // items wanted over all key heads; 0: no sequence is cut
  int least;     // fewest keys worth a part of their own
  int items;     // items a key head and chunk, at most
  float *po;     // [items][heads' chunks][rows][D] of parts
  float2 *pml;   // [items][heads' chunks][rows]: maximum (base 2) and sum
};

struct AttnItem {
  int seq, tile, part, parts;
  int first;     // item index of the tile's part 0
  bool live;
};

// Keys that the tiles of a sequence pass over, at most.
__device__ __forceinline__ int span_keys(const SeqSpan &sp, int window, int tpt) {
  return window > 0 ? (int)min((int64_t)sp.len, (int64_t)window + tpt + 63) : sp.len;
}

// The x-th item (by_tile: part 0 of the x-th tile) in order of sequences, tiles and
// parts; on one wave, 64 sequences a step.  Parts are as long as makes `target` of
// all of them, so at most target + tiles exist.
__device__ AttnItem find_item(const KvArgs &kv, const AttnPlan &p, int window, int x,
                              bool by_tile, int lane) {
  const int shares = kv.heads * p.hchunks;
  int64_t work = 0;
  if (p.target > 0) {
    for (int s0 = 0; s0 < kv.n_seqs; s0 += 64) {
      if (s0 + lane < kv.n_seqs) {
        const SeqSpan sp = kv_span(kv, s0 + lane);
        work += (int64_t)((sp.rows + p.tpt - 1) / p.tpt) * span_keys(sp, window, p.tpt);
      }
    }
    for (int m = 1; m < 64; m <<= 1) work += __shfl_xor(work, m);
  }
  const int64_t span =
      p.target > 0 ? max((int64_t)p.least, (work * shares + p.target - 1) / p.target) : INT32_MAX;
  AttnItem it;
  it.live = false;
  int done = 0, done_items = 0;
  for (int s0 = 0; s0 < kv.n_seqs; s0 += 64) {
    int tiles = 0, parts = 1;
    if (s0 + lane < kv.n_seqs) {
      const SeqSpan sp = kv_span(kv, s0 + lane);
      tiles = (sp.rows + p.tpt - 1) / p.tpt;
      parts = max(1, (int)((span_keys(sp, window, p.tpt) + span - 1) / span));
    }
    const int n = tiles * parts, c = by_tile ? tiles : n;
    int inc = c, inc_items = n;
    for (int m = 1; m < 64; m <<= 1) {
      const int u = __shfl_up(inc, m), v = __shfl_up(inc_items, m);
      if (lane >= m) inc += u, inc_items += v;
    }
    const uint64_t past = __ballot(x < done + inc);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      const int i = x - done - __shfl(inc - c, l);
      it.seq = s0 + l;
      it.parts = __shfl(parts, l);
      it.tile = by_tile ? i : i / it.parts;
      it.part = by_tile ? 0 : i % it.parts;
      it.first = done_items + __shfl(inc_items - n, l) + it.tile * it.parts;
      // (sums that wrapped, of starts that make no sense, end here)
      it.live = i >= 0 && it.tile < __shfl(tiles, l) && it.first >= 0 &&
                it.first <= p.items - it.parts;
      break;
    }
    done += __shfl(inc, 63);
    done_items += __shfl(inc_items, 63);
  }
  return it;
}

// A tile's rows and the keys that they see.
struct AttnTile {
  int row0, tokens;     // batch row of its first token
  int pos0;
  int start, end;       // keys that any row sees, start rounded down to 64
  int full0, full1;     // keys that every row sees
};
__device__ __forceinline__ AttnTile attn_tile(const SeqSpan &sp, int tile, int tpt, int window) {
  AttnTile t;
  const int tok0 = tile * tpt;
  t.row0 = sp.first + tok0;
  t.tokens = min(tpt, sp.rows - tok0);
  t.pos0 = sp.base + tok0;
  int lo0, hi0, lo1, hi1;
  seen_keys(t.pos0, sp.len, window, &lo0, &hi0);
  seen_keys(t.pos0 + t.tokens - 1, sp.len, window, &lo1, &hi1);
  t.start = lo0 & ~63;
  t.end = hi1;
  t.full0 = lo1;
  t.full1 = hi0;
  return t;
}

__device__ __forceinline__ float other_half(float v) {   // the value of lane ^ 32
  const uint32_t b = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// 16-byte piece c of row `row` stands at piece c ^ swz of that row.  K is read 16
// rows a phase at one piece, V 4 rows at four neighbouring ones.
template <int D>
__device__ __forceinline__ int swz_k(int row) {
  return D == 128 ? (row & 15) : ((row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int swz_v(int row) {
  return D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
}

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Bits [a, b) of a word of 64.
__device__ __forceinline__ uint64_t bit_range(int a, int b) {
  a = max(a, 0);
  b = min(b, 64);
  if (b <= a) return 0;
  return (~0ull >> (64 - (b - a))) << a;
}

// QW waves side by side on 32 rows each share the tiles of keys; or KW waves take
// every KW-th tile for the same 32 rows and are joined at the end.
template <class T, int D, int QW, int KW, int BK>
__global__ __launch_bounds__(64 * QW * KW, QW > 1 ? 2 : 1) void attn_kernel(AttnArgs a, AttnPlan p) {
  static_assert(QW == 1 || KW == 1, "one of the two");
  using M = Mfma32<T>;
  constexpr int kRows = 32 * QW;
  constexpr int kTileBytes = BK * D * 2;         // of K, and of V
  constexpr int kRowsPerLoad = 1024 / (2 * D);   // rows that one wave load brings
  constexpr int kLoads = kTileBytes / 1024 / QW; // a wave's loads of K, and of V
  constexpr int kPieces = D / 8;                 // 16-byte pieces a row
  __shared__ __align__(1024) char lds[KW * 4 * kTileBytes];   // [KW][2][K tile, V tile]
  __shared__ unsigned long long all_bad;
  const KvArgs &kv = a.kv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wq = QW > 1 ? wave : 0, wk = KW > 1 ? wave : 0;
  const int shares = kv.heads * p.hchunks;
  const int share = blockIdx.x % shares;
  // the last items first: a sequence's later rows see the most keys
  const int x = gridDim.x / shares - 1 - blockIdx.x / shares;
  const AttnItem it = find_item(kv, p, a.window, x, false, lane);
  if (!it.live) return;
  const SeqSpan sp = kv_span(kv, it.seq);
  if (!sp.ok && threadIdx.x == 0) flag_error_bits(kErrBadBatch);
  const AttnTile tl = attn_tile(sp, it.tile, p.tpt, a.window);
  const int hk = share / p.hchunks;
  const int group = a.heads / kv.heads;
  const int h0 = (share % p.hchunks) * p.hpt;

  // this lane's row
  const int r = wq * 32 + (lane & 31), hi = lane >> 5;
  const int tok = r / p.hpt, hh = h0 + r % p.hpt;
  const bool row_live = tok < tl.tokens && hh < group;
  const int t = tl.row0 + tok, h = hk * group + hh;
  int lo_key = 0, hi_key = 0;
  if (row_live) seen_keys(tl.pos0 + tok, sp.len, a.window, &lo_key, &hi_key);
  u32x4_t q[D / 16];
#pragma unroll
  for (int st = 0; st < D / 16; ++st) {
    q[st] = (u32x4_t){0, 0, 0, 0};
    if (row_live)
      q[st] = *reinterpret_cast<const u32x4_t *>(a.q + t * a.q_st + h * a.q_sh + 16 * st + 8 * hi);
  }

  // this part's keys
  const int n_keys = max(0, tl.end - tl.start);
  const int per = ((n_keys + it.parts - 1) / it.parts + BK * KW - 1) / (BK * KW) * (BK * KW);
  const int k0 = tl.start + it.part * per;
  const int k1 = min(tl.end, k0 + per);

  const int32_t *table = kv.table + (int64_t)it.seq * kv.width;
  auto entry_of = [&](int j0) {   // lane j: the page of key j0 + j, -1 past the end
    const int j = j0 + lane;
    return lane < BK && j < k1 ? table[j >> kv.page_shift] : -1;
  };
  auto valid_of = [&](int entry) { return __ballot(entry >= 0 && entry < kv.n_pages); };
  char *const mine = lds + wk * 4 * kTileBytes;
  // Rows of one load lie in one page (pages hold 16 rows or more, and tiles start at
  // a multiple of 32); a row with no page is read from page 0 and not used.
  auto fetch = [&](int j0, int entry, int buf) {
    char *const kb = mine + buf * 2 * kTileBytes, *const vb = kb + kTileBytes;
    const int sub = lane / kPieces, piece = lane % kPieces;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int n = i * QW + wq, row = n * kRowsPerLoad;
      int e = __builtin_amdgcn_readlane(entry, row);
      e = e >= 0 && e < kv.n_pages ? e : 0;
      const int64_t base =
          page_row(e, kv.n_pages, kv.heads, hk, kv.page_shift, j0 + row, D) + sub * D;
      const uint16_t *gk = kv.k + base + (piece ^ swz_k<D>(row + sub)) * 8;
      const uint16_t *gv = kv.v + base + (piece ^ swz_v<D>(row + sub)) * 8;
      __builtin_amdgcn_global_load_lds((global_void *)gk, (lds_void *)(kb + n * 1024), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((global_void *)gv, (lds_void *)(vb + n * 1024), 16, 0, 0);
    }
  };
  auto landed = [&] {   // this tile's bytes are in LDS, the other buffer is free
    if (QW > 1) {
      __syncthreads();
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  const float c = fmaxf(a.scale * kLog2e, 1e-37f);
  float m = kNoMax, l = 0.f;
  f32x16 o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[i][j] = 0.f;

  int j0 = k0 + wk * BK;
  int entry = j0 < k1 ? entry_of(j0) : -1, buf = 0;
  if (j0 < k1) fetch(j0, entry, 0);
  int entry_next = j0 + BK * KW < k1 ? entry_of(j0 + BK * KW) : -1;
  for (; j0 < k1; j0 += BK * KW, buf ^= 1) {
    landed();
    const uint64_t valid = valid_of(entry);
    const bool in_full = j0 >= tl.full0 && j0 + BK <= tl.full1;
    const bool full = in_full && (uint64_t)(valid << (64 - BK)) >> (64 - BK) == ~0ull >> (64 - BK);
    entry = entry_next;
    if (j0 + BK * KW < k1) {
      fetch(j0 + BK * KW, entry, buf ^ 1);
      entry_next = j0 + 2 * BK * KW < k1 ? entry_of(j0 + 2 * BK * KW) : -1;
    }
    const char *const kb = mine + buf * 2 * kTileBytes;
    char *const vb = mine + buf * 2 * kTileBytes + kTileBytes;

    uint64_t vis = 0;   // keys that this lane's row sees, where the tile is not full
    if (!full) {
      if ((valid | ~bit_range(0, k1 - j0)) != ~0ull && lane == 0) flag_error_bits(kErrBadBatch);
      vis = bit_range(lo_key - j0, min(hi_key, k1) - j0) & valid;
      // 0 * v is not 0 where v is not finite: such values, and what pages hold past the
      // sequence, become zero, and rows that do see one become NaN.
      uint64_t bad = 0;
      constexpr int kIters = BK * kPieces / (64 * QW);
#pragma unroll
      for (int i = 0; i < kIters; ++i) {
        const int at = (i * QW + wq) * 64 + lane, row = at / kPieces;
        u32x4_t w = *reinterpret_cast<u32x4_t *>(vb + at * 16);
        const bool use = (valid >> row) & 1;
        bool b = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t x0 = M::kExp, x1 = M::kExp << 16;
          uint32_t keep = ~0u;
          if ((w[e] & x0) == x0) keep &= 0xffff0000u;
          if ((w[e] & x1) == x1) keep &= 0x0000ffffu;
          b |= keep != ~0u;
          w[e] &= use ? keep : 0u;
        }
        b &= use;
        if (b || !use) *reinterpret_cast<u32x4_t *>(vb + at * 16) = w;
        const uint64_t lanes = __ballot(b);
#pragma unroll
        for (int k = 0; k < 64 / kPieces; ++k)
          if ((lanes >> (k * kPieces)) & ((1u << kPieces) - 1))
            bad |= 1ull << ((i * QW + wq) * (64 / kPieces) + k);
      }
      if (QW > 1) {   // each wave looked at a share of the rows
        if (threadIdx.x == 0) all_bad = 0;
        __syncthreads();
        if (lane == 0 && bad) atomicOr(&all_bad, (unsigned long long)bad);
        __syncthreads();
        bad = all_bad;
      }
      if (bad & vis) l = __builtin_nanf("");
    }

    // S^T: this lane's row against keys 32 kb + 8 (r / 4) + 4 hi + r % 4
    f32x16 s[BK / 32];
#pragma unroll
    for (int b = 0; b < BK / 32; ++b) {
      const int row = 32 * b + (lane & 31);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[b][e] = 0.f;
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        const u32x4_t kf = *reinterpret_cast<const u32x4_t *>(
            kb + row * (2 * D) + ((2 * st + hi) ^ swz_k<D>(row)) * 16);
        s[b] = M::mul(kf, q[st], s[b]);
      }
    }
    if (!full) {
      const uint64_t v = vis >> (4 * hi);
#pragma unroll
      for (int b = 0; b < BK / 32; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!((v >> (32 * b + 8 * (e / 4) + e % 4)) & 1)) s[b][e] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < BK / 32; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[b][e]);
    mx = fmaxf(mx, other_half(mx)) * c;
    // The maximum moves only when a score passes it by 2^8: exponentials up to that
    // are as exact, and most tiles rescale nothing.  A row's own scores decide.
    const bool moves = mx > m + 8.f;
    if (__any(moves)) {
      const float m1 = moves ? mx : m;
      const float f = __builtin_amdgcn_exp2f(m - m1);
      m = m1;
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] *= f;
    }
    u32x4_t pf[BK / 16];
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < BK / 32; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[b][e], c, -m));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[b][e + 1], c, -m));
        sum += p0 + p1;
        // rounded to the values' type for the matrix unit: half a step of a weight
        pf[2 * b + e / 8][(e % 8) / 2] = M::pack(p0, p1);
      }
    l += sum;
    // O^T: a step of 16 keys, in the order in which S^T left them
#pragma unroll
    for (int st = 0; st < BK / 16; ++st) {
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        // lanes 16 g + i of a half read 4 keys of 16 columns, lane i column i of them
        const int i = lane & 15;
        const int piece = 4 * d + 2 * ((lane >> 4) & 1) + (i & 3) / 2;
        u32x4_t vf;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int row = 16 * st + 8 * k + 4 * hi + i / 4;
          const char *at = vb + row * (2 * D) + (piece ^ swz_v<D>(row)) * 16 + (i & 1) * 8;
          const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4 *)(at));
          const uint2 u = __builtin_bit_cast(uint2, w);
          vf[2 * k] = u.x;
          vf[2 * k + 1] = u.y;
        }
        o[d] = M::mul(vf, pf[st], o[d]);
      }
    }
  }
  l += other_half(l);

  if (KW > 1) {   // the waves' keys joined on wave 0, one after the other
    for (int w = 1; w < KW; ++w) {
      __syncthreads();
      float *const box = reinterpret_cast<float *>(lds);
      if (wk == w) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) box[(i * 16 + e) * 64 + lane] = o[i][e];
        box[D / 2 * 64 + lane] = m;
        box[D / 2 * 64 + 64 + lane] = l;
      }
      __syncthreads();
      if (wk == 0) {
        const float m2 = box[D / 2 * 64 + lane], l2 = box[D / 2 * 64 + 64 + lane];
        const float mm = fmaxf(m, m2);
        const float f = __builtin_amdgcn_exp2f(m - mm), g = __builtin_amdgcn_exp2f(m2 - mm);
        m = mm;
        l = l * f + l2 * g;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[i][e] = o[i][e] * f + box[(i * 16 + e) * 64 + lane] * g;
      }
    }
    if (wk != 0) return;
  }
  if (!row_live) return;
  if (it.parts > 1) {
    const int64_t at = ((int64_t)x * shares + share) * kRows + r;
    if (hi == 0) p.pml[at] = make_float2(m, l);
    if (l == 0.f) return;   // no key of this part is seen
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4 *>(p.po + at * D + 32 * i + 2 * e + 4 * hi) =
            (f32x4){o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
    return;
  }
  float f = 1.f;
  if (a.sinks != nullptr) {
    const float sink = a.sinks[h] * kLog2e, mm = fmaxf(m, sink);
    f = __builtin_amdgcn_exp2f(m - mm);
    l = l * f + __builtin_amdgcn_exp2f(sink - mm);
  }
  f = l == 0.f ? 0.f : f / l;
  uint16_t *const out = a.out + ((int64_t)t * a.heads + h) * D;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<uint2 *>(out + 32 * i + 2 * e + 4 * hi) =
          make_uint2(M::pack(o[i][e] * f, o[i][e + 1] * f),
                     M::pack(o[i][e + 2] * f, o[i][e + 3] * f));
}

// Joins the parts of tiles that were cut.  D / 4 lanes hold a row; ALL: all of the
// workgroup's groups of lanes share one row's parts (few rows of many parts),
// otherwise each takes rows of its own.
template <class T, int D, int kRows, bool ALL>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, AttnPlan p) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ f32x4 acc[ALL ? 256 : 1];
  __shared__ float2 ml[kGroups];
  const KvArgs &kv = a.kv;
  const int lane = threadIdx.x & 63;
  const int shares = kv.heads * p.hchunks, share = blockIdx.y;
  const AttnItem it = find_item(kv, p, a.window, blockIdx.x, true, lane);
  if (!it.live || it.parts < 2) return;
  const SeqSpan sp = kv_span(kv, it.seq);
  const AttnTile tl = attn_tile(sp, it.tile, p.tpt, a.window);
  const int group = a.heads / kv.heads;
  const int g = threadIdx.x / kLanes, col = (threadIdx.x % kLanes) * 4;
  const int step = ALL ? gridDim.z : gridDim.z * kGroups;
  for (int r = ALL ? blockIdx.z : blockIdx.z * kGroups + g; r < p.tpt * p.hpt; r += step) {
    const int tok = r / p.hpt, hh = (share % p.hchunks) * p.hpt + r % p.hpt;
    if (tok >= tl.tokens) break;
    if (hh >= group) continue;
    const int h = (share / p.hchunks) * group + hh;
    const float sink = a.sinks != nullptr ? a.sinks[h] * kLog2e : -INFINITY;
    float m = kNoMax, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    // eight parts a step, so that their loads are on their way together
    const int stride = ALL ? kGroups : 1;
    for (int i0 = ALL ? g : 0; i0 < it.parts; i0 += 8 * stride) {
      float2 w[8];
      f32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = min(i0 + k * stride, it.parts - 1);
        const int64_t at = ((int64_t)(it.first + i) * shares + share) * kRows + r;
        w[k] = p.pml[at];
        v[k] = *reinterpret_cast<const f32x4 *>(p.po + at * D + col);
        if (i0 + k * stride >= it.parts) w[k] = make_float2(kNoMax, 0.f);
      }
      float mm = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) mm = fmaxf(mm, w[k].x);
      float f = __builtin_amdgcn_exp2f(m - mm);
      l *= f;
      o *= f;
      m = mm;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (w[k].y == 0.f) continue;   // (its columns were not written)
        f = __builtin_amdgcn_exp2f(w[k].x - m);
        l = fmaf(w[k].y, f, l);
        o += v[k] * f;
      }
    }
    if (ALL) {
      __syncthreads();
      acc[threadIdx.x] = o;
      if (col == 0) ml[g] = make_float2(m, l);
      __syncthreads();
      if (g != 0) continue;
      float mm = kNoMax;
      for (int k = 0; k < kGroups; ++k) mm = fmaxf(mm, ml[k].x);
      l = 0.f;
      o = (f32x4){0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < kGroups; ++k) {
        const float f = __builtin_amdgcn_exp2f(ml[k].x - mm);
        l = fmaf(ml[k].y, f, l);
        o += acc[k * kLanes + threadIdx.x] * f;
      }
      m = mm;
    }
    const float mm = fmaxf(m, sink);
    float f = __builtin_amdgcn_exp2f(m - mm);
    l = l * f + __builtin_amdgcn_exp2f(sink - mm);
    f = l == 0.f ? 0.f : f / l;
    uint16_t *const out = a.out + ((int64_t)(tl.row0 + tok) * a.heads + h) * D + col;
    *reinterpret_cast<uint2 *>(out) =
        make_uint2(Mfma32<T>::pack(o[0] * f, o[1] * f), Mfma32<T>::pack(o[2] * f, o[3] * f));
  }
}

bool attn_supported(int dim, int heads, int kv_heads) {
  return (dim == 64 || dim == 128) && heads % kv_heads == 0 && heads / kv_heads <= 64;
}

namespace {

// Rows of a tile: 256 (8 waves on the same keys) where a sequence brings that many
// rows a key head on average, otherwise 32 (2 waves on keys of their own).
struct AttnShape {
  bool wide;
  AttnPlan plan;
  int tiles;
};
constexpr int kWideRows = 256, kNarrowRows = 32;
AttnShape attn_shape(const KvArgs &kv, int heads) {
  AttnShape s;
  const int group = heads / kv.heads;
  s.wide = (int64_t)kv.total * group >= (int64_t)96 * kv.n_seqs;
  const int rows = s.wide ? kWideRows : kNarrowRows;
  s.plan.hpt = std::min(group, rows);
  s.plan.hchunks = (group + s.plan.hpt - 1) / s.plan.hpt;
  s.plan.tpt = rows / s.plan.hpt;
  // a tile holds a token at least
  s.tiles = (int)std::min<int64_t>(kv.total, (int64_t)kv.total / s.plan.tpt + kv.n_seqs);
  s.plan.target = s.wide ? 512 : 1024;
  s.plan.least = s.wide ? 512 : 256;
  const int shares = kv.heads * s.plan.hchunks;
  s.plan.items = s.tiles + (s.plan.target + shares - 1) / shares;
  return s;
}
size_t attn_part_bytes(const KvArgs &kv, const AttnShape &s) {
  return (size_t)s.plan.items * kv.heads * s.plan.hchunks * (s.wide ? kWideRows : kNarrowRows);
}

}  // namespace

// Launches count threads in 32 bits.
bool attn_fits(const KvArgs &kv, int heads) {
  const AttnShape s = attn_shape(kv, heads);
  const int64_t shares = (int64_t)kv.heads * s.plan.hchunks;
  return shares < 65536 && ((int64_t)s.plan.items * shares) < (1 << 23) && s.tiles < (1 << 24);
}

size_t attn_workspace(const KvArgs &kv, int heads) {
  const AttnShape s = attn_shape(kv, heads);
  return (attn_part_bytes(kv, s) * (kv.dim * 4 + 8) + 255) & ~(size_t)255;
}

template <class T, int D>
static void attn_go(const AttnArgs &a, void *ws, hipStream_t s) {
  AttnShape sh = attn_shape(a.kv, a.heads);
  const size_t n = attn_part_bytes(a.kv, sh);
  sh.plan.po = static_cast<float *>(ws);
  sh.plan.pml = reinterpret_cast<float2 *>(sh.plan.po + n * D);
  const int shares = a.kv.heads * sh.plan.hchunks;
  const dim3 g((unsigned)(sh.plan.items * shares));
  if (sh.wide) {
    constexpr int BK = 64;
    hipLaunchKernelGGL((attn_kernel<T, D, 8, 1, BK>), g, dim3(512), 0, s, a,
                       sh.plan);
    hipLaunchKernelGGL((attn_join_kernel<T, D, kWideRows, false>), dim3(sh.tiles, shares, 4),
                       dim3(256), 0, s, a, sh.plan);
  } else {
    constexpr int BK = D == 128 ? 32 : 64, KW = 2;
    hipLaunchKernelGGL((attn_kernel<T, D, 1, KW, BK>), g, dim3(64 * KW), 0, s,
                       a, sh.plan);
    hipLaunchKernelGGL((attn_join_kernel<T, D, kNarrowRows, true>),
                       dim3(sh.tiles, shares, sh.plan.hpt), dim3(256), 0, s, a, sh.plan);
  }
}

void launch_attn(const AttnArgs &a, int dtype, void *ws, hipStream_t s) {
  if (dtype == MOE_DTYPE_BF16) {
    if (a.kv.dim == 64) attn_go<Bf16, 64>(a, ws, s);
    else attn_go<Bf16, 128>(a, ws, s);
  } else {
    if (a.kv.dim == 64) attn_go<F16, 64>(a, ws, s);
    else attn_go<F16, 128>(a, ws, s);
  }
}

}  // namespace moe
