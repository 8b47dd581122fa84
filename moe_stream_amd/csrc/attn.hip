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
#include <type_traits>

#include "layer.h"

namespace moe {

// 16-bit products and conversions.
template <class T>
struct Mat;
template <>
struct Mat<Bf16> {
  static constexpr uint32_t kExp = 0x7f807f80u;    // exponents of a pair
  static constexpr uint32_t kCarry = 0x00800080u;  // carries out of an exponent of ones
  static __device__ __forceinline__ f32x16 mul(u32x4_t a, u32x4_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mul(u32x4_t a, u32x4_t b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    bf16x2_t v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};
template <>
struct Mat<F16> {
  static constexpr uint32_t kExp = 0x7c007c00u;
  static constexpr uint32_t kCarry = 0x04000400u;
  static __device__ __forceinline__ f32x16 mul(u32x4_t a, u32x4_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mul(u32x4_t a, u32x4_t b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
};

// A block of RB x RB results: RB lanes a row, 64 / RB groups of lanes g that hold 4
// neighbouring keys (or columns of O) in each 4 registers: value e of a lane is at
//   (4 * 64 / RB) * (e / 4) + 4 g + e % 4.
template <int RB>
struct Block;
template <>
struct Block<32> {
  typedef f32x16 acc;
};
template <>
struct Block<16> {
  typedef f32x4 acc;
};

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNoMax = -3e38f;   // a row's maximum before its first key: finite, below all scores

struct AttnPlan {
  int tpt;       // tokens a tile
  int hpt;       // heads a token in a tile
  int hchunks;   // tiles that share a key head and its tokens
  int target;    // items wanted over all key heads
  int least;     // fewest keys worth a part of their own
  int items;     // items a key head and chunk, at most
  float *po;     // [items][heads' chunks][rows][D] of parts
  float2 *pml;   // [items][heads' chunks][rows]: maximum (base 2) and sum
};

struct AttnItem {
  int seq, tile, part, parts;
  int first;     // item index of the tile's part 0
  SeqSpan sp;
  bool live;
};

// Keys that the tiles of a sequence pass over, at most.
MOE_HD int span_keys(const SeqSpan &sp, int window, int tpt) {
  const int64_t most = (int64_t)window + tpt + 63;
  return window > 0 && most < sp.len ? (int)most : sp.len;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_rows(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
// Sum over this and all lower lanes.
__device__ __forceinline__ int scan64(int v) {
  v += dpp_rows<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8
  v += dpp_rows<0x112, 0xf>(v);
  v += dpp_rows<0x114, 0xf>(v);
  v += dpp_rows<0x118, 0xf>(v);
  v += dpp_rows<0x142, 0xa>(v);   // the row before, then the half before
  v += dpp_rows<0x143, 0xc>(v);
  return v;
}

// The x-th item (by_tile: part 0 of the x-th tile) in order of sequences, tiles and
// parts; on one wave, 64 sequences a step.  A part is as long as makes `target` of
// all of them (in 32 bits, the same in every workgroup), so that at most target / shares
// + 1 + tiles exist.
__device__ AttnItem find_item(const KvArgs &kv, const AttnPlan &p, int window, int x,
                              bool by_tile, int lane) {
  const int shares = kv.heads * p.hchunks;
  const SeqSpan none = {0, 0, 0, 0, true};
  SeqSpan sp = none;
  float work = 0.f;
  for (int s0 = 0; s0 < kv.n_seqs; s0 += 64) {
    sp = s0 + lane < kv.n_seqs ? kv_span(kv, s0 + lane) : none;
    work += (float)((sp.rows + p.tpt - 1) / p.tpt) * (float)span_keys(sp, window, p.tpt);
  }
  work = group_sum<64>(work) * (float)shares;
  const int span = max(p.least, (int)fminf(work / (float)p.target, 2e9f) + 1);
  AttnItem it;
  it.live = false;
  int done = 0, done_items = 0;
  for (int s0 = 0; s0 < kv.n_seqs; s0 += 64) {
    if (kv.n_seqs > 64) sp = s0 + lane < kv.n_seqs ? kv_span(kv, s0 + lane) : none;
    const int tiles = (sp.rows + p.tpt - 1) / p.tpt;
    const int parts = max(1, (int)(((int64_t)span_keys(sp, window, p.tpt) + span - 1) / span));
    const int n = tiles * parts, c = by_tile ? tiles : n;
    const int inc_items = scan64(n), inc = by_tile ? scan64(c) : inc_items;
    const uint64_t past = __ballot(x < done + inc);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int i = x - done - of(inc - c);
      it.seq = s0 + l;
      it.parts = of(parts);
      it.tile = by_tile ? i : i / it.parts;
      it.part = by_tile ? 0 : i % it.parts;
      it.first = done_items + of(inc_items - n) + it.tile * it.parts;
      it.sp.first = of(sp.first);
      it.sp.rows = of(sp.rows);
      it.sp.len = of(sp.len);
      it.sp.base = of(sp.base);
      it.sp.ok = of(sp.ok);
      // (sums that wrapped, of starts that make no sense, end here)
      it.live = i >= 0 && it.tile < of(tiles) && it.first >= 0 && it.first <= p.items - it.parts;
      break;
    }
    done += __builtin_amdgcn_readlane(inc, 63);
    done_items += __builtin_amdgcn_readlane(inc_items, 63);
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

// Over the groups of lanes that hold one row.
template <int RB, class F>
__device__ __forceinline__ float over_groups(float v, F f) {
  uint32_t b = __float_as_uint(v);
  auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  if (RB == 16) {
    b = __float_as_uint(v);
    r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// 16-byte piece c of row `row` stands at piece c ^ swz of that row.  K is read 16
// rows a phase at one piece; V 4 rows a phase at four neighbouring pieces (RB 32) or
// 8 rows at two.
template <int D>
__device__ __forceinline__ int swz_k(int row) {
  return D == 128 ? (row & 15) : ((row >> 1) & 7);
}
template <int D, int RB>
__device__ __forceinline__ int swz_v(int row) {
  if (RB == 32) return D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
  return D == 128 ? (row & 7) << 1 : ((row >> 1) & 3) << 1;
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

// QW waves side by side on RB rows each share the tiles of keys; or KW waves take
// every KW-th tile for the same RB rows and are joined at the end.
//
// A step of the loop interleaves, instruction by instruction, the scores of tile i + 1
// with the exponentials of tile i, and the output of tile i with the maxima of tile
// i + 1: a wave's vector instructions run beside its own matrix instruction, but those of
// two waves of a SIMD do not (measured: a wave of products alone beside a wave of
// multiply-adds alone takes longer than one after the other), so the pairs are made here.
//
// Many rows are bound by instruction issue: 4096 rows of 32/4 heads of 128 over 8192 keys
// take 630 us, 1.09 PFLOP/s of the 1.24 that a large library product reaches, the matrix unit
// busy 53 % of the cycles, no bank conflicts; 9 chunks of 64/8 heads of 64 127 us, 690
// TFLOP/s, 33 % (two exponentials a product of 16 columns cost as much issue as it).  Few
// rows are bound by the bytes of the keys: 48 tokens over 64/8 heads of 64 read 435 MB in
// 82 us, 5.3 TB/s, what a large copy reaches, and join in 5 us; one token over 40000 keys
// reads 82 MB in 17 us (4.9 TB/s) and joins in 6.
template <class T, int D, int RB, int QW, int KW, int BK>
__global__ __launch_bounds__(64 * QW * KW, QW > 4 ? 2 : QW > 1 ? 3 : 1)
void attn_kernel(AttnArgs a, AttnPlan p) {
  static_assert(QW == 1 || KW == 1, "one of the two");
  using M = Mat<T>;
  using Acc = typename Block<RB>::acc;
  using Yes = std::true_type;
  using No = std::false_type;
  constexpr int NG = 64 / RB;                    // groups of lanes
  constexpr int AE = RB / NG;                    // values of a block a lane
  constexpr int kRows = RB * QW;
  constexpr int kTileBytes = BK * D * 2;         // of K, and of V
  constexpr int kRowsPerLoad = 1024 / (2 * D);   // rows that one wave load brings
  constexpr int kLoads = kTileBytes / 1024 / QW; // a wave's loads of K, and of V
  constexpr int kPieces = D / 8;                 // 16-byte pieces a row
  constexpr int kSteps = BK / (8 * NG);          // steps of 8 NG keys of the second product
  // Two tiles of K and of V a key wave, each an array of its own: loads to one are under
  // way while another is read, which the compiler waits for unless it tells them apart.
  __shared__ __align__(1024) char lds_k0[KW * kTileBytes], lds_k1[KW * kTileBytes];
  __shared__ __align__(1024) char lds_v0[KW * kTileBytes], lds_v1[KW * kTileBytes];
  __shared__ unsigned long long all_bad;
  const KvArgs &kv = a.kv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wq = QW > 1 ? wave : 0, wk = KW > 1 ? wave : 0;
  const int shares = kv.heads * p.hchunks;
  const int share = blockIdx.x % shares;
  // many rows: the last items first, since a sequence's later rows see the most keys
  const int x = QW > 1 ? gridDim.x / shares - 1 - blockIdx.x / shares : blockIdx.x / shares;
  const AttnItem it = find_item(kv, p, a.window, x, false, lane);
  if (!it.live) return;
  const SeqSpan sp = it.sp;
  if (!sp.ok && threadIdx.x == 0) flag_error_bits(kErrBadBatch);
  const AttnTile tl = attn_tile(sp, it.tile, p.tpt, a.window);
  const int hk = share / p.hchunks;

  // this part's keys
  const int n_keys = max(0, tl.end - tl.start);
  const int per = ((n_keys + it.parts - 1) / it.parts + BK * KW - 1) / (BK * KW) * (BK * KW);
  const int k0 = tl.start + it.part * per;
  const int k1 = min(tl.end, k0 + per);

  const int32_t *table = kv.table + (int64_t)it.seq * kv.width;
  // Lane j: the page of key j0 + j, past the end that of the last key.
  auto entry_of = [&](int j0) {
    return table[(uint32_t)min(j0 + lane, k1 - 1) >> kv.page_shift];
  };
  auto k_tile = [&](auto odd) {
    return (decltype(odd)::value ? lds_k1 : lds_k0) + wk * kTileBytes;
  };
  auto v_tile = [&](auto odd) {
    return (decltype(odd)::value ? lds_v1 : lds_v0) + wk * kTileBytes;
  };
  // Lane j: the address of key j0 + j's row of K; V's is as far from it as the arrays
  // are.  A row without a page is read from page 0, and not used.  Rows of one load lie
  // in one page (pages hold 16 rows or more, and tiles start at a multiple of 32), so a
  // load goes from its first row's address, and the lanes' places in it are the wave's own.
  const uint32_t page_bytes = (uint32_t)kv.heads << kv.page_shift << (D == 128 ? 8 : 7);
  const uint64_t k_base =
      reinterpret_cast<uint64_t>(kv.k) + ((uint64_t)(uint32_t)hk << kv.page_shift) * (2 * D);
  const int64_t v_from_k =
      reinterpret_cast<const char *>(kv.v) - reinterpret_cast<const char *>(kv.k);
  auto rows_of = [&](int j0, int entry) {
    const uint32_t e = (uint32_t)entry < (uint32_t)kv.n_pages ? (uint32_t)entry : 0u;
    const uint32_t in_page = (uint32_t)((j0 + lane) & ((1 << kv.page_shift) - 1)) * (2 * D);
    return (uint64_t)e * page_bytes + (k_base + in_page);
  };
  const int sub = lane / kPieces, piece = lane % kPieces;
  auto fetch = [&](bool is_v, uint64_t rows, int i, char *to) __attribute__((always_inline)) {
    const int n = i * QW + wq, row = n * kRowsPerLoad;
    const int swz = is_v ? swz_v<D, RB>(row + sub) : swz_k<D>(row + sub);
    uint32_t at = sub * (2 * D) + (piece ^ swz) * 16;
    asm("" : "+v"(at));   // (a 32-bit offset from a scalar address)
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)rows, row);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(rows >> 32), row);
    const char *src =
        reinterpret_cast<const char *>((((uint64_t)hi << 32) | lo) + (is_v ? v_from_k : 0));
    __builtin_amdgcn_global_load_lds((global_void *)(src + at), (lds_void *)(to + n * 1024), 16, 0,
                                     0);
  };

  // this lane's row
  const int group = a.heads / kv.heads;
  const int h0 = (share % p.hchunks) * p.hpt;
  const int r = wq * RB + lane % RB, g = lane / RB;
  const int tok = r / p.hpt, hh = h0 + r % p.hpt;
  const bool row_live = tok < tl.tokens && hh < group;
  const int t = tl.row0 + tok, h = hk * group + hh;
  u32x4_t q[D / (8 * NG)];
  auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int st = 0; st < D / (8 * NG); ++st) {
      q[st] = (u32x4_t){0, 0, 0, 0};
      if (row_live)
        q[st] = *reinterpret_cast<const u32x4_t *>(a.q + t * a.q_st + h * a.q_sh + 8 * NG * st +
                                                   8 * g);
    }
  };
  int lo_key = 0, hi_key = 0;
  if (row_live) seen_keys(tl.pos0 + tok, sp.len, a.window, &lo_key, &hi_key);

  // Keys of a tile that have a page; whether every row sees all of it; the keys that
  // this lane's row sees.
  auto valid_of = [&](int j0, int entry) {
    return __ballot((uint32_t)entry < (uint32_t)kv.n_pages) & bit_range(0, min(BK, k1 - j0));
  };
  auto is_full = [&](int j0, uint64_t valid) {
    return j0 >= tl.full0 && j0 + BK <= tl.full1 &&
           (uint64_t)(valid << (64 - BK)) >> (64 - BK) == ~0ull >> (64 - BK);
  };
  auto seen_of = [&](int j0, uint64_t valid) __attribute__((always_inline)) {
    if ((valid | ~bit_range(0, min(BK, k1 - j0))) != ~0ull && lane == 0)
      flag_error_bits(kErrBadBatch);
    return bit_range(lo_key - j0, hi_key - j0) & valid;
  };

  const float c = fmaxf(a.scale * kLog2e, 1e-37f);
  float m = kNoMax, l = 0.f;
  Acc o[D / RB];
  u32x4_t pf[kSteps];
#pragma unroll
  for (int i = 0; i < D / RB; ++i)
#pragma unroll
    for (int e = 0; e < AE; ++e) o[i][e] = 0.f;

  constexpr int kVals = BK / NG;                           // scores of a tile a lane
  constexpr int kMulS = BK / RB * (D / (8 * NG));          // products of the scores
  constexpr int kMulO = kSteps * (D / RB);                 // and of the output
  constexpr int kAheadK = QW == 4 ? 3 : 4, kAheadV = 3;    // operands read ahead
  typedef Acc Scores[BK / RB];

  // Where a lane reads in a tile, but for the operand's number: the pieces' permutation is
  // the same in every block of rows, so the number only flips bits of it.  (Held as one
  // value each: through long sums the compiler loses sight of which array is read.)
  const int i16 = lane & 15;
  int k_at = lane % RB * (2 * D) + (g ^ swz_k<D>(lane % RB)) * 16;
  int v_at = (4 * g + i16 / 4) * (2 * D) + (i16 & 1) * 8 +
             (((RB == 32 ? 2 * ((lane >> 4) & 1) : 0) + (i16 & 3) / 2) ^
              swz_v<D, RB>(4 * g + i16 / 4)) * 16;
  asm("" : "+v"(k_at), "+v"(v_at));
  auto k_operand = [&](const char *kb, int u) __attribute__((always_inline)) {
    const int b = u / (D / (8 * NG)), st = u % (D / (8 * NG));
    return *reinterpret_cast<const u32x4_t *>(kb + (k_at ^ (NG * st * 16)) + RB * b * (2 * D));
  };
  // 16 lanes read 4 keys of 16 columns, and lane i gets column i of them.
  auto v_operand = [&](const char *vb, int u) __attribute__((always_inline)) {
    const int st = u / (D / RB), d = u % (D / RB);
    u32x4_t vf;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4 *)(vb + (v_at ^ (d * RB * 2)) +
                                                      (2 * st + k) * 4 * NG * (2 * D)));
      const uint2 x2 = __builtin_bit_cast(uint2, w);
      vf[2 * k] = x2.x;
      vf[2 * k + 1] = x2.y;
    }
    return vf;
  };
  // Tile i's weights from its scores sc, beside tile i + 1's scores into sn (next).
  // A lane's row stands against keys 4 NG (e / 4) + 4 g + e % 4 of the tile.
  // The loads of what comes next, one after the other, go between the first products.
  auto weigh = [&](Scores &sc, Scores &sn, const char *kb, auto now, auto next, auto load)
      __attribute__((always_inline)) {
    constexpr bool kNow = decltype(now)::value, kNext = decltype(next)::value;
    constexpr int kEach = (2 * kLoads + kMulS - 1) / kMulS;   // loads a product
    u32x4_t kf[kAheadK];
    if constexpr (kNext) {
#pragma unroll
      for (int u = 0; u < kAheadK && u < kMulS; ++u) kf[u] = k_operand(kb, u);
    }
#pragma unroll
    for (int u = 0; u < kMulS; ++u) {
      if constexpr (kNow) {
#pragma unroll
        for (int k = 2 * (u * (kVals / 2) / kMulS); k < 2 * ((u + 1) * (kVals / 2) / kMulS);
             k += 2) {
          // rounded to the values' type for the matrix unit: half a step of a weight
          const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[k / AE][k % AE], c, -m));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[k / AE][k % AE + 1], c, -m));
          uint32_t w = M::pack(p0, p1);
          l += p0 + p1;
          asm volatile("" : "+v"(w), "+v"(l));   // (taken here, not where they are used)
          pf[k / 8][(k % 8) / 2] = w;
        }
      }
      if constexpr (kNext) {
        const int b = u / (D / (8 * NG)), st = u % (D / (8 * NG));
        sn[b] = M::mul(kf[u % kAheadK], q[st], st == 0 ? Acc{} : sn[b]);
        if (u + kAheadK < kMulS) kf[u % kAheadK] = k_operand(kb, u + kAheadK);
#pragma unroll
        for (int k = u * kEach; k < (u + 1) * kEach && k < 2 * kLoads; ++k) load(k);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto hide = [&](Scores &sn, uint64_t vis) __attribute__((always_inline)) {
    const uint64_t v = vis >> (4 * g);
#pragma unroll
    for (int b = 0; b < BK / RB; ++b)
#pragma unroll
      for (int e = 0; e < AE; ++e)
        if (!((v >> (RB * b + 4 * NG * (e / 4) + e % 4)) & 1)) sn[b][e] = -INFINITY;
  };
  // The output of tile i, keys in the order in which the scores left them (a step takes
  // two runs of 4 keys a group), beside the largest next score.
  auto output = [&](const char *vb, Scores &sn, auto next) __attribute__((always_inline)) {
    constexpr bool kNext = decltype(next)::value;
    u32x4_t vf[kAheadV];
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kAheadV && u < kMulO; ++u) vf[u] = v_operand(vb, u);
#pragma unroll
    for (int u = 0; u < kMulO; ++u) {
      const int st = u / (D / RB), d = u % (D / RB);
      o[d] = M::mul(vf[u % kAheadV], pf[st], o[d]);
      if (u + kAheadV < kMulO) vf[u % kAheadV] = v_operand(vb, u + kAheadV);
      if constexpr (kNext) {
#pragma unroll
        for (int k = u * kVals / kMulO; k < (u + 1) * kVals / kMulO; ++k)
          mx = fmaxf(mx, sn[k / AE][k % AE]);
      }
      asm volatile("" : "+v"(mx));   // (here, between the products)
      __builtin_amdgcn_sched_barrier(0);
    }
    return mx;
  };
  // Where a row does not see the whole tile, 0 * v has to be 0 whatever v is: values that
  // are not finite become zero in LDS first, and rows that do see one become NaN.
  auto scrub = [&](char *vb, uint64_t vis) __attribute__((always_inline)) {
    constexpr int kIters = BK * kPieces / (64 * QW);
    uint64_t bad = 0;   // keys with such a value
    if (QW > 1 && threadIdx.x == 0) all_bad = 0;
    if (QW > 1) __syncthreads();
#pragma unroll 1
    for (int i = 0; i < kIters; ++i) {
      const int at = (i * QW + wq) * 64 + lane;
      u32x4_t w = *reinterpret_cast<u32x4_t *>(vb + at * 16);
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t odd = ((w[e] & M::kExp) + M::kCarry) & 0x80008000u;   // sign bits
        any |= odd;
        w[e] &= ~((odd >> 15) * 0xffffu);
      }
      const uint64_t lanes = __ballot(any != 0);
      if (lanes == 0) continue;
      *reinterpret_cast<u32x4_t *>(vb + at * 16) = w;
#pragma unroll
      for (int k = 0; k < 64 / kPieces; ++k)
        if ((lanes >> (k * kPieces)) & ((1u << kPieces) - 1))
          bad |= 1ull << ((i * QW + wq) * (64 / kPieces) + k);
    }
    if (QW > 1) {   // each wave looked at a share of the rows
      if (lane == 0 && bad) atomicOr(&all_bad, (unsigned long long)bad);
      __syncthreads();
      bad = all_bad;
    }
    if (bad & vis) l = __builtin_nanf("");
  };
  auto largest = [&](Scores &sn) __attribute__((always_inline)) {
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVals; ++k) mx = fmaxf(mx, sn[k / AE][k % AE]);
    return mx;
  };
  // The maximum moves only when a score passes it by 2^8: exponentials up to that are
  // as exact, and most tiles rescale nothing.  A row's own scores decide.
  auto rescale = [&](float mx) __attribute__((always_inline)) {
    mx = over_groups<RB>(mx, [](float u, float v) { return fmaxf(u, v); }) * c;
    const bool moves = mx > m + 8.f;
    if (__any(moves)) {
      const float m1 = moves ? mx : m;
      const float f = __builtin_amdgcn_exp2f(m - m1);
      m = m1;
      l *= f;
#pragma unroll
      for (int i = 0; i < D / RB; ++i)
#pragma unroll
        for (int e = 0; e < AE; ++e) o[i][e] *= f;
    }
  };

  // This wave's tiles: n of them, tile i at key_of(i).  Before step i, the keys of tile
  // i + 1 and the values of tile i land; what step i - 1 read is free for the next.
  auto key_of = [&](int i) { return k0 + (wk + i * KW) * BK; };
  const int n = (max(0, k1 - k0 - wk * BK) + BK * KW - 1) / (BK * KW);
  int e0 = 0, e1 = 0;
  if (n > 0) e0 = entry_of(key_of(0)), e1 = entry_of(key_of(1));
  load_q();
  // A workgroup barrier alone does not wait for loads that go to LDS.  (As a builtin, so
  // that the compiler knows of the wait and adds none of its own before the reads.)
  auto landed = [&]() __attribute__((always_inline)) {
    issue_order_fence();
    __builtin_amdgcn_s_waitcnt(loads_left(0));
    if (QW > 1) __syncthreads();
    issue_order_fence();
  };
  Scores s0, s1;
  bool full = true;
  uint64_t vis = 0, valid_next = 0;
  uint64_t rows = 0;   // of tile i + 1
  if (n > 0) {
    const uint64_t first = rows_of(key_of(0), e0);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) fetch(false, first, k, k_tile(No()));
    landed();
    const uint64_t valid = valid_of(key_of(0), e0);
    rows = rows_of(key_of(1), e1);
    valid_next = valid_of(key_of(1), e1);
    e0 = entry_of(key_of(2));
    weigh(s0, s0, k_tile(No()), No(), Yes(), [&](int k) __attribute__((always_inline)) {
      if (k < kLoads) fetch(true, first, k, v_tile(No()));
      else fetch(false, rows, k - kLoads, k_tile(Yes()));
    });
    full = is_full(key_of(0), valid);
    if (!full) hide(s0, vis = seen_of(key_of(0), valid));
    rescale(largest(s0));
  }
  auto step = [&](int i, Scores &sc, Scores &sn, auto odd, auto next)
      __attribute__((always_inline)) {
    constexpr bool kNext = decltype(next)::value;
    using Other = std::bool_constant<!decltype(odd)::value>;   // tile i + 1's buffers
    landed();
    const uint64_t valid = valid_next;
    const uint64_t rows_v = rows;
    if constexpr (kNext) {   // (tiles past the end are some tile's again, not used)
      rows = rows_of(key_of(i + 2), e0);
      valid_next = valid_of(key_of(i + 2), e0);
      e0 = entry_of(key_of(i + 3));
    }
    if (!full) scrub(v_tile(odd), vis);
    weigh(sc, sn, k_tile(Other()), Yes(), next, [&](int k) __attribute__((always_inline)) {
      if (k < kLoads) fetch(true, rows_v, k, v_tile(Other()));
      else fetch(false, rows, k - kLoads, k_tile(odd));
    });
    bool full_next = true;
    uint64_t vis_next = 0;
    if constexpr (kNext) {
      full_next = is_full(key_of(i + 1), valid);
      if (!full_next) hide(sn, vis_next = seen_of(key_of(i + 1), valid));
    }
    const float mx = output(v_tile(odd), sn, next);
    if constexpr (kNext) rescale(mx);
    full = full_next;
    vis = vis_next;
  };
  int i = 0;
  for (; i + 2 < n; i += 2) {
    step(i, s0, s1, No(), Yes());
    step(i + 1, s1, s0, Yes(), Yes());
  }
  if (i + 1 < n) {
    step(i, s0, s1, No(), Yes());
    step(i + 1, s1, s0, Yes(), No());
  } else if (i < n) {
    step(i, s0, s1, No(), No());
  }
  __builtin_amdgcn_s_waitcnt(loads_left(0));   // (LDS is used for something else, or given back)
  l = over_groups<RB>(l, [](float u, float v) { return u + v; });

  if (KW > 1) {   // the waves' keys joined on wave 0, in order
    constexpr int kBox = D / NG * 64;
    float *const box = reinterpret_cast<float *>(lds_k0) + lane;
    float2 *const stat = reinterpret_cast<float2 *>(lds_v0) + lane;
    static_assert((KW - 1) * kBox * 4 <= KW * kTileBytes, "the boxes fit the tiles");
    __syncthreads();
    if (wk > 0) {
#pragma unroll
      for (int i = 0; i < D / NG; ++i) box[(wk - 1) * kBox + i * 64] = o[i / AE][i % AE];
      stat[(wk - 1) * 64] = make_float2(m, l);
    }
    __syncthreads();
    if (wk != 0) return;
    for (int w = 0; w < KW - 1; ++w) {
      const float2 s2 = stat[w * 64];
      const float mm = fmaxf(m, s2.x);
      const float f = __builtin_amdgcn_exp2f(m - mm), f2 = __builtin_amdgcn_exp2f(s2.x - mm);
      m = mm;
      l = l * f + s2.y * f2;
#pragma unroll
      for (int i = 0; i < D / NG; ++i)
        o[i / AE][i % AE] = o[i / AE][i % AE] * f + box[w * kBox + i * 64] * f2;
    }
  }
  if (!row_live) return;
  if (it.parts > 1) {
    const int64_t at = ((int64_t)x * shares + share) * kRows + r;
    if (g == 0) p.pml[at] = make_float2(m, l);
    if (l == 0.f) return;   // no key of this part is seen
#pragma unroll
    for (int i = 0; i < D / RB; ++i)
#pragma unroll
      for (int e = 0; e < AE; e += 4)
        *reinterpret_cast<f32x4 *>(p.po + at * D + RB * i + NG * e + 4 * g) =
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
  for (int i = 0; i < D / RB; ++i)
#pragma unroll
    for (int e = 0; e < AE; e += 4)
      *reinterpret_cast<uint2 *>(out + RB * i + NG * e + 4 * g) =
          make_uint2(M::pack(o[i][e] * f, o[i][e + 1] * f),
                     M::pack(o[i][e + 2] * f, o[i][e + 3] * f));
}

// Joins the parts of tiles that were cut.  D / 4 lanes hold a row's columns; up to 8
// parts go to one such group, whose loads are on their way together, and more to
// several groups, joined through LDS.  The workgroups z of a tile share its rows.
constexpr int kJoinThreads = 512;
template <class T, int D>
__global__ __launch_bounds__(kJoinThreads) void attn_join_kernel(AttnArgs a, AttnPlan p, int rows) {
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes;
  __shared__ f32x4 acc[kJoinThreads];
  __shared__ float2 ml[kGroups];
  const KvArgs &kv = a.kv;
  const int lane = threadIdx.x & 63;
  const int shares = kv.heads * p.hchunks, share = blockIdx.y;
  const AttnItem it = find_item(kv, p, a.window, blockIdx.x, true, lane);
  if (!it.live || it.parts < 2) return;
  const AttnTile tl = attn_tile(it.sp, it.tile, p.tpt, a.window);
  const int group = a.heads / kv.heads;
  const int g = threadIdx.x / kLanes, col = (threadIdx.x % kLanes) * 4;
  int each = 1;   // groups a row
  while (each < kGroups && 8 * each < it.parts) each *= 2;
  const int side = kGroups / each, mine = g % each;   // rows at a time
  for (int r0 = blockIdx.z * side; r0 < tl.tokens * p.hpt; r0 += gridDim.z * side) {
    const int r = r0 + g / each;
    const int tok = r / p.hpt, hh = (share % p.hchunks) * p.hpt + r % p.hpt;
    const bool live = tok < tl.tokens && hh < group;
    float m = kNoMax, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = mine; live && i0 < it.parts; i0 += 8 * each) {
      float2 w[8];
      f32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = min(i0 + k * each, it.parts - 1);
        const int64_t at = ((int64_t)(it.first + i) * shares + share) * rows + r;
        w[k] = p.pml[at];
        v[k] = *reinterpret_cast<const f32x4 *>(p.po + at * D + col);
        if (i0 + k * each >= it.parts) w[k] = make_float2(kNoMax, 0.f);
      }
      float mm = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) mm = fmaxf(mm, w[k].x);
      const float f = __builtin_amdgcn_exp2f(m - mm);
      l *= f;
      o *= f;
      m = mm;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = __builtin_amdgcn_exp2f(w[k].x - m);
        l = fmaf(w[k].y, f, l);
        // (a part of no seen key wrote no columns)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = w[k].y == 0.f ? o[e] : fmaf(v[k][e], f, o[e]);
      }
    }
    if (each > 1) {
      __syncthreads();
      acc[threadIdx.x] = o;
      if (col == 0) ml[g] = make_float2(m, l);
      __syncthreads();
      if (mine == 0) {
        float mm = m;
        for (int k = 1; k < each; ++k) mm = fmaxf(mm, ml[g + k].x);
        float f = __builtin_amdgcn_exp2f(m - mm);
        l *= f;
        o *= f;
        for (int k = 1; k < each; ++k) {
          f = __builtin_amdgcn_exp2f(ml[g + k].x - mm);
          l = fmaf(ml[g + k].y, f, l);
          o += acc[threadIdx.x + k * kLanes] * f;
        }
        m = mm;
      }
    }
    if (mine != 0 || !live) continue;
    const int h = (share / p.hchunks) * group + hh;
    if (a.sinks != nullptr) {
      const float sink = a.sinks[h] * kLog2e, mm = fmaxf(m, sink);
      const float f = __builtin_amdgcn_exp2f(m - mm);
      l = l * f + __builtin_amdgcn_exp2f(sink - mm);
      o *= f;
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    uint16_t *const out = a.out + ((int64_t)(tl.row0 + tok) * a.heads + h) * D + col;
    *reinterpret_cast<uint2 *>(out) =
        make_uint2(Mat<T>::pack(o[0] * f, o[1] * f), Mat<T>::pack(o[2] * f, o[3] * f));
  }
}

bool attn_supported(int dim, int heads, int kv_heads) {
  return (dim == 64 || dim == 128) && heads % kv_heads == 0 && heads / kv_heads <= 64;
}

namespace {

// Rows of a tile: 256 (128 for heads of 64) on waves that share their keys, where a
// sequence brings more than 64 rows a key head on average, otherwise 32 or 16 on waves
// with keys of their own.  8 sequences of 9000 keys, 32/4 heads of 128: 16 rows each 37.8 us
// on tiles of 16, 51 on 256; 24 rows 40.5 on 32 and 44.7 on 16; 64 rows 45.8 on 32, 54.7 on
// 256 and 65 on 16; 80 rows 71 on 32 and 57 on 256; 192 rows 117 and 71.  64/8 heads of 64 go
// alike (80 rows: 63.6 and 44.3 us).
//   Heads of 64 leave registers for three waves a SIMD with tiles of 128 rows: 9 chunks of
// 64/8 heads 127 us, with 256 rows 139; 4096 rows over 12288 keys 770 and 794.  Heads of 128
// do not: 4096 rows of 32/4 heads over 8192 keys take 620 us with 256 rows, 637 with 128.
//   target: items enough to even out the lengths, few enough that joining them is small
// (48 single tokens, 64/8 heads of 64: 512 items 89 us, 640 91, 768 86, 1024 95; 8 x 8 tokens,
// tiles of 32: 768 47.5, 1024 44.7).
//   least: shorter parts would gain little (4 tokens over 3000 keys: 13.0 us with parts from
// 128 keys, 15.2 from 256), and would give windows of 128 keys a second launch.
struct AttnShape {
  int rows;
  AttnPlan plan;
  int tiles;
  bool cut;   // whether a sequence may come in parts
};
constexpr int kWaves64 = 4, kWaves128 = 8;   // of 32 rows
AttnShape attn_shape(const KvArgs &kv, int heads, int window) {
  AttnShape s;
  const int group = heads / kv.heads;
  const int64_t mean = ((int64_t)kv.total * group + kv.n_seqs - 1) / kv.n_seqs;
  const bool wide = mean > 64;
  s.rows = wide ? 32 * (kv.dim == 64 ? kWaves64 : kWaves128) : mean > 16 ? 32 : 16;
  s.plan.hpt = std::min(group, s.rows);
  s.plan.hchunks = (group + s.plan.hpt - 1) / s.plan.hpt;
  s.plan.tpt = s.rows / s.plan.hpt;
  // a tile holds a token at least
  s.tiles = (int)std::min<int64_t>(kv.total, (int64_t)kv.total / s.plan.tpt + kv.n_seqs);
  s.plan.target = s.rows == 256 ? 512 : s.rows == 32 ? 1024 : 768;
  s.plan.least = wide ? 512 : 256;
  SeqSpan longest = {};
  longest.len = kv.width << kv.page_shift;
  s.cut = span_keys(longest, window, s.plan.tpt) > s.plan.least;
  const int shares = kv.heads * s.plan.hchunks;
  s.plan.items = s.tiles + s.plan.target / shares + 2;
  return s;
}
size_t attn_part_rows(const KvArgs &kv, const AttnShape &s) {
  return (size_t)s.plan.items * kv.heads * s.plan.hchunks * s.rows;
}

}  // namespace

// Launches count threads in 32 bits.
bool attn_fits(const KvArgs &kv, int heads, int window) {
  const AttnShape s = attn_shape(kv, heads, window);
  const int64_t shares = (int64_t)kv.heads * s.plan.hchunks;
  return shares < 65536 && ((int64_t)s.plan.items * shares) < (1 << 23) && s.tiles < (1 << 24);
}

size_t attn_workspace(const KvArgs &kv, int heads, int window) {
  const AttnShape s = attn_shape(kv, heads, window);
  return s.cut ? (attn_part_rows(kv, s) * (kv.dim * 4 + 8) + 255) & ~(size_t)255 : 0;
}

template <class T, int D, int RB, int QW, int KW, int BK>
static void attn_run(const AttnArgs &a, const AttnShape &sh, hipStream_t s) {
  const int shares = a.kv.heads * sh.plan.hchunks;
  hipLaunchKernelGGL((attn_kernel<T, D, RB, QW, KW, BK>),
                     dim3((unsigned)(sh.plan.items * shares)), dim3(64 * QW * KW), 0, s, a,
                     sh.plan);
  if (!sh.cut) return;
  // (few tiles have many parts, and then a workgroup a row; many have few)
  const int z = std::min(sh.plan.tpt * sh.plan.hpt, std::max(1, 512 / (sh.tiles * shares)));
  hipLaunchKernelGGL((attn_join_kernel<T, D>), dim3(sh.tiles, shares, z), dim3(kJoinThreads), 0,
                     s, a, sh.plan, sh.rows);
}

template <class T, int D>
static void attn_go(const AttnArgs &a, void *ws, hipStream_t s) {
  AttnShape sh = attn_shape(a.kv, a.heads, a.window);
  sh.plan.po = static_cast<float *>(ws);
  sh.plan.pml = reinterpret_cast<float2 *>(sh.plan.po + attn_part_rows(a.kv, sh) * D);
  constexpr int KW = D == 128 ? 1 : 2;
  if (sh.rows > 32) attn_run<T, D, 32, D == 64 ? kWaves64 : kWaves128, 1, 64>(a, sh, s);
  else if (sh.rows == 32) attn_run<T, D, 32, 1, KW, 32>(a, sh, s);
  else attn_run<T, D, 16, 1, KW, 32>(a, sh, s);
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
