// Attention of new tokens over a key / value cache (kvq.h): one token (a decode step), a chain (a
// piece of a prompt) or a tree of drafted tokens, whose keys and values stand in the slots behind
// the row's context.
//
//   o_t = sum_j p_tj v_j,  p_t = softmax_j(scale q_t . k_j)   over the context slots j < start that
//   the mask keeps and the new tokens u that token t sees.
//
// One pass over the keys with the running maximum and sum of each row.  A wave takes tiles of 32
// slots:
//   S^T [32 slots x 32 rows] = K . Q^T   (v_mfma_f32_32x32x16_bf16; rows are (token, q head of the
//                                         KV head's group), so a group and a tree share each key)
//   O^T [D x 32 rows] += V^T . P^T
// The score tile's row order is chosen so that a lane's 16 scores are those of slots 16 u + 8 h + i
// (h = lane / 32): exactly the operand that the second product wants from that lane, so the
// probabilities never leave its registers.
//   The running maximum lives in powers of two: p = 2^(s scale log2(e) - m).  A slot's two scales are
// held one a lane and reach the 16 scores as row broadcasts, an operand form that costs nothing.
#include <utility>

#include "engine_internal.h"
#include "kvq.h"

namespace mtts {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// context, new tokens and visible slots of row b.  New token u stands at slot start + u, if there is one:
// behind the cache's end there is none, nor before slot 0 (a negative start leaves no context)
struct RowLen {
  int start, n, nk;
};
__device__ __forceinline__ RowLen row_len(const AttnKvArgs& a, int b) {
  RowLen r;
  r.start = min(max(a.start[b], -(1 << 30)), a.c.slots);
  r.n = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  r.nk = (int)max((int64_t)0, min((int64_t)r.start + r.n, (int64_t)a.c.slots));
  return r;
}

// Work.  The batch's rows differ in length and only the device knows by how much, so the blocks of a KV
// head (and row block) share out the tiles of all rows as one run: block x takes tiles x share ..
// (x + 1) share - 1 of it, in segments of one row each.  A row that lies in one block is finished there;
// of a longer one every block leaves a partial (m, l, o), in slot 2 x + 1 if the row begins in it and
// 2 x if it began before, and the join adds them up in order: the first block and the number of blocks of
// each row stand at the head of the workspace.  share 0: a block a row, nothing to join.
// A segment more costs a block about SEG tiles (its loads start anew), so a row counts for SEG more.
// Where a row is cut follows from the lengths of all rows, and so do the maxima that its parts start with and
// the last bits of its result (cuts that each row had for itself would leave the blocks uneven).
__device__ __forceinline__ int tiles_of(const RowLen& r) { return r.n ? max(1, (r.nk + 31) >> 5) : 0; }
// sum up to and with this lane: rows of 16 lanes by shifts, then the rows' sums by broadcasts
__device__ __forceinline__ int wave_iscan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // lane 15 of rows 0 and 2 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // lane 31 into rows 2 and 3
  return v;
}
struct Seg {
  int b, t0, t1, slot;  // tiles [t0, t1) of row b; slot -1: the whole row
  RowLen len;
};
template <int SEG>
struct Segments {
  const AttnKvArgs& a;
  RowLen r;
  int64_t lo, hi;
  uint64_t hit;
  int x, b0, beg, end, off, lane;
  bool direct;

  __device__ __forceinline__ void rows_at(int from) {  // 64 rows: their lengths, their places in the run
    b0 = from;
    r = b0 + lane < a.B ? row_len(a, b0 + lane) : RowLen{0, 0, 0};
    const int t = tiles_of(r), run = t ? t + SEG : 0;
    end = off + wave_iscan(run);
    beg = end - t;
  }
  __device__ __forceinline__ Segments(const AttnKvArgs& a, int NS, int least, int x, bool head)
      : a(a), r{0, 0, 0}, hit(1), x(x), b0(0), beg(0), end(0), off(0), lane(threadIdx.x & 63), direct(least == 0) {
    if (direct) return;
    int total = 0;
    for (int from = (a.B - 1) & ~63; from >= 0; from -= 64) {
      rows_at(from);
      total += __builtin_amdgcn_readlane(end, 63);
    }
    const int share = max(least, (total + NS - 1) / NS);
    lo = (int64_t)x * share;
    hi = lo + share;
    if (head)
      for (int from = 0; from < a.B; from += 64) {
        if (from) rows_at(from);
        if (threadIdx.x < 64 && b0 + lane < a.B) {
          const int x0 = beg / share, ns = beg < end ? (end - 1) / share - x0 + 1 : 0;
          *reinterpret_cast<int2*>(a.part + 2 * (b0 + lane)) = make_int2(x0, ns);
        }
        off = __builtin_amdgcn_readlane(end, 63);
      }
    off = 0;
    if (head && a.B > 64) rows_at(0);
    hit = __ballot(beg < end && beg < hi && end > lo);
  }
  __device__ __forceinline__ bool next(Seg& g) {
    if (direct) {
      if (!hit) return false;
      hit = 0;
      g = Seg{x, 0, INT_MAX, -1, row_len(a, x)};
      return true;
    }
    while (!hit) {
      off = __builtin_amdgcn_readlane(end, 63);
      if (b0 + 64 >= a.B || off >= hi) return false;
      rows_at(b0 + 64);
      hit = __ballot(beg < end && beg < hi && end > lo);
    }
    const int f = __ffsll((unsigned long long)hit) - 1;
    hit &= hit - 1;
    const int sb = __builtin_amdgcn_readlane(beg, f), se = __builtin_amdgcn_readlane(end, f);
    g.b = b0 + f;
    g.t0 = (int)max(lo, (int64_t)sb) - sb;
    g.t1 = (int)min(hi, (int64_t)se) - sb;
    g.slot = sb >= lo && se <= hi ? -1 : 2 * x + (sb >= lo ? 1 : 0);
    g.len = RowLen{__builtin_amdgcn_readlane(r.start, f), __builtin_amdgcn_readlane(r.n, f), __builtin_amdgcn_readlane(r.nk, f)};
    return true;
  }
};
// f of each segment of block x.  Unsplit launches (SPLIT false) have a kernel of their own: with the sharing
// out in it too it is twice the code, whose fetching a short call waits for (one token over 389 bf16 slots
// 10.3 us and not 8), and the loop over 32 rows of 2,063 to 4,000 slots took 94 us and not 81.
template <bool SPLIT, int SEG, class F>
__device__ __forceinline__ void for_segments(const AttnKvArgs& a, int NS, int least, int x, bool head, F&& f) {
  if constexpr (SPLIT) {
    Segments<SEG> it(a, NS, least, x, head);
    for (Seg sg; it.next(sg);) f(sg);
  } else {
    f(Seg{x, 0, INT_MAX, -1, row_len(a, x)});
  }
}
// floats at the head of the workspace
__host__ __device__ __forceinline__ size_t head_floats(int B) { return ((size_t)2 * B + 63) / 64 * 64; }

// eight codes as bf16: exact, both types have at most 8 significant bits
template <int KT>
__device__ __forceinline__ bf16x8 frag8(uint32_t lo, uint32_t hi) {
  union {
    uint32_t w[4];
    bf16x2 h[4];
    bf16x8 v;
  } o;
  if constexpr (KT == KV_E4M3) {
    o.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    o.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    o.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    o.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  } else {
    const uint32_t w[2] = {lo, hi};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = (float)(int)__builtin_amdgcn_sbfe(w[i >> 1], 16 * (i & 1), 8);
      const float y = (float)(int)__builtin_amdgcn_sbfe(w[i >> 1], 16 * (i & 1) + 8, 8);
      o.w[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);  // the high halves
    }
  }
  return o.v;
}

// compile-time unrolled: the lane of a row broadcast is part of the instruction
template <int N, class F, int... I>
__device__ __forceinline__ void unrolled_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void unrolled(F&& f) {
  unrolled_impl<N>(f, std::make_integer_sequence<int, N>{});
}
// lane i's value of each row of 16 lanes, in all of the row
template <int I>
__device__ __forceinline__ float row_bcast(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x150 + I, 0xf, 0xf, true));
}

// Of the 8 slots from k0 on (bits): live, the context slots that the mask keeps and the new tokens'
// (every other slot's bytes are anything); fresh, the new tokens' alone.
struct Live8 {
  uint32_t live, fresh;
};
__device__ __forceinline__ Live8 live8(const AttnKvArgs& a, int b, const RowLen& len, int k0) {
  const int cn = min(max(len.start - k0, 0), 8), ln = min(max(len.nk - k0, 0), 8);
  uint32_t ctx = (1u << cn) - 1;
  const uint32_t fresh = ((1u << ln) - 1) & ~ctx;
  if (a.mask) {
    const uint2 mk = *reinterpret_cast<const uint2*>(a.mask + (size_t)b * a.c.slots + k0);
    uint32_t mb = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      mb |= ((mk.x >> (8 * i)) & 0xff ? 1u << i : 0) | ((mk.y >> (8 * i)) & 0xff ? 16u << i : 0);
    ctx &= mb;
  }
  return {ctx | fresh, fresh};
}

// A lane's row: its token and, for a tree, what the token sees.
struct Row {
  int tok;
  uint64_t tw;
};
// the 16 slots of lane half h in a tile that may hold slots the row does not see: bit 8 u + i for slot
// 16 u + 8 h + i; live as above
__device__ __forceinline__ void edge_bits(const AttnKvArgs& a, int b, const RowLen& len, int tile, int h, const Row& row,
                                          uint32_t* live, uint32_t* sees) {
  *live = *sees = 0;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int k0 = tile * 32 + 16 * u + 8 * h, d0 = k0 - len.start;  // d0: the new token of the first slot
    const Live8 l = live8(a, b, len, k0);
    uint32_t w;
    if (a.tree) w = d0 >= 0 ? (d0 < 64 ? (uint32_t)(row.tw >> d0) : 0) : d0 > -8 ? (uint32_t)row.tw << -d0 : 0;
    else w = (1u << min(max(row.tok + 1 - d0, 0), 8)) - 1;
    *live |= l.live << (8 * u);
    *sees |= ((l.live & ~l.fresh) | (l.fresh & w)) << (8 * u);
  }
}

// a value fragment whose slots are dead: zero, whatever the bytes are
template <int KT>
__device__ __forceinline__ u32x4 clear_dead(u32x4 f, uint32_t live) {  // 8-bit: 16 slots; bf16: 8
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = f[i];
    if constexpr (KT == KV_BF16) {
      w &= (live >> (2 * i) & 1 ? 0xffffu : 0) | (live >> (2 * i + 1) & 1 ? 0xffff0000u : 0);
    } else {
      uint32_t keep = 0;
#pragma unroll
      for (int y = 0; y < 4; ++y) keep |= live >> (4 * i + y) & 1 ? 0xffu << (8 * y) : 0;
      w &= keep;
      if constexpr (KT == KV_E4M3) {
        // (append writes no NaN code, a NaN row has a NaN scale; a new token's slot that was never
        // written may hold one, and rows that do not see it are spared)
        const uint32_t nan = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
        w &= ~(nan * 0xffu);
      }
    }
    f[i] = w;
  }
  return f;
}

// the larger of the two lane halves' values, in both
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// One row tile's running softmax and output, 32 rows a wave (lane n = lane % 32's row).
template <int KT, int D>
struct RowState {
  static constexpr int DT = D / 32;
  f32x16 o[DT];
  float m, l;

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  }

  // Scores to probabilities in two parts, so that the second can stand beside other products.
  // scores: s raw products, c = scale log2(e), kcl = c times this lane's slot's key scale (8-bit types).
  __device__ __forceinline__ void scores(f32x16& s, float c, float kcl, bool edge, uint32_t sees) {
    if constexpr (KT != KV_BF16) unrolled<16>([&](auto i) { s[i.value] *= row_bcast<i.value>(kcl); });
    if (edge) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = sees >> i & 1 ? s[i] : -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = half_max(mx);
    if constexpr (KT == KV_BF16) mx *= c;
    // m follows the maximum only once that has outgrown it by 2^8: p stays below 256, which costs no bit of
    // it, and the 16 D / 32 products of the output's rescaling are rare (at each new maximum of any of 32
    // rows they were two fifths of the loop)
    const bool up = mx > m + 8.f;  // (each row for itself: its result is the same whatever rows it shares a wave with)
    if (__any(up)) {
      const float mn = up ? mx : m;
      const float al = m == -INFINITY ? (mn == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= al;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= al;
    }
  }
  // probs: vsl this lane's slot's value scale.  p: the operand of the second product, rounded to bf16, the
  // product's type: half a step of 2^-8 at random signs over the keys.  l sums the rounded values, so that
  // a key that takes nearly all keeps nearly all of 1, whatever its rounding (8-bit types: with COMP, which
  // costs 16 more instructions a tile, nothing to 1 us of 42 where the cache's bytes are the bound; without,
  // the values before rounding: one key at 0.987, the output is off by 0.0018 with it and 0.0030 without).  Sums
  // stay in 32 bits.
  template <bool COMP>
  __device__ __forceinline__ void probs(const f32x16& s, float c, float vsl, uint32_t sees, bool special, bf16x8* p) {
    constexpr bool Q8 = KT != KV_BF16;
    const float mu = m == -INFINITY ? 0.f : m;
    float e[16], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      e[i] = __builtin_amdgcn_exp2f(Q8 ? s[i] - mu : fmaf(s[i], c, -mu));
      if (Q8 && !COMP) sum[0] += e[i];
    }
    float rvs = 0.f;
    if constexpr (Q8) {
      if (COMP) {
        vsl = vsl == 0.f ? 1.f : vsl;  // (its codes are 0)
        rvs = fabsf(vsl) < INFINITY ? __builtin_amdgcn_rcpf(vsl) : 1.f;  // (1: p says who sees it)
      }
      unrolled<16>([&](auto i) { e[i.value] *= row_bcast<i.value>(vsl); });
      if (special) {  // some slot's scale is not finite: it counts for the rows that see it alone
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = sees >> i & 1 ? e[i] : 0.f;
      }
    }
    union {
      uint32_t w[4];
      bf16x2 h[4];
      bf16x8 v;
    } r[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) r[u].v[i] = (__bf16)e[8 * u + i];
    p[0] = r[0].v;
    p[1] = r[1].v;
    if constexpr (!Q8) {
      const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) sum[u] = __builtin_amdgcn_fdot2_f32_bf16(r[u].h[i], one, sum[u], false);
    } else if constexpr (COMP) {
      unrolled<16>([&](auto i) {
        const uint32_t w = r[i.value >> 3].w[(i.value & 7) >> 1];
        const float x = __uint_as_float(i.value & 1 ? w & 0xffff0000u : w << 16), y = row_bcast<i.value>(rvs);
        sum[i.value & 1] = fmaf(x, y, sum[i.value & 1]);
      });
    }
    l += sum[0] + sum[1];
  }
};

// A drafted token's value may hold an infinity or a NaN that only some rows see; 0 * inf would hand it to
// all of them (bf16; an 8-bit code is finite).  The loop takes such values of new tokens out of the
// product (spare_fresh) and remembers that there were any; behind the loop they are added to the rows
// that see them: +inf, -inf, or both for a NaN, where a product of indicators counts any.
__device__ __forceinline__ u32x4 spare_fresh(u32x4 f, uint32_t fresh, bool* spared) {  // 8 slots of one dim
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = f[i];
    const bool lo = (w & 0x7f80u) == 0x7f80u && (fresh >> (2 * i) & 1);
    const bool hi = (w & 0x7f800000u) == 0x7f800000u && (fresh >> (2 * i + 1) & 1);
    f[i] = w & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
    *spared |= lo || hi;
  }
  return f;
}
template <int D>
__device__ __forceinline__ void add_specials(const AttnKvArgs& a, int b, const RowLen& len, const bf16_t* v, int tile, int n,
                                             int h, const Row& row, f32x16* o) {
  uint32_t live, sees;
  edge_bits(a, b, len, tile, h, row, &live, &sees);
  // pairs of 1.0 and 0.0 in bf16
  auto ones = [](bool lo, bool hi) { return (lo ? 0x3f80u : 0u) | (hi ? 0x3f800000u : 0u); };
  uint4 one[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const uint32_t m = (sees & (live8(a, b, len, tile * 32 + 16 * u + 8 * h).fresh << (8 * u))) >> (8 * u);
    one[u] = make_uint4(ones(m & 1, m & 2), ones(m & 4, m & 8), ones(m & 16, m & 32), ones(m & 64, m & 128));
  }
#pragma unroll
  for (int t = 0; t < D / 32; ++t) {
    uint4 f[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      f[u] = *reinterpret_cast<const uint4*>(v + (size_t)(32 * t + n) * a.c.slots + (size_t)tile * 32 + 16 * u + 8 * h);
    for (int sg = 0; sg < 2; ++sg) {
      const uint32_t inf = sg ? 0xff80u : 0x7f80u;
      auto bad = [&](uint32_t z) { return (z & 0x7fffu) > 0x7f80u || z == inf; };
      auto pair = [&](uint32_t w) { return ones(bad(w & 0xffffu), bad(w >> 16)); };
      f32x16 cnt;
#pragma unroll
      for (int i = 0; i < 16; ++i) cnt[i] = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 ind = make_uint4(pair(f[u].x), pair(f[u].y), pair(f[u].z), pair(f[u].w));
        cnt = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ind), __builtin_bit_cast(bf16x8, one[u]), cnt,
                                                      0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (cnt[i] > 0.f) o[t][i] += sg ? -INFINITY : INFINITY;
    }
  }
}

// The block's place.  Blocks are dealt round-robin over the 8 XCDs, and over the CUs of each: the row
// blocks of a unit stay on one XCD, where the second finds the first's keys in L2.  Rows that are split
// (all blocks are on the card at once) go row block by row block, so that a CU gets different ones (with
// the row block innermost, CUs got two full ones or two that were nearly empty); unsplit ones, of which
// there may be many more, go unit by unit.
struct Place {
  int unit, rb, hkv, x;
};
__device__ __forceinline__ Place place_of(int NS, int least, int RB, int Hkv) {
  Place p;
  const int k = (int)(blockIdx.x >> 3), xcd = (int)(blockIdx.x & 7);
  if (RB == 1) {
    p.unit = k * 8 + xcd;
    p.rb = 0;
  } else if (least) {
    const int upx = (NS * Hkv + 7) >> 3;
    p.rb = k / upx;
    p.unit = (k - p.rb * upx) * 8 + xcd;
  } else {
    p.unit = k / RB * 8 + xcd;
    p.rb = k % RB;
  }
  p.hkv = p.unit % Hkv;
  p.x = p.unit / Hkv;
  return p;
}

// Everything that a loop takes from before it has arrived.  (Without it the compiler, which cannot tell the
// first turn from the others, waits for q's loads in every turn, and with them for the tiles in flight.)
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// this lane's row r: token, tree word, and the q fragments (16-byte pieces of dims 32 j + 16 h + 8 e)
template <int D>
__device__ __forceinline__ Row load_row(const AttnKvArgs& a, int b, int hkv, const RowLen& len, int G, int t, int g, int h,
                                        bf16x8* qf) {
  const bf16_t* q = a.q + ((size_t)b * a.T + t) * a.ldq + (size_t)(hkv * G + g) * D + h * 16;
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      qf[2 * j + e] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(q + 32 * j + 8 * e));
  const int seen = len.nk - len.start;  // new tokens that have a slot
  return {t, a.tree ? a.tree[(size_t)b * a.T + t] & (seen >= 64 ? ~0ull : (1ull << seen) - 1) : 0};
}

// The loads of a tile that W waves share, and their way into LDS as the fragments of the two products
// (lane l's 16 bytes of fragment k: at k / 2 .. see FB).  8-bit: a wave-wide load is a KiB as it lies, two
// fragments in bf16.  bf16: 16 rows (K) or dims (V^T) of 64 bytes each, so that a load touches 16 lines
// and not 64.
constexpr int FB = 512 + 32;  // bytes of 32 lanes' fragments; 32 more, so that neighbours' writes meet no bank twice
template <int KT, int D, int W>
struct Stage {
  static constexpr bool Q8 = KT != KV_BF16;
  static constexpr int NG = Q8 ? D / 32 : D / 16;  // wave-wide loads of a tile's K, and of its V
  static constexpr int NL = (NG + W - 1) / W;
  static constexpr int BYTES = D / 8 * FB;         // of K, and of V, in LDS
  u32x4 f[NL];
  float ks, vs;  // of this lane's slot

  __device__ __forceinline__ void load_scales(const AttnKvArgs& a, size_t head, int tile, int lane) {
    if constexpr (Q8) {
      const uint32_t sl = 16 * ((lane & 15) >> 3) + 8 * (lane >> 5) + (lane & 7);
      ks = (a.c.ks + head + tile * 32)[sl];
      vs = (a.c.vs + head + tile * 32)[sl];
    }
  }
  // (wave-wide bases and 32 bits of offset a lane: slots is below 2^25)
  __device__ __forceinline__ void load_k(const char* kb, int tile, int w, int lane) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int g = w + i * W;
      if (NG % W && g >= NG) break;
      const char* p = kb + (Q8 ? (size_t)tile * (32 * D) + g * 1024
                               : ((size_t)tile * 32 + (g & 1) * 16) * (2 * D) + (g >> 1) * 64);
      f[i] = *reinterpret_cast<const u32x4*>(p + (uint32_t)(Q8 ? lane * 16 : (lane >> 2) * (2 * D) + (lane & 3) * 16));
    }
  }
  __device__ __forceinline__ void load_v(const char* vb, int slots, int tile, int w, int lane) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int g = w + i * W;
      if (NG % W && g >= NG) break;
      const char* p = vb + (Q8 ? (size_t)tile * (32 * D) + g * 1024 : ((size_t)(g * 16) * slots + (size_t)tile * 32) * 2);
      f[i] = *reinterpret_cast<const u32x4*>(p + (uint32_t)(Q8 ? lane * 16 : (lane >> 2) * (2 * slots) + (lane & 3) * 16));
    }
  }
  __device__ __forceinline__ void store_k(int w, int lane, char* kd) {
    const int n = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int g = w + i * W;
      if (NG % W && g >= NG) break;
      if constexpr (Q8) {  // steps 2 g and 2 g + 1
        put8(kd + (4 * g + h) * FB + n * 16, f[i]);
      } else {
        const int cc = (g >> 1) * 4 + (lane & 3);  // the row's 16-byte piece: dims 8 cc..
        const int m = kv_row_of_slot((g & 1) * 16 + (lane >> 2));
        *reinterpret_cast<u32x4*>(kd + (((cc >> 2) * 2 + (cc & 1)) * 2 + (cc >> 1 & 1)) * FB + m * 16) = f[i];
      }
    }
  }
  // true: a new token's value was not finite and has been spared (bf16)
  __device__ __forceinline__ bool store_v(const AttnKvArgs& a, int b, const RowLen& len, int tile, int w, int lane, char* vd) {
    const int n = lane & 31, h = lane >> 5;
    bool spared = false;
    if (a.mask != nullptr || tile * 32 + 32 > len.start) {
      if constexpr (Q8) {
        const uint32_t live = live8(a, b, len, tile * 32 + 8 * h).live | live8(a, b, len, tile * 32 + 16 + 8 * h).live << 8;
#pragma unroll
        for (int i = 0; i < NL; ++i) f[i] = clear_dead<KT>(f[i], live);
      } else {
        const Live8 l = live8(a, b, len, tile * 32 + (lane & 3) * 8);
#pragma unroll
        for (int i = 0; i < NL; ++i) f[i] = spare_fresh(clear_dead<KT>(f[i], l.live), l.fresh, &spared);
      }
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int g = w + i * W;
      if (NG % W && g >= NG) break;
      if constexpr (Q8) {  // the two halves of the slots
        put8(vd + (4 * g + h) * FB + n * 16, f[i]);
      } else {
        const int d = g * 16 + (lane >> 2);
        *reinterpret_cast<u32x4*>(vd + ((d >> 5) * 4 + (lane & 3)) * FB + (d & 31) * 16) = f[i];
      }
    }
    return spared;
  }
  static __device__ __forceinline__ void put8(char* d, const u32x4& f) {
    *reinterpret_cast<bf16x8*>(d) = frag8<KT>(f[0], f[1]);
    *reinterpret_cast<bf16x8*>(d + 2 * FB) = frag8<KT>(f[2], f[3]);
  }
};

// The (m, l, o) of N groups of waves that went through different tiles of the same rows [r0, r1), into one,
// in order: to the output, or as the partial of a split row (slot >= 0), which the join divides.  src: the
// first group's o, [rows][D + 4], `step` bytes from one to the next; ml: pairs, `mstep` of them to the next.
template <int D, int N>
__device__ __forceinline__ void merge_groups(const AttnKvArgs& a, int b, int hkv, int G, int r0, int r1, int slot, float* po,
                                             int rows, const char* src, int step, const float* ml, int mstep) {
  for (int q = threadIdx.x; q < (r1 - r0) * (D / 4); q += blockDim.x) {
    const int r = q / (D / 4), d = q % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < N; ++w) M = fmaxf(M, ml[(w * mstep + r) * 2]);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < N; ++w) {
      const float2 x = *reinterpret_cast<const float2*>(ml + (w * mstep + r) * 2);
      const float f = x.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x.x - M);
      const float4 z = *reinterpret_cast<const float4*>(src + (size_t)w * step + (r * (D + 4) + d) * 4);
      L += f * x.y;
      y.x += f * z.x; y.y += f * z.y; y.z += f * z.z; y.w += f * z.w;
    }
    if (slot >= 0) {
      *reinterpret_cast<float4*>(po + (size_t)r * D + d) = y;
      if (d == 0) *reinterpret_cast<float2*>(po + (size_t)rows * D + r * 2) = make_float2(M, L);
    } else {
      const float sc = L == 0.f ? 0.f : 1.f / L;  // (a row that saw nothing is 0)
      const int t = (r0 + r) / G;
      bf16_t* dst = a.out + ((size_t)b * a.T + t) * a.ldo + (size_t)(hkv * G + r0 + r - t * G) * D + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(y.x * sc, y.y * sc), pack2(y.z * sc, y.w * sc));
    }
  }
}

// Up to 32 rows a KV head (a decode step, a small tree): bound by the cache's bytes.  The NW waves of a
// block take tiles in turn, loaded one tile ahead, with no barrier in the loop, and merge once at the
// end.  8-bit fragments go from memory straight into registers, bf16 ones through LDS of the wave's own
// (straight, a wave-wide load of them touched 64 lines of memory).
//   Measured with 32 q heads on 8 KV heads of 128, one token a row, without a mask: 32 rows of 4,000 slots
// bf16 93 us (5.7 TB/s), e4m3 48 us (5.7 TB/s), rows of 2,063 to 4,000 slots 80 and 40 us (5.0 and 5.1 TB/s:
// the long rows' blocks end last); one row of 130,000 bf16 111 us (4.8 TB/s, with the join), e4m3 69 us
// (4.0 TB/s); a large copy reaches 4.9.  One row of 389 bf16 slots 8 us: a chain of dependent loads
// (length, tiles, merge) and the first fetch of 20 KB of code.  A mask makes an edge tile of every tile, and its
// bytes are waited for inside the turn, with the tiles in flight.
template <int KT, int D, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, 2) void attn_kv_keys(AttnKvArgs a, int NS, int least, uint32_t rG) {
  constexpr bool Q8 = KT != KV_BF16;
  constexpr int NF = D / 32;
  constexpr int DT = D / 32;
  using St = Stage<KT, D, 1>;
  constexpr int OS = 32 * (D + 4) * 4, WL = Q8 || 2 * St::BYTES < OS ? OS : 2 * St::BYTES;  // LDS of a wave
  __shared__ __attribute__((aligned(16))) char lds[NW * WL];
  __shared__ float mls[NW][32][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int Hkv = a.c.n_kv, G = a.Hq / Hkv, slots = a.c.slots;
  const int hkv = blockIdx.x, x = blockIdx.y;
  const float c = a.scale * 1.44269504088896340736f;  // softmax in powers of two
  const uint32_t sl = 16 * ((lane & 15) >> 3) + 8 * h + (lane & 7);  // the slot whose scales this lane holds
  char* mylds = lds + wave * WL;

  const char *kb, *vb;
  size_t head;
  u32x4 kf[NF], vf[NF];  // 8-bit
  St sk, sv;             // bf16
  float ksn = 0.f, vsn = 0.f;
  auto row_at = [&](int b) {
    head = ((size_t)b * Hkv + hkv) * slots;
    kb = (const char*)a.c.k + head * D * (Q8 ? 1 : 2);
    vb = (const char*)a.c.v + head * D * (Q8 ? 1 : 2);
  };
  auto load_k = [&](int t) {
    const char* p = kb + (size_t)t * (32 * D);
#pragma unroll
    for (int j = 0; j < NF; ++j) kf[j] = *reinterpret_cast<const u32x4*>(p + (uint32_t)(j * 1024 + lane * 16));
    ksn = (a.c.ks + head + t * 32)[sl];
    vsn = (a.c.vs + head + t * 32)[sl];
  };
  auto load_v = [&](int t) {
    const char* p = vb + (size_t)t * (32 * D);
#pragma unroll
    for (int j = 0; j < NF; ++j) vf[j] = *reinterpret_cast<const u32x4*>(p + (uint32_t)(j * 1024 + lane * 16));
  };
  auto load_tile = [&](int t) {
    if constexpr (Q8) {
      load_k(t);
      load_v(t);
    } else {
      sk.load_k(kb, t, 0, lane);
      sv.load_v(vb, slots, t, 0, lane);
    }
  };
  // an unsplit row's first tiles are known before its length is (and there, whatever that turns out to be)
  if constexpr (!SPLIT) {
    row_at(x);
    load_tile(min(wave, (slots >> 5) - 1));
  }
  for_segments<SPLIT, 16>(a, NS, least, x, hkv == 0 && x == 0, [&](const Seg& sg) {
    const int b = sg.b;
    const RowLen len = sg.len;
    const int R = len.n * G;
    if (R == 0) return;
    const int t1 = min(sg.t1, (len.nk + 31) >> 5);
    int tile = sg.t0 + wave;
    if constexpr (SPLIT) {
      row_at(b);
      if (tile < t1) load_tile(tile);
    }
    bf16x8 qf[D / 16];
    const int tk = n < R ? n * rG >> 16 : 0;  // n / G, exact for n and G of at most 32
    const Row row = load_row<D>(a, b, hkv, len, G, tk, n < R ? n - tk * G : 0, h, qf);
    RowState<KT, D> st;
    st.clear();
    bool spared = false;
    loads_done();
    for (; tile < t1; tile += NW) {
      const int nxt = min(tile + NW, t1 - 1);  // (the last turn reads its own tile or a later one again: in bounds)
      f32x16 s;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f;
      const char* kp = mylds + h * FB + n * 16;
      if constexpr (Q8) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          const bf16x8 k = j & 1 ? frag8<KT>(kf[j >> 1].z, kf[j >> 1].w) : frag8<KT>(kf[j >> 1].x, kf[j >> 1].y);
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, qf[j], s, 0, 0, 0);
        }
      } else {
        sk.store_k(0, lane, mylds);
        spared |= sv.store_v(a, b, len, tile, 0, lane, mylds + St::BYTES);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        sk.load_k(kb, nxt, 0, lane);
        sv.load_v(vb, slots, nxt, 0, lane);
        bf16x8 k[D / 16];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) k[j] = *reinterpret_cast<const bf16x8*>(kp + 2 * j * FB);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[j], qf[j], s, 0, 0, 0);
      }
      const float kcl = ksn * c;
      float vsl = vsn;
      if constexpr (Q8) load_k(nxt);
      const bool edge = a.mask != nullptr || tile * 32 + 32 > len.start;
      bool special = false;
      uint32_t live = 0xffff, sees = 0xffff;
      if (edge) {
        edge_bits(a, b, len, tile, h, row, &live, &sees);
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < NF; ++j) vf[j] = clear_dead<KT>(vf[j], live);
          vsl = live >> (lane & 15) & 1 ? vsl : 0.f;
          special = __any(!(fabsf(vsl) < INFINITY));
        }
      }
      bf16x8 p[2];
      st.scores(s, c, kcl, edge, sees);
      st.template probs<true>(s, c, vsl, sees, special, p);
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          bf16x8 v;
          if constexpr (Q8) v = u ? frag8<KT>(vf[t].z, vf[t].w) : frag8<KT>(vf[t].x, vf[t].y);
          else v = *reinterpret_cast<const bf16x8*>(kp + St::BYTES + (4 * t + 2 * u) * FB);
          st.o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p[u], st.o[t], 0, 0, 0);
        }
      if constexpr (Q8) load_v(nxt);
      else __builtin_amdgcn_wave_barrier();
    }
    if constexpr (!Q8)
      if (__any(spared))
        for (tile = sg.t0 + wave; tile < t1; tile += NW)
          if (tile * 32 + 32 > len.start) add_specials<D>(a, b, len, (const bf16_t*)vb, tile, n, h, row, st.o);

    // ---- the block's waves into one (m, l, o), in wave order ----
    st.l = half_sum(st.l);
    if (h == 0) {
      mls[wave][n][0] = st.m;
      mls[wave][n][1] = st.l;
    }
    float* os = reinterpret_cast<float*>(mylds) + n * (D + 4) + 4 * h;
    if (n < R) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4*>(os + 32 * t + 2 * i) =
              make_float4(st.o[t][i], st.o[t][i + 1], st.o[t][i + 2], st.o[t][i + 3]);
    }
    __syncthreads();
    merge_groups<D, NW>(a, b, hkv, G, 0, R, SPLIT ? sg.slot : -1,
                        a.part + head_floats(a.B) + (size_t)(sg.slot * Hkv + hkv) * 32 * (D + 2), 32, lds, WL, mls[0][0], 32);
    if constexpr (SPLIT) __syncthreads();  // (the next segment writes LDS)
  });
}

// More rows: bound by the arithmetic on the scores (of a tile's turn the products take about a third, the powers,
// the maximum and the roundings the rest, and two waves a SIMD hide little of one behind the other).  W waves,
// 32 rows each, go through the same tiles, whose fragments they load, turn into bf16 and put into LDS
// together, once for all rows, a turn ahead of the products (two halves of LDS, one barrier a turn).
//   A block has KS such groups, which take the tiles in turn and are merged at the end: with a block each
// (KS 1), four or two times the partials went through memory: 4 rows of 4,688 to 7,500 e4m3 slots and 16 tokens
// of 4 heads wrote and read 32 MB of them beside the cache's 50 MB (42 us, 36 like this; left pads).
//   Measured with 32 q heads on 8 KV heads of 128, without a mask: one row of 130,001 slots, 33 tokens, bf16
// 137 us, e4m3 141, int8 151 (510, 500, 470 TFLOP/s; three of the eight waves have no rows there); 16 rows of
// 4,000 slots, 64 tokens, 97, 97, 100 (700, 710, 680 TFLOP/s; of it 12 us the join); a large plain matrix
// product reaches 1,150.  4 rows of 7,500 slots, 16 tokens: 39, 27, 28, and 54, 39, 39 with a mask, for which
// every tile is an edge tile: two looks at its bytes, the selects, and a wait for the tiles in flight.
template <int KT, int D, int W, int KS>
__global__ __launch_bounds__(64 * W * KS, 2) void attn_kv_rows(AttnKvArgs a, int NS, int least, int RB) {
  constexpr bool Q8 = KT != KV_BF16;
  constexpr int DT = D / 32, rows = 32 * W;
  constexpr int TT = W == 2 ? 1 : 2;  // tiles of a group a turn (what LDS holds)
  using St = Stage<KT, D, W>;
  constexpr int OS = KS > 1 ? rows * (D + 4) * 4 : 0, GL = 4 * TT * St::BYTES < OS ? OS : 4 * TT * St::BYTES;
  __shared__ __attribute__((aligned(16))) char lds[KS][GL];  // of a group: two halves of TT tiles, K and V; then its o
  __shared__ float mls[KS][KS > 1 ? rows : 1][2];
  __shared__ int spared;
  const int lane = threadIdx.x & 63, wv0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wv0 % W, kg = wv0 / W;
  char* const mylds = lds[kg];
  auto lk = [&](int half, int i) { return mylds + ((half * TT + i) * 2) * St::BYTES; };
  auto lv = [&](int half, int i) { return mylds + ((half * TT + i) * 2 + 1) * St::BYTES; };
  const int n = lane & 31, h = lane >> 5;
  const int Hkv = a.c.n_kv, G = a.Hq / Hkv, slots = a.c.slots;
  const Place pl = place_of(NS, least, RB, Hkv);
  if (pl.unit >= NS * Hkv) return;
  const float c = a.scale * 1.44269504088896340736f;

  Segments<4 + 3 * KS> it(a, NS, least, pl.x, blockIdx.x == 0);
  for (Seg sg; it.next(sg);) {
    const int b = sg.b;
    const RowLen len = sg.len;
    const int r0 = pl.rb * rows, Rend = min(len.n * G, r0 + rows);  // this block's rows of (row, KV head)
    if (r0 >= Rend) continue;
    // a chain's row block sees no slot behind its last token's
    const int nk = a.tree ? len.nk : min(len.nk, len.start + (Rend - 1) / G + 1);
    const int t0 = sg.t0, t1 = min(sg.t1, (nk + 31) >> 5);
    const int myr = r0 + wave * 32 + n;
    const bool act = r0 + wave * 32 < Rend;  // (a wave without rows only helps with the tiles)

    const size_t head = ((size_t)b * Hkv + pl.hkv) * slots;
    const char* kb = (const char*)a.c.k + head * D * (Q8 ? 1 : 2);
    const char* vb = (const char*)a.c.v + head * D * (Q8 ? 1 : 2);
    RowState<KT, D> st;
    st.clear();
    if (threadIdx.x == 0) spared = 0;
    // A turn works on TT tiles out of one half of LDS, while the next TT go from registers into the other
    // half and the TT behind them are loaded: what a turn waits for was asked for a whole turn ago.
    St gk[TT], gv[TT];
    const int wv = W - 1 - wave;  // (a tile of fewer loads than waves: K by the first waves, V by the last)
    float ks[TT], vs[TT], kn[TT], vn[TT];  // scales of this turn's tiles and of the next one's
    const uint32_t at = h * FB + n * 16;
    auto fetch = [&](int tile) {
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const int t = min(tile + i, t1 - 1);  // (past the end the last tile again: in bounds, not used)
        gk[i].load_scales(a, head, t, lane);
        gk[i].load_k(kb, t, wave, lane);
        gv[i].load_v(vb, slots, t, wv, lane);
      }
    };
    auto put = [&](int tile, int half) {
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        gk[i].store_k(wave, lane, lk(half, i));
        if (gv[i].store_v(a, b, len, min(tile + i, t1 - 1), wv, lane, lv(half, i))) spared = 1;
        if constexpr (Q8) {
          kn[i] = gk[i].ks * c;
          vn[i] = gk[i].vs;
        }
      }
    };
    if (t0 < t1) fetch(t0 + kg * TT);
    bf16x8 qf[D / 16];
    const int tk = myr < Rend ? myr / G : 0;
    const Row row = load_row<D>(a, b, pl.hkv, len, G, tk, myr < Rend ? myr - tk * G : 0, h, qf);
    __syncthreads();  // (spared is 0, and the last segment's tiles have been read)
    loads_done();
    if (t0 < t1) {
      put(t0 + kg * TT, 0);
      fetch(t0 + (KS + kg) * TT);
    }
    for (int tb = t0, half = 0; tb < t1; tb += KS * TT, half ^= 1) {
      const int tile = tb + kg * TT;
      if constexpr (Q8) {
#pragma unroll
        for (int i = 0; i < TT; ++i) {
          ks[i] = kn[i];
          vs[i] = vn[i];
        }
      }
      __syncthreads();  // this turn's fragments are there, the other half has been read
      if (tb + KS * TT < t1) {
        put(tile + KS * TT, half ^ 1);
        fetch(tile + 2 * KS * TT);
      }
      if (act) {
#pragma unroll
        for (int i = 0; i < TT; ++i) {
          const int tl = tile + i;
          if (tl >= t1) break;
          const char *kp = lk(half, i) + at, *vp = lv(half, i) + at;
          // (all reads before the first product: one at a time, each product waits out LDS's latency)
          bf16x8 k[D / 16];
#pragma unroll
          for (int j = 0; j < D / 16; ++j) k[j] = *reinterpret_cast<const bf16x8*>(kp + 2 * j * FB);
          __builtin_amdgcn_sched_barrier(0);
          f32x16 s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[0], qf[0], f32x16{}, 0, 0, 0);
#pragma unroll
          for (int j = 1; j < D / 16; ++j) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[j], qf[j], s, 0, 0, 0);
          const bool edge = a.mask != nullptr || tl * 32 + 32 > len.start;
          bool special = false;
          uint32_t live = 0xffff, sees = 0xffff;
          float vsl = vs[i];
          if (edge) {
            edge_bits(a, b, len, tl, h, row, &live, &sees);
            if constexpr (Q8) {
              vsl = live >> (lane & 15) & 1 ? vsl : 0.f;
              special = __any(!(fabsf(vsl) < INFINITY));
            }
          }
          st.scores(s, c, ks[i], edge, sees);
          bf16x8 p[2];
          st.template probs<false>(s, c, vsl, sees, special, p);
          bf16x8 v[DT][2];
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) v[t][u] = *reinterpret_cast<const bf16x8*>(vp + (4 * t + 2 * u) * FB);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int t = 0; t < DT; ++t)
              st.o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[t][u], p[u], st.o[t], 0, 0, 0);
        }
      }
    }
    if constexpr (!Q8) {
      __syncthreads();
      if (spared && act)
        for (int tile = max(t0, len.start >> 5); tile < t1; ++tile)
          if ((tile - t0) / TT % KS == kg) add_specials<D>(a, b, len, (const bf16_t*)vb, tile, n, h, row, st.o);
      if (least) __syncthreads();  // (the next segment clears it)
    }
    st.l = half_sum(st.l);
    float* po = a.part + head_floats(a.B) + ((size_t)(sg.slot * Hkv + pl.hkv) * RB + pl.rb) * rows * (D + 2);
    if constexpr (KS > 1) {  // the groups into one
      __syncthreads();  // (the tiles have been read)
      if (h == 0) *reinterpret_cast<float2*>(mls[kg][wave * 32 + n]) = make_float2(st.m, st.l);
      float* os = reinterpret_cast<float*>(mylds) + (wave * 32 + n) * (D + 4) + 4 * h;
      if (act) {
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(os + 32 * t + 2 * i) =
                make_float4(st.o[t][i], st.o[t][i + 1], st.o[t][i + 2], st.o[t][i + 3]);
      }
      __syncthreads();
      merge_groups<D, KS>(a, b, pl.hkv, G, r0, Rend, sg.slot, po, rows, lds[0], GL, mls[0][0], rows);
      continue;  // (the next segment writes LDS behind its first barrier)
    }
    if (myr >= Rend) continue;
    if (sg.slot >= 0) {  // a split row is divided by the join
      const int rr = wave * 32 + n;
      if (h == 0) *reinterpret_cast<float2*>(po + (size_t)rows * D + rr * 2) = make_float2(st.m, st.l);
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<float4*>(po + (size_t)rr * D + 32 * t + 2 * i + 4 * h) =
              make_float4(st.o[t][i], st.o[t][i + 1], st.o[t][i + 2], st.o[t][i + 3]);
    } else {
      const float sc = st.l == 0.f ? 0.f : 1.f / st.l;  // (a row that saw nothing is 0)
      bf16_t* dst = a.out + ((size_t)b * a.T + row.tok) * a.ldo + (size_t)(pl.hkv * G + myr - row.tok * G) * D;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<uint2*>(dst + 32 * t + 2 * i + 4 * h) =
              make_uint2(pack2(st.o[t][i] * sc, st.o[t][i + 1] * sc), pack2(st.o[t][i + 2] * sc, st.o[t][i + 3] * sc));
    }
  }
}

// Joins the partials of a row.  Bound by their bytes (16 rows x 64 tokens x 32 heads, two blocks a row: 42 MB in
// 11.6 us) or, for few rows, by the loads' latency: GS groups of D / 4 threads (4 dims each) take every GS-th block's partial,
// four loads in flight, and the groups' sums are added in order.
template <int D, int GS>
__global__ __launch_bounds__(256) void attn_kv_join(AttnKvArgs a, int RB, int rows) {
  constexpr int TR = D / 4, RP = 256 / (TR * GS);  // threads a group, rows a block
  __shared__ float ms[RP][GS], ls[RP][GS];
  __shared__ __attribute__((aligned(16))) float ys[RP][GS][D];
  const int d = threadIdx.x % TR * 4, g = threadIdx.x / TR % GS, row = threadIdx.x / (TR * GS);
  const int64_t w = (int64_t)blockIdx.x * RP + row;
  const int TH = a.T * a.Hq, b = (int)min(w / TH, (int64_t)a.B - 1), th = (int)(w - (int64_t)b * TH), t = th / a.Hq,
            hq = th - t * a.Hq;
  const int2 xs = *reinterpret_cast<const int2*>(a.part + 2 * b);
  const int x0 = xs.x, ns = xs.y;
  const bool on = th < TH && ns > 1 && !(a.counts && t >= a.counts[b]);
  float M = -INFINITY, L = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  if (on) {
    const int G = a.Hq / a.c.n_kv, hkv = hq / G, r = t * G + hq - hkv * G, rb = r / rows, rr = r - rb * rows;
    const size_t step = (size_t)a.c.n_kv * RB * rows * (D + 2);  // from one slot to the next
    const float* p = a.part + head_floats(a.B) + (size_t)(hkv * RB + rb) * rows * (D + 2);
    const float *pm = p + (size_t)rows * D + rr * 2, *po = p + (size_t)rr * D + d;
    // the row begins in block x0 (slot 2 x0 + 1) and goes on in slots 2 x0 + 2, 2 x0 + 4, ..
    for (int s0 = g; s0 < ns; s0 += 4 * GS) {
      float2 ml[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = min(s0 + i * GS, ns - 1);
        const size_t at = (size_t)(2 * x0 + (s ? 2 * s : 1)) * step;
        ml[i] = *reinterpret_cast<const float2*>(pm + at);
        v[i] = *reinterpret_cast<const float4*>(po + at);
      }
      float mx = M;
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = s0 + i * GS < ns ? fmaxf(mx, ml[i].x) : mx;
      const float al = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - mx);
      M = mx;
      L *= al;
      y.x *= al; y.y *= al; y.z *= al; y.w *= al;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (s0 + i * GS >= ns) break;
        const float f = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - M);
        L += f * ml[i].y;
        y.x += f * v[i].x; y.y += f * v[i].y; y.z += f * v[i].z; y.w += f * v[i].w;
      }
    }
  }
  if constexpr (GS > 1) {
    *reinterpret_cast<float4*>(&ys[row][g][d]) = y;
    if (d == 0) {
      ms[row][g] = M;
      ls[row][g] = L;
    }
    __syncthreads();
    if (g) return;
    float mx = M;
#pragma unroll
    for (int i = 1; i < GS; ++i) mx = fmaxf(mx, ms[row][i]);
    L = 0.f;
    y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < GS; ++i) {
      const float m = ms[row][i], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
      const float4 v = *reinterpret_cast<const float4*>(&ys[row][i][d]);
      L += f * ls[row][i];
      y.x += f * v.x; y.y += f * v.y; y.z += f * v.z; y.w += f * v.w;
    }
  }
  if (!on) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;  // (a row that saw nothing is 0)
  bf16_t* dst = a.out + ((size_t)b * a.T + t) * a.ldo + (size_t)hq * D + d;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(y.x * inv, y.y * inv), pack2(y.z * inv, y.w * inv));
}

// The launch: the form (W = 0: attn_kv_keys; else attn_kv_rows of W waves), its row blocks, the blocks NS
// that share the tiles and the least share (0: a block a row).
struct AkvPlan {
  int W, RB, NS, least;
};
// Constants by measurement, 32 q heads on 8 KV heads of 128, bf16 / e4m3, us:
//   (rows of a batch: from the slots given down to about half of them)
//   form: one tile of rows stays with its waves' registers (keys); more go to the next of the groups that are
//     built, of two, four or eight waves: those beyond the rows' tiles help with the loads alone;
//   least (tiles a block): 1 row, 16 tokens, 2,000 slots: 8 19.2 / 19.0, 16 21.8 / 21.4; W 8 has no groups
//     that share a block's tiles: 4;
//   most (tiles up to which nothing is split): W 2, 1 row of 500 slots: 16 19.6 / 19.4, 32 17.8 / 16.5;
//     1 row of 2,000: 32 21.8 / 21.4, 64 32.1 / 30.4; W 4, 8 rows of 700: 12 28.6 / 27.1, 24 26.4 / 24.4;
//     8 rows of 1,400: 24 27.6 / 27.7, 48 37.2 / 35.9.
static AkvPlan plan(int B, int T, int Hq, int n_kv, int slots, int max_len) {
  AkvPlan p;
  const int64_t R = (int64_t)T * (Hq / n_kv), rt = (R + 31) / 32;
  p.W = rt <= 1 ? 0 : rt <= 2 ? 2 : rt <= 4 ? 4 : 8;
  p.RB = p.W ? (int)((rt + p.W - 1) / p.W) : 1;
  const int64_t len = std::min<int64_t>(slots, (int64_t)(max_len > 0 ? std::min(max_len, slots) : slots) + T);
  const int64_t tiles = (len + 31) / 32;                              // of the longest row
  const int64_t units = std::max<int64_t>(1, (int64_t)n_kv * p.RB);   // blocks a row, unsplit
  const int64_t room = 256;                                           // blocks that the card holds at once
  const int64_t most = p.W == 0 ? 64 : p.W == 8 ? 20 : p.W == 4 ? 24 : 32, least = p.W == 8 ? 4 : 8;
  p.least = (int)least;
  p.NS = (int)std::max<int64_t>(1, std::min(room / units, (int64_t)B * ((tiles + least - 1) / least)));
  // short rows, or enough of them: nothing to join
  if (tiles <= most || p.NS <= B) {
    p.least = 0;
    p.NS = B;
  }
  return p;
}

size_t attn_kv_ws_bytes(int B, int T, int Hq, int n_kv, int D, int slots, int max_len) {
  const AkvPlan p = plan(B, T, Hq, n_kv, slots, max_len);
  if (p.least == 0) return 0;
  return (head_floats(B) + (size_t)2 * p.NS * n_kv * p.RB * 32 * std::max(1, p.W) * (D + 2)) * sizeof(float);
}

template <int KT, int D, bool SPLIT>
static void launch_form(const AttnKvArgs& a, const AkvPlan& p, int64_t grid, hipStream_t s) {
  const dim3 g((unsigned)grid);
  switch (p.W) {
    case 0: {
      const uint32_t G = a.Hq / a.c.n_kv, rG = (65536 + G - 1) / G;
      hipLaunchKernelGGL((attn_kv_keys<KT, D, 8, SPLIT>), dim3(a.c.n_kv, p.NS), dim3(512), 0, s, a, p.NS, p.least, rG);
      break;
    }
    case 2: hipLaunchKernelGGL((attn_kv_rows<KT, D, 2, 4>), g, dim3(512), 0, s, a, p.NS, p.least, p.RB); break;
    case 4:
      // (64 rows of 1,000 slots, three row tiles: 52 us in blocks of 4 waves, two a CU, that never wait for
      // each other, and 67 in blocks of 8; 8 rows of 700, four: 34 and 26)
      if (!p.least && grid > 256) hipLaunchKernelGGL((attn_kv_rows<KT, D, 4, 1>), g, dim3(256), 0, s, a, p.NS, p.least, p.RB);
      else hipLaunchKernelGGL((attn_kv_rows<KT, D, 4, 2>), g, dim3(512), 0, s, a, p.NS, p.least, p.RB);
      break;
    default: hipLaunchKernelGGL((attn_kv_rows<KT, D, 8, 1>), g, dim3(512), 0, s, a, p.NS, p.least, p.RB);
  }
}
template <int KT, int D>
static hipError_t launch(const AttnKvArgs& a, const AkvPlan& p, hipStream_t s) {
  const int64_t grid = ((int64_t)p.NS * a.c.n_kv + 7) / 8 * 8 * p.RB;
  const int GS = p.NS > 4 * a.B ? 8 : 1;  // (rows of many partials: they are read at once, not one after the other)
  const int64_t join = ((int64_t)a.B * a.T * a.Hq * (D / 4) * GS + 255) / 256;
  if (grid > INT_MAX || join > INT_MAX || (p.W == 0 && p.NS > 65535)) return hipErrorInvalidValue;
  if (!p.least) {
    launch_form<KT, D, false>(a, p, grid, s);
    return hipGetLastError();
  }
  launch_form<KT, D, true>(a, p, grid, s);
  if (GS == 8)
    hipLaunchKernelGGL((attn_kv_join<D, 8>), dim3((unsigned)join), dim3(256), 0, s, a, p.RB, 32 * std::max(1, p.W));
  else
    hipLaunchKernelGGL((attn_kv_join<D, 1>), dim3((unsigned)join), dim3(256), 0, s, a, p.RB, 32 * std::max(1, p.W));
  return hipGetLastError();
}
template <int KT>
static hipError_t launch_d(const AttnKvArgs& a, const AkvPlan& p, hipStream_t s) {
  switch (a.c.D) {
    case 32: return launch<KT, 32>(a, p, s);
    case 64: return launch<KT, 64>(a, p, s);
    case 128: return launch<KT, 128>(a, p, s);
  }
  return hipErrorInvalidValue;
}

hipError_t attn_kv(const AttnKvArgs& a, hipStream_t s) {
  if (a.B == 0 || a.T == 0) return hipSuccess;
  const AkvPlan p = plan(a.B, a.T, a.Hq, a.c.n_kv, a.c.slots, a.max_len);
  switch (a.c.type) {
    case KV_BF16: return launch_d<KV_BF16>(a, p, s);
    case KV_E4M3: return launch_d<KV_E4M3>(a, p, s);
    case KV_INT8: return launch_d<KV_INT8>(a, p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace mtts
