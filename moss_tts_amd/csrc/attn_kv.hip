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
// probabilities never leave its registers, and K / V fragments come straight from memory: no LDS in
// the loop and no barrier.  The 4 waves of a block take tiles in turn and merge once at the end.
#include "engine_internal.h"
#include "kvq.h"

namespace mtts {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// context, new tokens and visible slots of row b; a row's slots end with the cache
struct RowLen {
  int start, n, nk;
};
__device__ __forceinline__ RowLen row_len(const AttnKvArgs& a, int b) {
  RowLen r;
  r.start = min(max(a.start[b], 0), a.c.slots);
  r.n = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  r.nk = (int)min((int64_t)r.start + r.n, (int64_t)a.c.slots);
  return r;
}

// Splits.  NS blocks (a KV head and row block each) are shared out over the batch's rows by their
// lengths, which only the device knows: row b gets 1 + (NS - B) nt_b / sum(nt), at most one for each
// 4 tiles.  Every block works the table out for itself (one wave-wide scan of the lengths).
struct Split {
  int b, s, ns, x0;
};
__device__ __forceinline__ int splits_of(int nt, int total, int extra) {
  const int want = total > 0 ? 1 + (int)((int64_t)extra * nt / total) : 1;
  return max(1, min(want, (nt + 3) / 4));
}
// the split with number x (b = -1: none), or with x < 0 row `row`'s first
__device__ Split find_split(const AttnKvArgs& a, int NS, int x, int row) {
  Split r{-1, 0, 1, 0};
  if (NS == a.B) {
    r.b = x < 0 ? row : x;
    r.x0 = r.b;
    return r;
  }
  const int lane = threadIdx.x & 63;
  int total = 0, nt = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    nt = b0 + lane < a.B ? (row_len(a, b0 + lane).nk + 31) >> 5 : 0;
    int t = nt;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    total += t;
  }
  int off = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    if (a.B > 64) nt = b0 + lane < a.B ? (row_len(a, b0 + lane).nk + 31) >> 5 : 0;
    const int ns = b0 + lane < a.B ? splits_of(nt, total, NS - a.B) : 0;
    int incl = ns;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(incl, o, 64);
      if (lane >= o) incl += v;
    }
    const uint64_t hit = __ballot(x < 0 ? b0 + lane == row : ns > 0 && x < off + incl);
    if (hit) {
      const int f = __ffsll((unsigned long long)hit) - 1;
      r.b = b0 + f;
      r.ns = __builtin_amdgcn_readfirstlane(__shfl(ns, f, 64));
      r.x0 = __builtin_amdgcn_readfirstlane(off + __shfl(incl, f, 64)) - r.ns;
      r.s = x - r.x0;
      return r;
    }
    off += __builtin_amdgcn_readfirstlane(__shfl(incl, 63, 64));
  }
  return r;
}

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
      const float x = (float)(int8_t)(w[i >> 1] >> (16 * (i & 1)));
      const float y = (float)(int8_t)(w[i >> 1] >> (16 * (i & 1) + 8));
      o.w[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);  // the high halves
    }
  }
  return o.v;
}

template <int KT, int D, int RT>
__global__ __launch_bounds__(256, RT == 1 ? 2 : 1) void attn_kv_kernel(AttnKvArgs a, int NS, int RB) {
  constexpr bool Q8 = KT != KV_BF16;
  constexpr int NF = Q8 ? D / 32 : D / 16;  // 16-byte fragments of K, and of V, a lane takes of a tile
  constexpr int DT = D / 32;                // 32-dim tiles of the output
  constexpr int OW = DT > 1 ? 64 : 32;      // dims that one round of the merge holds
  __shared__ __attribute__((aligned(16))) float os[4][32][OW + 4];
  __shared__ float mls[4][32 * RT][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5;
  const int Hkv = a.c.n_kv, G = a.Hq / Hkv, slots = a.c.slots;
  // blocks are dealt round-robin over the 8 XCDs: the row blocks of one split stay on one, where the
  // second finds the first's keys in L2
  const int unit = (int)(blockIdx.x >> 3) / RB * 8 + (blockIdx.x & 7), rb = (blockIdx.x >> 3) % RB;
  if (unit >= NS * Hkv) return;
  const int hkv = unit % Hkv, x = unit / Hkv;
  const Split sp = find_split(a, NS, x, 0);
  if (sp.b < 0) return;
  const int b = sp.b;
  const RowLen len = row_len(a, b);
  const int R = len.n * G, r0 = rb * 32 * RT;  // rows of this (row, KV head); this block's first
  if (r0 >= R) return;
  // a chain's row block sees no slot behind its last token's
  int nk = len.nk;
  if (!a.tree) nk = min(nk, len.start + (min(R, r0 + 32 * RT) - 1) / G + 1);
  const int nt = (nk + 31) >> 5;
  const int t0 = (int)((int64_t)nt * sp.s / sp.ns), t1 = (int)((int64_t)nt * (sp.s + 1) / sp.ns);

  // ---- this lane's rows: q fragments and what the token sees ----
  bf16x8 qf[RT][D / 16];
  uint64_t tw[RT];
  int tok[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = r0 + rt * 32 + n, t = r / G, g = r - t * G;
    const bool on = r < R;
    tok[rt] = on ? t : 0;
    const bf16_t* q = a.q + ((size_t)b * a.T + tok[rt]) * a.ldq + (size_t)(hkv * G + (on ? g : 0)) * D + h * 16;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        qf[rt][2 * j + e] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(q + 32 * j + 8 * e));
    const int seen = len.nk - len.start;  // new tokens that have a slot
    tw[rt] = a.tree ? a.tree[(size_t)b * a.T + tok[rt]] & (seen >= 64 ? ~0ull : (1ull << seen) - 1) : 0;
  }

  const size_t head = ((size_t)b * Hkv + hkv) * slots;
  const char* kb = (const char*)a.c.k + head * D * (Q8 ? 1 : 2);
  const char* vb = (const char*)a.c.v + head * D * (Q8 ? 1 : 2);
  const int kap = kv_slot_of_row(n);
  auto load_k = [&](int tile, uint4* f) {
    if constexpr (Q8) {
      const char* p = kb + (size_t)tile * (32 * D) + lane * 16;
#pragma unroll
      for (int j = 0; j < NF; ++j) f[j] = *reinterpret_cast<const uint4*>(p + j * 1024);
    } else {
      const char* p = kb + ((size_t)tile * 32 + kap) * (2 * D) + h * 32;
#pragma unroll
      for (int j = 0; j < NF; ++j) f[j] = *reinterpret_cast<const uint4*>(p + (j >> 1) * 64 + (j & 1) * 16);
    }
  };
  auto load_v = [&](int tile, uint4* f) {
    if constexpr (Q8) {
      const char* p = vb + (size_t)tile * (32 * D) + lane * 16;
#pragma unroll
      for (int j = 0; j < NF; ++j) f[j] = *reinterpret_cast<const uint4*>(p + j * 1024);
    } else {
      const char* p = vb + ((size_t)n * slots + (size_t)tile * 32 + 8 * h) * 2;
#pragma unroll
      for (int j = 0; j < NF; ++j) f[j] = *reinterpret_cast<const uint4*>(p + (size_t)(j >> 1) * 64 * slots + (j & 1) * 32);
    }
  };
  auto k_frag = [&](const uint4* f, int s) -> bf16x8 {  // step s of the 16-dim steps
    if constexpr (Q8) return s & 1 ? frag8<KT>(f[s >> 1].z, f[s >> 1].w) : frag8<KT>(f[s >> 1].x, f[s >> 1].y);
    else return __builtin_bit_cast(bf16x8, f[s]);
  };
  auto v_frag = [&](const uint4* f, int t, int u) -> bf16x8 {
    if constexpr (Q8) return u ? frag8<KT>(f[t].z, f[t].w) : frag8<KT>(f[t].x, f[t].y);
    else return __builtin_bit_cast(bf16x8, f[2 * t + u]);
  };

  f32x16 o[RT][DT];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[rt][t][i] = 0.f;
  }
  const float c = a.scale * 1.44269504088896340736f;  // softmax in powers of two

  uint4 kf[NF], vf[NF];
  int tile = t0 + wave;
  if (tile < t1) {
    load_k(tile, kf);
    load_v(tile, vf);
  }
  for (; tile < t1; tile += 4) {
    const int nxt = min(tile + 4, t1 - 1);  // (the last turn reads its own tile again: in bounds)
    f32x16 s[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[rt][i] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const bf16x8 k = k_frag(kf, j);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, qf[rt][j], s[rt], 0, 0, 0);
    }
    load_k(nxt, kf);
    float vs[16];
    if constexpr (Q8) {
      float ks[16];
      const float* p = a.c.ks + head + tile * 32 + 8 * h;
      const float* w = a.c.vs + head + tile * 32 + 8 * h;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<float4*>(&ks[8 * u + i]) = *reinterpret_cast<const float4*>(p + 16 * u + i);
          *reinterpret_cast<float4*>(&vs[8 * u + i]) = *reinterpret_cast<const float4*>(w + 16 * u + i);
        }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float kc = ks[i] * c;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][i] *= kc;
      }
    } else {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[rt][i] *= c;
    }
    uint32_t sees[RT];  // bit 8 u + i: the row sees slot 16 u + 8 h + i of the tile
    const bool edge = a.mask != nullptr || tile * 32 + 32 > len.start;
    if (edge) {
      uint32_t live = 0;  // slots that some row may see: the others' bytes are anything
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sees[rt] = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k0 = tile * 32 + 16 * u + 8 * h, d0 = k0 - len.start;  // d0: the first slot's new token
        const int cn = min(max(-d0, 0), 8), ln = min(max(len.nk - k0, 0), 8);
        uint32_t ctx = (1u << cn) - 1;
        const uint32_t fresh = ((1u << ln) - 1) & ~ctx;
        if (a.mask) {
          const uint2 mk = *reinterpret_cast<const uint2*>(a.mask + (size_t)b * slots + k0);
          uint32_t mb = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mb |= ((mk.x >> (8 * i)) & 0xff ? 1u << i : 0) | ((mk.y >> (8 * i)) & 0xff ? 16u << i : 0);
          ctx &= mb;
        }
        live |= (ctx | fresh) << (8 * u);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          uint32_t w;
          if (a.tree) w = d0 >= 0 ? (d0 < 64 ? (uint32_t)(tw[rt] >> d0) : 0) : d0 > -8 ? (uint32_t)tw[rt] << -d0 : 0;
          else w = (1u << min(max(tok[rt] + 1 - d0, 0), 8)) - 1;
          sees[rt] |= (ctx | (fresh & w)) << (8 * u);
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[rt][i] = sees[rt] >> i & 1 ? s[rt][i] : -INFINITY;
      // values of slots that nobody sees (never written, padded away) must not reach a product
      if constexpr (Q8) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t keep = 0;
#pragma unroll
          for (int y = 0; y < 4; ++y) keep |= live >> (4 * w + y) & 1 ? 0xffu << (8 * y) : 0;
#pragma unroll
          for (int j = 0; j < NF; ++j) {
            uint32_t& z = reinterpret_cast<uint32_t*>(&vf[j])[w];
            z &= keep;
            if constexpr (KT == KV_E4M3) {
              // (append writes no NaN code, a NaN row has a NaN scale; a new token's slot that was never
              // written may hold one, and rows that do not see it are spared)
              const uint32_t nan = (((z & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
              z &= ~(nan * 0xffu);
            }
          }
        }
      } else {
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          const uint32_t keep = (live >> (2 * w) & 1 ? 0xffffu : 0) | (live >> (2 * w + 1) & 1 ? 0xffff0000u : 0);
#pragma unroll
          for (int t = 0; t < DT; ++t) reinterpret_cast<uint32_t*>(&vf[2 * t + (w >> 2)])[w & 3] &= keep;
        }
      }
    }
    bf16x8 p[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mx = s[rt][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[rt][i]);
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      if (__any(mx > m[rt])) {
        const float mn = fmaxf(m[rt], mx);
        const float al = m[rt] == -INFINITY ? (mn == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(m[rt] - mn);
        m[rt] = mn;
        l[rt] *= al;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[rt][t][i] *= al;
      }
      const float mu = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = __builtin_amdgcn_exp2f(s[rt][8 * u + i] - mu);
          l[rt] += e;
          float w = e;
          // (a slot's scale counts for the rows that see it alone)
          if constexpr (Q8) w = edge && !(sees[rt] >> (8 * u + i) & 1) ? 0.f : e * vs[8 * u + i];
          // p is rounded to bf16, the product's type: half a step of 2^-8 at random signs over the
          // keys, less than the output's own rounding
          p[rt][u][i] = (__bf16)w;
        }
    }
    if constexpr (!Q8) {
      // A drafted token's value may hold an infinity or a NaN that only some rows see; 0 * inf would
      // hand it to all of them.  Such values are taken out of the product and added to the rows that
      // see them: as many +inf (NaN: both signs) as there are, found by a product of indicators.
      bool bad = false;
      if (edge) {
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t z = reinterpret_cast<uint32_t*>(&vf[j])[w];
            bad |= (z & 0x7f80u) == 0x7f80u || (z & 0x7f800000u) == 0x7f800000u;
          }
      }
      if (__any(bad)) {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
#pragma unroll
          for (int sg = 0; sg < 2; ++sg) {
            bf16x8 ind[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t z = reinterpret_cast<const uint32_t*>(&vf[2 * t + u])[i >> 1] >> (16 * (i & 1)) & 0xffff;
                const bool nan = (z & 0x7fff) > 0x7f80, inf = z == (sg ? 0xff80u : 0x7f80u);
                ind[u][i] = nan || inf ? (__bf16)1.0f : (__bf16)0.0f;
              }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              f32x16 cnt;
#pragma unroll
              for (int i = 0; i < 16; ++i) cnt[i] = 0.f;
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                bf16x8 one;
#pragma unroll
                for (int i = 0; i < 8; ++i) one[i] = sees[rt] >> (8 * u + i) & 1 ? (__bf16)1.0f : (__bf16)0.0f;
                cnt = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ind[u], one, cnt, 0, 0, 0);
              }
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (cnt[i] > 0.f) o[rt][t][i] += sg ? -INFINITY : INFINITY;
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t& z = reinterpret_cast<uint32_t*>(&vf[2 * t + u])[w];
              if ((z & 0x7f80u) == 0x7f80u) z &= 0xffff0000u;
              if ((z & 0x7f800000u) == 0x7f800000u) z &= 0xffffu;
            }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8 v = v_frag(vf, t, u);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, p[rt][u], o[rt][t], 0, 0, 0);
      }
    load_v(nxt, vf);
  }

  // ---- the block's 4 waves into one (m, l, o), in wave order ----
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += __shfl_xor(l[rt], 32, 64);
    if (h == 0) {
      mls[wave][rt * 32 + n][0] = m[rt];
      mls[wave][rt * 32 + n][1] = l[rt];
    }
  }
  __syncthreads();
  float* po = a.part + ((size_t)((size_t)x * Hkv + hkv) * RB + rb) * (32 * RT) * (D + 2);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float M = -INFINITY, L = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, mls[w][rt * 32 + n][0]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = mls[w][rt * 32 + n][0];
      f[w] = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
      L += mls[w][rt * 32 + n][1] * f[w];
    }
    const float mine = wave == 0 ? f[0] : wave == 1 ? f[1] : wave == 2 ? f[2] : f[3];
    // (a row that saw nothing is 0; one block's row is divided here, a split one's by the join)
    const float sc = sp.ns > 1 ? mine : L == 0.f ? 0.f : mine / L;
    if (sp.ns > 1 && wave == 0 && h == 0) {
      po[(size_t)(32 * RT) * D + (rt * 32 + n) * 2] = M;
      po[(size_t)(32 * RT) * D + (rt * 32 + n) * 2 + 1] = L;
    }
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += OW) {
#pragma unroll
      for (int t = 0; t < OW / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const f32x16& v = o[rt][d0 / 32 + t];
          *reinterpret_cast<float4*>(&os[wave][n][32 * t + 2 * i + 4 * h]) =
              make_float4(v[i] * sc, v[i + 1] * sc, v[i + 2] * sc, v[i + 3] * sc);
        }
      __syncthreads();
#pragma unroll
      for (int q = threadIdx.x; q < 32 * OW / 4; q += 256) {
        const int row = q / (OW / 4), d = q % (OW / 4) * 4, r = r0 + rt * 32 + row;
        float4 y = *reinterpret_cast<const float4*>(&os[0][row][d]);
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float4 z = *reinterpret_cast<const float4*>(&os[w][row][d]);
          y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
        if (r < R) {
          if (sp.ns > 1) {
            *reinterpret_cast<float4*>(po + (size_t)(rt * 32 + row) * D + d0 + d) = y;
          } else {
            const int t = r / G;
            bf16_t* dst = a.out + ((size_t)b * a.T + t) * a.ldo + (size_t)(hkv * G + r - t * G) * D + d0 + d;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(y.x, y.y), pack2(y.z, y.w));
          }
        }
      }
      __syncthreads();
    }
  }
}

// Joins the splits of a row: a wave per (token, q head), partials in split order.
template <int D>
__global__ __launch_bounds__(256) void attn_kv_join(AttnKvArgs a, int NS, int RB, int rows) {
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (int64_t)a.B * a.T * a.Hq) return;
  const int hq = (int)(w % a.Hq), t = (int)(w / a.Hq % a.T), b = (int)(w / a.Hq / a.T);
  if (t >= row_len(a, b).n) return;
  const Split sp = find_split(a, NS, -1, b);
  if (sp.ns == 1) return;
  const int G = a.Hq / a.c.n_kv, hkv = hq / G, r = t * G + hq % G, rb = r / rows, rr = r % rows;
  const size_t step = (size_t)a.c.n_kv * RB * rows * (D + 2);  // from one split to the next
  const float* p = a.part + ((size_t)((size_t)sp.x0 * a.c.n_kv + hkv) * RB + rb) * rows * (D + 2);
  float M = -INFINITY, L = 0.f;
  for (int s = lane; s < sp.ns; s += 64) M = fmaxf(M, p[s * step + (size_t)rows * D + rr * 2]);
  M = wave_max(M);
  constexpr int E = D > 64 ? 2 : 1;  // dims a lane
  float y[E];
#pragma unroll
  for (int e = 0; e < E; ++e) y[e] = 0.f;
  for (int s0 = 0; s0 < sp.ns; s0 += 64) {
    float f = 0.f;
    if (s0 + lane < sp.ns) {
      const float* ml = p + (s0 + lane) * step + (size_t)rows * D + rr * 2;
      f = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - M);
      L += f * ml[1];
    }
    const int n = min(64, sp.ns - s0);
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float fs = __shfl(f, s, 64);
      const float* src = p + (s0 + s) * step + (size_t)rr * D + lane * E;
      if (D >= 64 || lane < D) {
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] += fs * src[e];
      }
    }
  }
  L = wave_sum(L);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  bf16_t* dst = a.out + ((size_t)b * a.T + t) * a.ldo + (size_t)hq * D + lane * E;
  if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = pack2(y[0] * inv, y[1] * inv);
  else if (D >= 64 || lane < D) *dst = f2bf(y[0] * inv);
}

// The launch: row tiles of 32 a wave (RT), row blocks and splits.  RT 2 halves the loads of a key for
// trees of more than 32 rows a KV head.
struct AkvPlan {
  int RT, RB, NS;
};
static AkvPlan plan(int B, int T, int Hq, int n_kv, int slots, int max_len) {
  AkvPlan p;
  const int64_t R = (int64_t)T * (Hq / n_kv);
  p.RT = R > 32 ? 2 : 1;
  p.RB = (int)((R + 32 * p.RT - 1) / (32 * p.RT));
  // enough blocks for every CU to hold two (RT 2: one), no split under 4 tiles of the longest row
  const int64_t want = (p.RT == 1 ? 512 : 256) / std::max<int64_t>(1, (int64_t)n_kv * p.RB);
  const int64_t len = std::min<int64_t>(slots, (int64_t)(max_len > 0 ? std::min(max_len, slots) : slots) + T);
  const int64_t most = (int64_t)B * std::max<int64_t>(1, ((len + 31) / 32 + 3) / 4);
  p.NS = (int)std::max<int64_t>(B, std::min(want, most));
  return p;
}

size_t attn_kv_ws_bytes(int B, int T, int Hq, int n_kv, int D, int slots, int max_len) {
  const AkvPlan p = plan(B, T, Hq, n_kv, slots, max_len);
  if (p.NS <= B) return 0;
  return (size_t)p.NS * n_kv * p.RB * 32 * p.RT * (D + 2) * sizeof(float);
}

template <int KT, int D>
static hipError_t launch(const AttnKvArgs& a, const AkvPlan& p, hipStream_t s) {
  const int64_t grid = ((int64_t)p.NS * a.c.n_kv + 7) / 8 * 8 * p.RB;
  if (grid > INT_MAX) return hipErrorInvalidValue;
  if (p.RT == 1) hipLaunchKernelGGL((attn_kv_kernel<KT, D, 1>), dim3((unsigned)grid), dim3(256), 0, s, a, p.NS, p.RB);
  else hipLaunchKernelGGL((attn_kv_kernel<KT, D, 2>), dim3((unsigned)grid), dim3(256), 0, s, a, p.NS, p.RB);
  if (p.NS > a.B) {
    const int64_t waves = (int64_t)a.B * a.T * a.Hq;
    if ((waves + 3) / 4 > INT_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL(attn_kv_join<D>, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s, a, p.NS, p.RB, 32 * p.RT);
  }
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
