// Rotary positions, and the 8-bit key / value cache: append (head norm, rotation, quantisation),
// read back, and the compaction of an accepted path (layouts: kvq.h).
#include "kvq.h"

namespace mtts {

// ---------------------------------------------------------------------------
// Rotation.  Pair i of a head at position p turns by p * turns[i] revolutions; the product is taken
// in 64 bits and only its fraction of a turn kept, so a position of 131,071 loses nothing to the
// 32-bit range.
__device__ __forceinline__ void rope_cs(double turns, int pos, float factor, float* c, float* s) {
  double r = turns * (double)pos;
  r -= rint(r);
  float sn, cs;
  sincospif(2.0f * (float)r, &sn, &cs);
  *c = cs * factor;
  *s = sn * factor;
}

// A thread holds V pairs of a head, 2 V values: x[0..V) are dims d0.. and x[V..2V) dims d1..
// (V = 8: two 16-byte pieces; V = 1: any even rot).  Half layout: pair (x[k], x[V + k]);
// interleaved: (x[2k], x[2k + 1]).  Chunks past the rotary dims pass through.
template <int V>
struct Chunk {
  int d0, d1;
  bool rot;
  __device__ __forceinline__ Chunk(const RopeView& r, int c) {
    rot = 2 * V * c < r.rot;
    const bool half = rot && !r.interleaved;
    d0 = half ? V * c : 2 * V * c;
    d1 = half ? r.rot / 2 + V * c : d0 + V;
  }
};

template <int V>
__device__ __forceinline__ void load_pieces(const bf16_t* row, const Chunk<V>& ch, float* x) {
  if constexpr (V == 8) {
    unpack8(*reinterpret_cast<const uint4*>(row + ch.d0), x);
    unpack8(*reinterpret_cast<const uint4*>(row + ch.d1), x + 8);
  } else {
    x[0] = bf2f(row[ch.d0]);
    x[1] = bf2f(row[ch.d1]);
  }
}
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
}
template <int V>
__device__ __forceinline__ void store_pieces(bf16_t* row, const Chunk<V>& ch, const float* x) {
  if constexpr (V == 8) {
    *reinterpret_cast<uint4*>(row + ch.d0) = pack8(x);
    *reinterpret_cast<uint4*>(row + ch.d1) = pack8(x + 8);
  } else {
    row[ch.d0] = f2bf(x[0]);
    row[ch.d1] = f2bf(x[1]);
  }
}

template <int V>
__device__ __forceinline__ void rope_angles(const RopeView& r, int c, int pos, float* cs, float* sn) {
#pragma unroll
  for (int k = 0; k < V; ++k) rope_cs(r.turns[V * c + k], pos, r.factor, &cs[k], &sn[k]);
}
template <int V>
__device__ __forceinline__ void rotate(const RopeView& r, const float* cs, const float* sn, float* x) {
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int i = r.interleaved ? 2 * k : k, j = r.interleaved ? 2 * k + 1 : V + k;
    const float a = x[i], b = x[j];
    x[i] = fmaf(a, cs[k], -(b * sn[k]));
    x[j] = fmaf(b, cs[k], a * sn[k]);
  }
}

// One wave per (token, run of hpc heads): D / (2 V) lanes a head, the wave's other lanes the next
// heads; a lane's angles (64-bit products, the sine and cosine: more work than the rotation) are computed
// once and used for all its heads.  Bound by its bytes: 6,001 tokens of 40 heads of 128, 123 MB, 22 us
// (5.6 TB/s; a large copy reaches 4.9); 4 tokens 3.7 us, which is a launch.
template <int V>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int hpc) {
  const int lane = threadIdx.x & 63;
  const int runs = (a.H + hpc - 1) / hpc;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (int64_t)a.M * runs) return;
  const int m = (int)(w / runs), h0 = (int)(w % runs) * hpc, h1 = min(h0 + hpc, a.H);
  const int pt = a.D / (2 * V);  // lanes a head
  const bf16_t* x = a.x + (size_t)m * a.ldx;
  bf16_t* y = a.y + (size_t)m * a.ldy;
  const int pos = a.pos[m];
  // (a head of more than 64 lanes is walked in 64-lane steps)
  const int step = pt < 64 ? 64 / pt : 1;
  for (int c = pt < 64 ? lane % pt : lane; c < pt; c += 64) {
    if (pt < 64 && lane / pt >= step) break;  // lanes that no whole head fills
    const Chunk<V> ch(a.r, c);
    if (!ch.rot && a.x == a.y) continue;
    float cs[V], sn[V];
    if (ch.rot) rope_angles<V>(a.r, c, pos, cs, sn);
    for (int h = h0 + (pt < 64 ? lane / pt : 0); h < h1; h += step) {
      float v[2 * V];
      load_pieces<V>(x + (size_t)h * a.hsx, ch, v);
      if (ch.rot) rotate<V>(a.r, cs, sn, v);
      store_pieces<V>(y + (size_t)h * a.hsy, ch, v);
    }
  }
}

static inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

hipError_t rope_apply(const RopeArgs& a, hipStream_t s) {
  if (a.M == 0 || a.H == 0) return hipSuccess;
  const bool v8 = a.r.rot % 16 == 0 && a.D % 16 == 0 && a.ldx % 8 == 0 && a.ldy % 8 == 0 && a.hsx % 8 == 0 &&
                  a.hsy % 8 == 0 && al16(a.x) && al16(a.y);
  const int per = v8 ? (a.D >= 1024 ? 1 : 1024 / a.D) : (a.D >= 128 ? 1 : 128 / a.D);  // heads a wave holds at once
  int hpc = per;
  while (hpc < a.H && (int64_t)a.M * ((a.H + hpc - 1) / hpc) > 4096) hpc += per;
  const int64_t waves = (int64_t)a.M * ((a.H + hpc - 1) / hpc);
  if ((waves + 3) / 4 > INT_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)((waves + 3) / 4));
  if (v8) hipLaunchKernelGGL(rope_kernel<8>, grid, dim3(256), 0, s, a, hpc);
  else hipLaunchKernelGGL(rope_kernel<1>, grid, dim3(256), 0, s, a, hpc);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Quantisation of a (slot, head) row: with the row's largest magnitude a and Q = 448 (e4m3) or 127
// (int8), code = nearest(x Q / a), ties to even, and scale = a / Q; the value is code * scale.
// x Q is exact for bf16 x, and the quotient is rounded correctly (one residual step behind the
// product with the rounded reciprocal), so a tie stays a tie.  Rows with a < 2^-100 are stored as
// zeros; a row that holds a NaN or an infinity is stored as NaN in whole (scale NaN, codes 0): a
// code of such a slot never reaches a sum of another.
struct Quant {
  float q, a, rcp, scale;
  bool live;
  __device__ __forceinline__ Quant(float amax, int type) {
    const float Q = type == KV_E4M3 ? 448.f : 127.f;
    live = amax >= 0x1p-100f && amax < INFINITY;
    // (large rows are shifted by 2^-64, so x Q stays finite)
    const float sh = amax > 0x1p100f ? 0x1p-64f : 1.f;
    q = Q * sh;
    a = live ? amax * sh : 1.f;
    rcp = 1.f / a;
    scale = amax < 0x1p-100f ? 0.f : live ? amax / Q : __builtin_nanf("");
  }
  __device__ __forceinline__ float at(float x, int type) const {
    const float n = x * q, p = n * rcp;
    const float y = fmaf(fmaf(-p, a, n), rcp, p);
    const float Q = type == KV_E4M3 ? 448.f : 127.f;
    return live ? fminf(fmaxf(y, -Q), Q) : 0.f;
  }
};
// the codes of four values, one byte each
__device__ __forceinline__ uint32_t codes4(const Quant& z, const float* x, int type) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = z.at(x[i], type);
  if (type == KV_E4M3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)rintf(y[i]) & 0xffu) << (8 * i);
  return w;
}
__device__ __forceinline__ uint8_t code1(const Quant& z, float x, int type) {
  const float y = z.at(x, type);
  if (type == KV_E4M3) return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xff);
  return (uint8_t)((int)rintf(y) & 0xff);
}
// the four values of a word of codes
__device__ __forceinline__ void values4(uint32_t w, int type, float* x) {
  if (type == KV_E4M3) {
    typedef __attribute__((ext_vector_type(2))) float f32x2;
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = lo.x; x[1] = lo.y; x[2] = hi.x; x[3] = hi.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
}
// max |x| that a NaN wins
__device__ __forceinline__ float amax_nan(float a, float x) {
  x = fabsf(x);
  return x > a || x != x ? x : a;
}

__device__ __forceinline__ int row_count(const int* counts, int b, int S) {
  return counts ? min(max(counts[b], 0), S) : S;
}

// Append.  Three kinds of blocks in one launch:
//   [0, nq)    q: a wave per (token, run of heads): norm, rotation, q_out
//   [.., +nk)  k: a block per (row, kv head, tile of 32 slots): norm, rotation, amax over the head's lanes,
//              codes through LDS into the tile's order, so that they leave in 16-byte pieces side by side
//   [.., +nk)  v: the same; a V tile holds 16 slots of one dim side by side
// One launch, so that a decode step pays once.  Rows of 2,117, 1,882 and 1,647 tokens, 32 q and 8 + 8 k and v
// heads of 128, to e4m3: 128 MB in 33.4 us (3.8 TB/s, where a large copy reaches 4.9; each K block computes
// its tokens' angles in 64 bits, their sines and cosines for its own KV head, so 8 times in all, and the rows'
// last tiles are partly empty); one token 5.4 us, of which the chain load, sum, angle, amax, store is most.
template <int V>
__device__ __forceinline__ float head_sum(float s, int pt) {
  for (int o = 1; o < pt; o <<= 1) s += __shfl_xor(s, o, 64);
  return s;
}
template <int V>
__device__ __forceinline__ void head_norm(float* x, const float* w, int pt, int D, float eps) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 2 * V; ++i) s = fmaf(x[i], x[i], s);
  const float r = 1.0f / sqrtf(head_sum<V>(s, pt) / (float)D + eps);
#pragma unroll
  for (int i = 0; i < 2 * V; ++i) x[i] *= r * w[i];
}

template <int V>
__device__ void append_q(const KvAppendArgs& a, int blk, int hpc) {
  const int D = a.c.D, pt = D / (2 * V), lane = threadIdx.x & 63, c = lane % pt;
  const int runs = (a.H + hpc - 1) / hpc;
  const int64_t w = (int64_t)blk * 4 + (threadIdx.x >> 6);
  if (w >= (int64_t)a.B * a.S * runs) return;
  const int m = (int)(w / runs), h0 = (int)(w % runs) * hpc, h1 = min(h0 + hpc, a.H);
  const int b = m / a.S, t = m - b * a.S;
  if (t >= row_count(a.counts, b, a.S)) return;
  const Chunk<V> ch(a.r, c);
  float cs[V], sn[V], nw[2 * V];
  if (ch.rot) rope_angles<V>(a.r, c, a.pos ? a.pos[m] : (int)((int64_t)a.start[b] + t), cs, sn);
  if (a.qn) load_pieces<V>(a.qn, ch, nw);
  const bf16_t* src = a.q + (size_t)m * a.ldq;
  bf16_t* dst = a.q_out + (size_t)m * a.ldqo;
  // (every lane of the wave takes the same number of turns: the norm's shuffles need them all)
  for (int h = h0; h < h1; h += 64 / pt) {
    const int hh = h + lane / pt;
    const bool on = hh < h1;
    float x[2 * V];
    load_pieces<V>(src + (size_t)(on ? hh : h0) * D, ch, x);
    if (a.qn) head_norm<V>(x, nw, pt, D, a.eps);
    if (ch.rot) rotate<V>(a.r, cs, sn, x);
    if (on) store_pieces<V>(dst + (size_t)hh * D, ch, x);
  }
}

constexpr int KV_DMAX = 128;

// the tile of 32 slots that K or V block `blk` works on: new tokens at its slots [lo, hi); false: none
struct KvTile {
  int b, h, start, lo, hi;
  int64_t base;  // its first slot
  size_t head;
};
__device__ __forceinline__ bool kv_tile(const KvAppendArgs& a, int blk, KvTile* t) {
  const int tiles = (a.S + 31) / 32 + 1;  // a row's new slots touch this many tiles at most
  t->b = blk / (tiles * a.c.n_kv);
  t->h = blk / tiles % a.c.n_kv;
  t->start = a.start[t->b];
  const int64_t end = (int64_t)t->start + row_count(a.counts, t->b, a.S);
  t->base = ((int64_t)(t->start >> 5) + blk % tiles) * 32;
  if (t->base < 0 || t->base >= a.c.slots || t->base >= end) return false;
  t->lo = (int)max((int64_t)0, t->start - t->base);
  t->hi = (int)min((int64_t)32, end - t->base);
  t->head = ((size_t)t->b * a.c.n_kv + t->h) * a.c.slots;
  return true;
}

// pieces of 2 V dims of one token each
template <int V>
__device__ void append_k(const KvAppendArgs& a, int blk, char* lds) {
  KvTile t;
  if (!kv_tile(a, blk, &t)) return;
  const int D = a.c.D, pt = D / (2 * V);
  for (int i = threadIdx.x; i < 32 * pt; i += 256) {  // (32 pt is a multiple of 64: whole waves)
    const int j = i / pt, c = i % pt;
    const bool on = j >= t.lo && j < t.hi;
    if (!__any(on)) continue;
    const int64_t slot = t.base + j;
    const size_t m = (size_t)t.b * a.S + (on ? slot - t.start : 0);
    const Chunk<V> ch(a.r, c);
    float x[2 * V];
    load_pieces<V>(a.k + m * a.ldk + (size_t)t.h * D, ch, x);
    if (a.kn) {
      float nw[2 * V];
      load_pieces<V>(a.kn, ch, nw);
      head_norm<V>(x, nw, pt, D, a.eps);
    }
    if (ch.rot) {
      float cs[V], sn[V];
      rope_angles<V>(a.r, c, a.pos ? a.pos[m] : (int)slot, cs, sn);
      rotate<V>(a.r, cs, sn, x);
    }
    if (a.c.type == KV_BF16) {
      if (on) store_pieces<V>((bf16_t*)a.c.k + (t.head + slot) * D, ch, x);
      continue;
    }
    float am = 0.f;
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) am = amax_nan(am, x[k]);
    for (int o = 1; o < pt; o <<= 1) am = amax_nan(am, __shfl_xor(am, o, 64));
    const Quant z(am, a.c.type);
    if constexpr (V == 8) {
      *reinterpret_cast<uint2*>(lds + kv_k_byte(j, ch.d0)) = make_uint2(codes4(z, x, a.c.type), codes4(z, x + 4, a.c.type));
      *reinterpret_cast<uint2*>(lds + kv_k_byte(j, ch.d1)) =
          make_uint2(codes4(z, x + 8, a.c.type), codes4(z, x + 12, a.c.type));
    } else {
      lds[kv_k_byte(j, ch.d0)] = (char)code1(z, x[0], a.c.type);
      lds[kv_k_byte(j, ch.d1)] = (char)code1(z, x[1], a.c.type);
    }
    if (on && c == 0) a.c.ks[t.head + slot] = z.scale;
  }
  if (a.c.type == KV_BF16) return;
  __syncthreads();
  uint8_t* tile = (uint8_t*)a.c.k + (t.head + t.base) * D;
  for (int i = threadIdx.x; i < 2 * D; i += 256) {  // 16 dims of the slot of tile row i % 32
    const int j = kv_slot_of_row(i & 31);
    if (j >= t.lo && j < t.hi) reinterpret_cast<uint4*>(tile)[i] = reinterpret_cast<const uint4*>(lds)[i];
  }
}

// v has no rotation: pieces of 16 dims (V = 8) or of 2, of one token each
template <int V>
__device__ void append_v(const KvAppendArgs& a, int vb, char* lds) {
  KvTile kt;
  if (!kv_tile(a, vb, &kt)) return;
  const int D = a.c.D, b = kt.b, h = kt.h, start = kt.start, lo = kt.lo, hi = kt.hi, pt = D / (2 * V);
  const int64_t base = kt.base;
  const size_t head = kt.head;
  if (a.c.type == KV_BF16) {
    bf16_t(*t)[KV_DMAX + 8] = reinterpret_cast<bf16_t(*)[KV_DMAX + 8]>(lds);
    for (int i = threadIdx.x; i < 32 * pt; i += 256) {
      const int j = i / pt, d = (i % pt) * 2 * V;
      if (j < lo || j >= hi) continue;
      const bf16_t* src = a.v + ((size_t)b * a.S + (base + j - start)) * a.ldv + (size_t)h * D + d;
      if constexpr (V == 8) {
        *reinterpret_cast<uint4*>(&t[j][d]) = *reinterpret_cast<const uint4*>(src);
        *reinterpret_cast<uint4*>(&t[j][d + 8]) = *reinterpret_cast<const uint4*>(src + 8);
      } else {
        t[j][d] = src[0];
        t[j][d + 1] = src[1];
      }
    }
    __syncthreads();
    bf16_t* dst = (bf16_t*)a.c.v + head * D + base;  // row d at + d * slots
    if (lo == 0 && hi == 32) {
      for (int i = threadIdx.x; i < D * 4; i += 256) {
        const int d = i >> 2, j = (i & 3) * 8;
        uint4 o;
        o.x = t[j][d] | (uint32_t)t[j + 1][d] << 16;
        o.y = t[j + 2][d] | (uint32_t)t[j + 3][d] << 16;
        o.z = t[j + 4][d] | (uint32_t)t[j + 5][d] << 16;
        o.w = t[j + 6][d] | (uint32_t)t[j + 7][d] << 16;
        *reinterpret_cast<uint4*>(dst + (size_t)d * a.c.slots + j) = o;
      }
    } else {
      const int nn = hi - lo;
      for (int i = threadIdx.x; i < D * nn; i += 256) {
        const int d = i / nn, j = lo + i % nn;
        dst[(size_t)d * a.c.slots + j] = t[j][d];
      }
    }
    return;
  }
  uint8_t(*t)[KV_DMAX + 4] = reinterpret_cast<uint8_t(*)[KV_DMAX + 4]>(lds);
  for (int i = threadIdx.x; i < 32 * pt; i += 256) {  // (32 pt is a multiple of 64: whole waves)
    const int j = i / pt, d = (i % pt) * 2 * V;
    const bool on = j >= lo && j < hi;
    float x[2 * V];
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) x[k] = 0.f;
    if (on) {
      const bf16_t* src = a.v + ((size_t)b * a.S + (base + j - start)) * a.ldv + (size_t)h * D + d;
      if constexpr (V == 8) {
        unpack8(*reinterpret_cast<const uint4*>(src), x);
        unpack8(*reinterpret_cast<const uint4*>(src + 8), x + 8);
      } else {
        x[0] = bf2f(src[0]);
        x[1] = bf2f(src[1]);
      }
    }
    float am = 0.f;
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) am = amax_nan(am, x[k]);
    for (int o = 1; o < pt; o <<= 1) am = amax_nan(am, __shfl_xor(am, o, 64));
    const Quant z(am, a.c.type);
    if (on) {
      if constexpr (V == 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t*>(&t[j][d + 4 * k]) = codes4(z, x + 4 * k, a.c.type);
      } else {
        t[j][d] = code1(z, x[0], a.c.type);
        t[j][d + 1] = code1(z, x[1], a.c.type);
      }
      if (d == 0) a.c.vs[head + base + j] = z.scale;
    }
  }
  __syncthreads();
  uint8_t* tile = (uint8_t*)a.c.v + (head + base) * D;
  if (lo == 0 && hi == 32) {
    for (int i = threadIdx.x; i < 2 * D; i += 256) {  // 16 bytes: slots 16 u + 8 h + i of one dim
      const int d = (i >> 6) * 32 + (i & 31), hh = (i >> 5) & 1;
      uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 16; ++k) o[k >> 2] |= (uint32_t)t[(k >> 3) * 16 + hh * 8 + (k & 7)][d] << (8 * (k & 3));
      *reinterpret_cast<uint4*>(tile + (size_t)i * 16) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
    const int nn = hi - lo;
    for (int i = threadIdx.x; i < D * nn; i += 256) {
      const int d = i / nn, j = lo + i % nn;
      tile[kv_v_byte(j, d)] = t[j][d];
    }
  }
}

template <int V>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a, int nq, int nk, int hq) {
  __shared__ __attribute__((aligned(16))) char lds[32 * (KV_DMAX + 8) * 2];
  const int blk = blockIdx.x;
  if (blk < nq) append_q<V>(a, blk, hq);
  else if (blk < nq + nk) append_k<V>(a, blk - nq, lds);
  else append_v<V>(a, blk - nq - nk, lds);
}

hipError_t kv_append(const KvAppendArgs& a, hipStream_t s) {
  if (a.B == 0 || a.S == 0) return hipSuccess;
  const int D = a.c.D;
  if (D != 32 && D != 64 && D != 128) return hipErrorInvalidValue;
  const bool v8 = a.r.rot % 16 == 0 && a.ldk % 8 == 0 && a.ldv % 8 == 0 && al16(a.k) && al16(a.v) &&
                  (!a.q || (a.ldq % 8 == 0 && a.ldqo % 8 == 0 && al16(a.q) && al16(a.q_out))) &&
                  (!a.qn || al16(a.qn)) && (!a.kn || al16(a.kn));
  const int pt = D / (v8 ? 16 : 2), tpw = 64 / pt;
  const int64_t M = (int64_t)a.B * a.S;
  int64_t nq = 0;
  int hq = tpw;
  if (a.q) {
    while (hq < a.H && M * ((a.H + hq - 1) / hq) > 4096) hq += tpw;
    nq = (M * ((a.H + hq - 1) / hq) + 3) / 4;
  }
  const int64_t nk = (int64_t)a.B * a.c.n_kv * ((a.S + 31) / 32 + 1);
  if (nq + 2 * nk > INT_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(nq + 2 * nk));
  if (v8) hipLaunchKernelGGL(kv_append_kernel<8>, grid, dim3(256), 0, s, a, (int)nq, (int)nk, hq);
  else hipLaunchKernelGGL(kv_append_kernel<1>, grid, dim3(256), 0, s, a, (int)nq, (int)nk, hq);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Read back: a block per (row, kv head, tile of 32 slots).  Both tiles go through LDS as they lie
// and leave as whole rows of bf16.  Bound by its bytes: 65,536 int8 slots of 8 heads of 128, 407 MB, 73 to
// 81 us (5.0 to 5.6 TB/s).
__global__ __launch_bounds__(256) void kv_read_kernel(KvReadArgs a, int tiles) {
  __shared__ __attribute__((aligned(16))) uint8_t kt[32 * KV_DMAX], vt[32 * KV_DMAX];
  const int D = a.c.D;
  const int b = blockIdx.x / (tiles * a.c.n_kv), h = blockIdx.x / tiles % a.c.n_kv;
  const int start = a.start ? a.start[b] : 0, n = row_count(a.counts, b, a.n);
  const int64_t base = ((int64_t)(start >> 5) + blockIdx.x % tiles) * 32;
  if (base >= (int64_t)start + a.n) return;
  const size_t head = ((size_t)b * a.c.n_kv + h) * a.c.slots;
  const bool in = base >= 0 && base < a.c.slots;
  const int type = a.c.type;
  if (in && type != KV_BF16) {
    const uint4* k = reinterpret_cast<const uint4*>((const uint8_t*)a.c.k + (head + base) * D);
    const uint4* v = reinterpret_cast<const uint4*>((const uint8_t*)a.c.v + (head + base) * D);
    for (int i = threadIdx.x; i < 2 * D; i += 256) {
      reinterpret_cast<uint4*>(kt)[i] = k[i];
      reinterpret_cast<uint4*>(vt)[i] = v[i];
    }
  }
  __syncthreads();
  const int pt = D / 16;
  for (int i = threadIdx.x; i < 32 * pt; i += 256) {
    const int j = i / pt, d = (i % pt) * 16;
    const int64_t o = base + j - start;  // the output row
    if (o < 0 || o >= a.n) continue;
    float k[16], v[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) k[x] = v[x] = 0.f;
    if (in && o < n) {
      if (type == KV_BF16) {
        const bf16_t* ks = (const bf16_t*)a.c.k + (head + base + j) * D + d;
        unpack8(*reinterpret_cast<const uint4*>(ks), k);
        unpack8(*reinterpret_cast<const uint4*>(ks + 8), k + 8);
        const bf16_t* vs = (const bf16_t*)a.c.v + head * D + base + j;
#pragma unroll
        for (int x = 0; x < 16; ++x) v[x] = bf2f(vs[(size_t)(d + x) * a.c.slots]);
      } else {
        const float ks = a.c.ks[head + base + j], vs = a.c.vs[head + base + j];
        const uint4 w = *reinterpret_cast<const uint4*>(kt + kv_k_byte(j, d));
        values4(w.x, type, k); values4(w.y, type, k + 4); values4(w.z, type, k + 8); values4(w.w, type, k + 12);
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
          uint32_t c = 0;
#pragma unroll
          for (int y = 0; y < 4; ++y) c |= (uint32_t)vt[kv_v_byte(j, d + x + y)] << (8 * y);
          values4(c, type, v + x);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          k[x] *= ks;
          v[x] *= vs;
        }
      }
    }
    const size_t at = (((size_t)b * a.c.n_kv + h) * a.n + o) * D + d;
    *reinterpret_cast<uint4*>(a.k + at) = pack8(k);
    *reinterpret_cast<uint4*>(a.k + at + 8) = pack8(k + 8);
    *reinterpret_cast<uint4*>(a.v + at) = pack8(v);
    *reinterpret_cast<uint4*>(a.v + at + 8) = pack8(v + 8);
  }
}

hipError_t kv_read(const KvReadArgs& a, hipStream_t s) {
  if (a.B == 0 || a.n == 0) return hipSuccess;
  if (a.c.D != 32 && a.c.D != 64 && a.c.D != 128) return hipErrorInvalidValue;
  const int tiles = (a.n + 31) / 32 + 1;
  const int64_t grid = (int64_t)a.B * a.c.n_kv * tiles;
  if (grid > INT_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)grid), dim3(256), 0, s, a, tiles);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Compaction: slot start + i <- slot start + path[i], i < took.  A block owns the K or the V of one
// (row, kv head) and reads every source before it writes any slot, so paths may overlap their destinations
// in any order.  An entry whose source or destination is no slot is left out.  K moves in 16-byte pieces.
// V has its slots side by side, so the window of slots that a path can touch goes through LDS in 16-byte
// pieces (a piece at an edge writes the slots beside the window back as they were): byte by byte, 64 rows
// of 64 tokens took 14.5 us; they take 9.2 (8 int8 heads of 128, about half of the tokens kept; the window is
// read and written whatever the path is, in one dependent chain a block).  1 row of 16 tokens 4.4, two
// dependent loads and a launch.
constexpr int KV_WIN = KV_PATH_MAX + 32;  // slots of the window: whole tiles (8-bit), or pieces of 8 (bf16)
__global__ __launch_bounds__(256) void kv_compact_kernel(KvCompactArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t win[KV_DMAX * (KV_PATH_MAX + 8) * 2];
  __shared__ int from[KV_PATH_MAX];  // the slot that entry i takes, -1: none
  const int D = a.c.D, unit = blockIdx.x >> 1, isv = blockIdx.x & 1, tid = threadIdx.x;
  const int b = unit / a.c.n_kv;
  const int start = a.start[b], n = min(max(a.took[b], 0), a.P), slots = a.c.slots;
  if (n == 0 || start >= slots) return;  // (nothing of a path behind the cache is a slot)
  const size_t head = (size_t)unit * slots;  // unit = b * n_kv + h
  const bool bf = a.c.type == KV_BF16;
  float* scales = isv ? a.c.vs : a.c.ks;
  float sc = 0.f;
  if (tid < n) {
    const int p = a.path[(size_t)b * a.P + tid];
    const int64_t f = (int64_t)start + p, t = (int64_t)start + tid;
    const bool ok = p >= 0 && p < KV_PATH_MAX && f >= 0 && f < slots && t >= 0 && t < slots;
    from[tid] = ok ? (int)f : -1;
    if (ok && !bf) sc = scales[head + f];
  }
  __syncthreads();
  if (!isv) {
    const int np = bf ? D / 8 : D / 16;  // pieces a slot
    uint8_t* k = (uint8_t*)a.c.k;
    auto at = [&](int slot, int c) -> u32x4* {
      return bf ? reinterpret_cast<u32x4*>(k + ((head + slot) * D + c * 8) * 2)
                : reinterpret_cast<u32x4*>(k + (head + (slot & ~31)) * D + kv_k_byte(slot & 31, c * 16));
    };
    u32x4 x[4];  // KV_PATH_MAX * KV_DMAX / 8 / 256
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid + 256 * j, e = i / np;
      if (e < n && from[e] >= 0) x[j] = *at(from[e], i - e * np);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid + 256 * j, e = i / np;
      if (e < n && from[e] >= 0) *at(start + e, i - e * np) = x[j];
    }
  } else if (bf) {
    // [D][KV_PATH_MAX + 8] values from slot `lo` on
    constexpr int NW = KV_PATH_MAX + 8;
    const int lo = max(start, 0) & ~7;
    bf16_t* w = reinterpret_cast<bf16_t*>(win);
    bf16_t* v = (bf16_t*)a.c.v + head * D + lo;
    for (int i = tid; i < D * (NW / 8); i += 256) {
      const int d = i / (NW / 8), c = i % (NW / 8) * 8;
      if (lo + c < slots) *reinterpret_cast<uint4*>(w + d * NW + c) = *reinterpret_cast<const uint4*>(v + (size_t)d * slots + c);
    }
    __syncthreads();
    for (int i = tid; i < D * (NW / 8); i += 256) {
      const int d = i / (NW / 8), c = i % (NW / 8) * 8;
      if (lo + c >= slots || lo + c >= (int64_t)start + n) continue;
      uint32_t o[4];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const int e = lo + c + y - start;
        const int f = e >= 0 && e < n && from[e] >= 0 ? from[e] - lo : c + y;
        const uint32_t z = w[d * NW + f];
        o[y >> 1] = y & 1 ? o[y >> 1] | z << 16 : z;
      }
      *reinterpret_cast<uint4*>(v + (size_t)d * slots + c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
    // the window's tiles as they lie
    const int t0 = max(start, 0) & ~31, nt = min(KV_WIN, slots - t0) >> 5;
    uint8_t* v = (uint8_t*)a.c.v + (head + t0) * D;
    for (int i = tid; i < nt * 2 * D; i += 256) reinterpret_cast<uint4*>(win)[i] = reinterpret_cast<const uint4*>(v)[i];
    __syncthreads();
    for (int i = tid; i < nt * 2 * D; i += 256) {
      const int tile = i / (2 * D), j = i - tile * 2 * D;  // 16 bytes: slots 16 u + 8 h + y of one dim
      if (t0 + tile * 32 >= (int64_t)start + n) break;
      const int d = (j >> 6) * 32 + (j & 31), hh = (j >> 5) & 1;
      uint32_t o[4] = {0, 0, 0, 0};
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const int s = tile * 32 + (y >> 3) * 16 + hh * 8 + (y & 7), e = t0 + s - start;
        const int f = e >= 0 && e < n && from[e] >= 0 ? from[e] - t0 : s;
        o[y >> 2] |= (uint32_t)win[(f >> 5) * 32 * D + kv_v_byte(f & 31, d)] << (8 * (y & 3));
      }
      reinterpret_cast<uint4*>(v)[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
  if (!bf && tid < n && from[tid] >= 0) scales[head + start + tid] = sc;
}

hipError_t kv_compact(const KvCompactArgs& a, hipStream_t s) {
  if (a.B == 0 || a.P == 0) return hipSuccess;
  if (a.P > KV_PATH_MAX || (a.c.D != 32 && a.c.D != 64 && a.c.D != 128)) return hipErrorInvalidValue;
  const int64_t grid = (int64_t)a.B * a.c.n_kv * 2;
  if (grid > INT_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kv_compact_kernel, dim3((unsigned)grid), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace mtts
