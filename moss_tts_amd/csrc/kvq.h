// The key / value cache of the drafted-token operators (kvcache.hip, attn_kv.hip): types, layouts
// and the launch entry points.
//
// MTTS_KV_BF16 is the layout of the engine's own cache: K [rows][n_kv][slots][D], V transposed
// [rows][n_kv][D][slots], bf16, no scales.
//
// MTTS_KV_E4M3 / MTTS_KV_INT8 hold one byte a value and one fp32 scale a (slot, head) for each of K
// and V, and lay the bytes out in tiles of 32 slots, in the order in which the attention's matrix
// instruction takes them: a wave's load of a fragment is ONE contiguous KiB.  A slot s of a tile is
// s % 32 = 16 u + 8 h + i (i < 8).
//   K  byte ((d / 16) 32 + m) 16 + d % 16 of the tile, m = 16 u + 8 (i / 4) + 4 h + i % 4: the row of
//      the 32x32 score tile whose results lane half h holds as its registers 8 u + i
//   V  byte ((d / 32) 64 + 32 h + d % 32) 16 + 8 u + i: the 16 slots that lane half h multiplies, for
//      one dim
// A tile is 32 D bytes of K and as many of V; slots is a multiple of 32.
#pragma once
#include "common.h"

namespace mtts {

enum KvType { KV_BF16 = 0, KV_E4M3 = 1, KV_INT8 = 2 };

struct KvView {
  void *k, *v;
  float *ks, *vs;  // [rows][n_kv][slots] (8-bit types)
  int type, rows, n_kv, D, slots;
};

// the 32-slot tile row (m) that slot kappa = slot % 32 has in the score tile, and back
__host__ __device__ inline int kv_row_of_slot(int kappa) {
  return (kappa & 0x10) | ((kappa & 4) << 1) | ((kappa & 8) >> 1) | (kappa & 3);
}
__host__ __device__ inline int kv_slot_of_row(int m) {
  return (m & 0x10) | ((m & 8) >> 1) | ((m & 4) << 1) | (m & 3);
}
// byte offsets inside a tile
__host__ __device__ inline int kv_k_byte(int kappa, int d) {
  return ((d >> 4) * 32 + kv_row_of_slot(kappa)) * 16 + (d & 15);
}
__host__ __device__ inline int kv_v_byte(int kappa, int d) {
  return ((d >> 5) * 64 + ((kappa >> 3) & 1) * 32 + (d & 31)) * 16 + (kappa >> 4) * 8 + (kappa & 7);
}

struct RopeView {
  const double* turns;  // device [rot / 2]: revolutions per position of each pair
  int rot, interleaved;
  float factor;         // on the rotated values
};

struct RopeArgs {
  const bf16_t* x;
  bf16_t* y;
  size_t ldx, hsx, ldy, hsy;  // elements between tokens and between heads
  const int* pos;             // device [M]
  int M, H, D;
  RopeView r;
};
hipError_t rope_apply(const RopeArgs& a, hipStream_t s);

struct KvAppendArgs {
  KvView c;
  const bf16_t *q, *k, *v;  // token m = b * S + t at + m * ld; heads D apart; q may be null
  size_t ldq, ldk, ldv;
  bf16_t* q_out;            // [.., H, D], tokens ldqo apart
  size_t ldqo;
  int H;                    // q heads
  const bf16_t *qn, *kn;    // head norm weights or null
  float eps;
  RopeView r;               // r.rot == 0: no rotation
  const int* pos;           // device [B * S], or null: the slot
  const int* start;         // device [B]
  const int* counts;        // device [B] or null: S
  int B, S;
};
hipError_t kv_append(const KvAppendArgs& a, hipStream_t s);

struct KvReadArgs {
  KvView c;
  bf16_t *k, *v;      // [B][n_kv][n][D], contiguous
  const int* start;   // device [B] or null: 0
  const int* counts;  // device [B] or null: n
  int B, n;
};
hipError_t kv_read(const KvReadArgs& a, hipStream_t s);

constexpr int KV_PATH_MAX = 64;
struct KvCompactArgs {
  KvView c;
  const int* start;  // device [B]
  const int* path;   // device [B][P]
  const int* took;   // device [B]
  int B, P;
};
hipError_t kv_compact(const KvCompactArgs& a, hipStream_t s);

constexpr int KV_TREE_MAX = 64;
struct AttnKvArgs {
  KvView c;
  const bf16_t* q;    // [B * T tokens ldq apart][Hq][D]
  bf16_t* out;        // [B * T tokens ldo apart][Hq][D]
  size_t ldq, ldo;
  const uint8_t* mask;   // [B][slots] or null
  const int* start;      // device [B]
  const int* counts;     // device [B] or null: T
  const uint64_t* tree;  // device [B][T] or null: token t sees new tokens 0..t
  float* part;           // attn_kv_ws_bytes
  int B, T, Hq;
  float scale;
  int max_len;           // an upper bound of start the caller knows, <= 0: slots
};
size_t attn_kv_ws_bytes(int B, int T, int Hq, int n_kv, int D, int slots, int max_len);
hipError_t attn_kv(const AttnKvArgs& a, hipStream_t s);

}  // namespace mtts
