"""Drafted-token decoding over an 8-bit key / value cache: rotary positions, the cache, and the
attention that reads it.

    rope = Rope(128, theta=1e6, scaling={"rope_type": "yarn", "factor": 4.0,
                                         "original_max_position_embeddings": 32768})
    cache = KVCache(rows=4, n_kv=8, slots=8192, head_dim=128, dtype="e4m3")
    q = cache.append(qkv, start, n_heads=32, rope=rope, positions=pos)   # norm, rotate, quantise, store
    out = cache.attend(q, start, tree=masks)                             # verify a tree of drafted tokens
    cache.compact(start, path, accepted)                                 # keep the accepted path

Every call runs on the caller's current stream through libmtts.so (include/mtts.h), without a host
synchronisation, and may be captured into a graph.  `start` (int32 [B], on the device) is the length
of each row's context: new tokens take the slots behind it.  Rows and slots follow the engine's own
cache: row b of a batch is row b of the cache.  Serving only: no gradients are recorded.
"""
import ctypes
from typing import List, Optional, Sequence, Tuple

import torch

from . import _native as N

DTYPES = {"bf16": 0, "e4m3": 1, "int8": 2}
TREE_MAX = 64

_KINDS = {"default": 0, "linear": 1, "ntk": 2, "yarn": 3, "llama3": 4}
# (attention_factor 0: by the formula)
_DEFAULTS = {"factor": 1.0, "original_max_position_embeddings": 0.0, "beta_fast": 32.0, "beta_slow": 1.0,
             "attention_factor": 0.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0}
_SCALING = {"rope_type", "type", *_DEFAULTS}


def rope_turns(rotary_dim: int, theta: float, scaling: Optional[dict] = None) -> Tuple[torch.Tensor, float]:
    """Host: (revolutions per position of each pair, float64 [rotary_dim / 2]; factor on the rotated
    values).  `scaling` takes the keys of a model config's `rope_scaling` / `rope_parameters`:
    rope_type (or type) default, linear, ntk, yarn or llama3; factor, and for yarn and llama3
    original_max_position_embeddings, which are required; beta_fast (32), beta_slow (1),
    attention_factor (0.1 ln(factor) + 1); low_freq_factor (1), high_freq_factor (4); rope_theta, if it
    is theta.  None is as a key that is not there; any other key that is set is refused: it would
    change the result."""
    sc = None
    if scaling is not None:
        scaling = {k: v for k, v in scaling.items() if v is not None}
        other = sorted(k for k, v in scaling.items() if k not in _SCALING and
                       not (k == "rope_theta" and float(v) == float(theta)) and not (k == "truncate" and v is True))
        if other:
            raise ValueError(f"rope scaling: {other} not supported")
        kinds = {scaling[k] for k in ("rope_type", "type") if k in scaling}
        _need(len(kinds) < 2, f"rope scaling: two types, {sorted(map(str, kinds))}")
        kind = kinds.pop() if kinds else "default"
        if kind not in _KINDS:
            raise ValueError(f"rope_type {kind!r}: one of {sorted(_KINDS)}")
        if kind == "default":  # (a scaling that lost its type, or a factor that would not be applied)
            lost = not ("rope_type" in scaling or "type" in scaling)
            given = sorted(k for k in scaling if k in _DEFAULTS and
                           (lost or k in ("factor", "attention_factor") and scaling[k] != 1))
            _need(not given, f"rope scaling: {given} without a type that uses them")
        else:
            _need("factor" in scaling, f"rope scaling: {kind} needs its factor")
        at = {k: float(scaling.get(k, d)) for k, d in _DEFAULTS.items()}
        _need("attention_factor" not in scaling or at["attention_factor"] > 0, "rope scaling: attention_factor > 0")
        sc = N.MttsRopeScaling(_KINDS[kind], at["factor"], at["original_max_position_embeddings"], at["beta_fast"],
                               at["beta_slow"], at["low_freq_factor"], at["high_freq_factor"], at["attention_factor"])
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim is even and at least 2")
    turns = torch.empty(rotary_dim // 2, dtype=torch.float64)
    factor = ctypes.c_float()
    N.call("mtts_rope_turns", float(theta), rotary_dim, None if sc is None else ctypes.byref(sc), turns.data_ptr(),
           ctypes.byref(factor))
    return turns, factor.value


def _need(cond, what):
    if not cond:
        raise ValueError(what)


def _call(name, fn, index, *args):
    """a launch on torch's current stream of the device that the call's tensors are on"""
    # (the raw handle: building a Stream object for each call costs as much as the launch)
    if torch.cuda.current_device() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        N.check(rc, name)


def _device(device):
    d = torch.device("cuda" if device is None else device)
    if d.type != "cuda" or not torch.cuda.is_available():
        raise RuntimeError("moss_tts_amd needs a ROCm GPU (MI355X); no CPU fallback exists")
    return torch.device("cuda", torch.cuda.current_device() if d.index is None else d.index)


class Rope:
    """Rotary positions of `rotary_dim` (default: all) of a head's dims: half layout (pair i, i +
    rotary_dim / 2) or interleaved (2i, 2i + 1), scaled as `rope_turns` says, or with explicit
    frequencies `inv_freq` (radians per position) and `factor`."""

    def __init__(self, head_dim: int, theta: float = 1e6, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 scaling: Optional[dict] = None, inv_freq: Optional[torch.Tensor] = None, factor: float = 1.0,
                 device=None):
        self.head_dim = head_dim
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        _need(head_dim >= 2 and head_dim % 2 == 0, "head_dim is even")
        _need(2 <= self.rotary_dim <= head_dim and self.rotary_dim % 2 == 0, "rotary_dim is even and at most head_dim")
        if inv_freq is None:
            _need(factor == 1.0, "factor goes with inv_freq; a scaling has its own")
            turns, self.factor = rope_turns(self.rotary_dim, theta, scaling)
        else:
            _need(scaling is None and inv_freq.numel() == self.rotary_dim // 2,
                  "inv_freq holds rotary_dim / 2 frequencies, without a scaling")
            turns, self.factor = inv_freq.detach().double().reshape(-1) / 6.283185307179586476925286766559, float(factor)
        self.interleaved = bool(interleaved)
        self.device = _device(device)
        self.turns = turns.to(self.device).contiguous()
        self._c = N.MttsRope(self.turns.data_ptr(), self.rotary_dim, int(self.interleaved), self.factor)
        self._ref = ctypes.addressof(self._c)
        self._fn, self._index = N.load().mtts_k_rope, self.device.index

    def apply(self, x: torch.Tensor, positions: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x bf16 [M, H, head_dim] (any strides between tokens and heads, 0 too) at int32 positions [M];
        `out` is x itself or shares no head with it (others are refused)."""
        if x.dim() != 3 or x.dtype is not torch.bfloat16 or x.shape[2] != self.head_dim or x.device != self.device:
            raise ValueError("x is bf16 [tokens, heads, head_dim] on the frequencies' device")
        M, H, D = x.shape
        xs = x.stride()
        if out is None:
            out, ys = torch.empty((M, H, D), dtype=torch.bfloat16, device=self.device), (H * D, D, 1)
        elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
            raise ValueError("out is like x")
        else:
            ys = out.stride()
        if xs[2] != 1 or ys[2] != 1:
            raise ValueError("a head's dims lie side by side")
        _call("rope", self._fn, self._index, x.data_ptr(), xs[0], xs[1], out.data_ptr(), ys[0], ys[1],
              _i32(positions, (M,), self.device, "positions"), M, H, D, self._ref)
        return out


def _i32(t, shape, device, what):
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: contiguous int32 {list(shape)} on {device}")
    return t.data_ptr()


def tree_masks(parents: Sequence[Sequence[int]]) -> Tuple[torch.Tensor, torch.Tensor]:
    """Host: drafted trees as parents ([B][T]; -1: a root, else an earlier token) to (`tree` int64
    [B, T] for `KVCache.attend`: bit u of entry t says that token t sees token u, its ancestors and
    itself; depths int32 [B, T], to add to `start` for the positions)."""
    masks: List[List[int]] = []
    depths: List[List[int]] = []
    for row in parents:
        _need(len(row) <= TREE_MAX and len(row) == len(parents[0]), "trees of at most 64 tokens, padded to one length")
        m: List[int] = []
        d: List[int] = []
        for t, p in enumerate(row):
            _need(-1 <= p < t, "a token's parent comes before it")
            m.append((m[p] if p >= 0 else 0) | 1 << t)
            d.append(d[p] + 1 if p >= 0 else 0)
        masks.append([x - (1 << 64) if x >> 63 else x for x in m])
        depths.append(d)
    return torch.tensor(masks, dtype=torch.int64), torch.tensor(depths, dtype=torch.int32)


class KVCache:
    """Keys and values of one layer: `rows` sequences of `slots` positions (rounded up to a multiple of
    64), dtype "bf16" (the engine's layout: k [rows, n_kv, slots, D], v [rows, n_kv, D, slots]),
    "e4m3" or "int8" (one byte a value in 32-slot tiles, one fp32 scale a slot and head)."""

    def __init__(self, rows: int, n_kv: int, slots: int, head_dim: int, dtype: str = "e4m3", device=None):
        _need(dtype in DTYPES, f"dtype: one of {sorted(DTYPES)}")
        _need(rows > 0 and n_kv > 0 and slots > 0, "rows, heads and slots")
        _need(head_dim in (32, 64, 128), "head_dim is 32, 64 or 128")
        self.device = _device(device)
        self.rows, self.n_kv, self.slots, self.head_dim, self.dtype = rows, n_kv, (slots + 63) // 64 * 64, head_dim, dtype
        if dtype == "bf16":
            self.k = torch.empty(rows, n_kv, self.slots, head_dim, dtype=torch.bfloat16, device=self.device)
            self.v = torch.empty(rows, n_kv, head_dim, self.slots, dtype=torch.bfloat16, device=self.device)
            self.k_scale = self.v_scale = None
        else:
            n = N.load().mtts_kv_bytes(DTYPES[dtype], rows, n_kv, head_dim, self.slots)
            self.k = torch.empty(n, dtype=torch.uint8, device=self.device)
            self.v = torch.empty(n, dtype=torch.uint8, device=self.device)
            self.k_scale = torch.empty(rows, n_kv, self.slots, dtype=torch.float32, device=self.device)
            self.v_scale = torch.empty_like(self.k_scale)
        self._c = N.MttsKvCache(self.k.data_ptr(), self.v.data_ptr(),
                                None if self.k_scale is None else self.k_scale.data_ptr(),
                                None if self.v_scale is None else self.v_scale.data_ptr(), DTYPES[dtype], rows, n_kv,
                                head_dim, self.slots)
        self._ref = ctypes.addressof(self._c)
        self._index = self.device.index
        L = N.load()
        self._f_append, self._f_read, self._f_compact = L.mtts_k_kv_append, L.mtts_k_kv_read, L.mtts_k_kv_compact
        self._f_attn, self._f_ws = L.mtts_k_attn_kv, L.mtts_k_attn_kv_ws_bytes

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)

    def _start(self, start, B):
        if B > self.rows:
            raise ValueError(f"{B} rows for a cache of {self.rows}")
        return _i32(start, (B,), self.device, "start")

    def _counts(self, counts, B):
        return None if counts is None else _i32(counts, (B,), self.device, "counts")

    def _norm(self, w, what):
        if w is None:
            return None
        if w.dtype is not torch.bfloat16 or w.shape != (self.head_dim,) or not w.is_contiguous() or w.device != self.device:
            raise ValueError(f"{what}: bf16 [head_dim]")
        return w.data_ptr()

    def _append(self, q, k, v, out, n_heads, ldq, ldk, ldv, B, S, start, rope, positions, counts, q_norm, k_norm, eps):
        r = None
        if rope is not None:
            if rope.head_dim != self.head_dim or rope.device != self.device:
                raise ValueError("rope is of another head or device")
            r = rope._ref
        _call("append", self._f_append, self._index, self._ref, q, ldq, k, ldk, v, ldv,
              None if out is None else out.data_ptr(), n_heads * self.head_dim, n_heads, self._norm(q_norm, "q_norm"),
              self._norm(k_norm, "k_norm"), eps, r,
              None if positions is None else _i32(positions, (B, S), self.device, "positions"), self._start(start, B),
              self._counts(counts, B), B, S)

    def append(self, qkv: torch.Tensor, start: torch.Tensor, n_heads: int, rope: Optional[Rope] = None,
               positions: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
               q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """qkv bf16 [B, S, (n_heads + 2 n_kv) * head_dim], the output of the q|k|v projection: norms and
        rotates q and k (positions int32 [B, S]; None: the slots), stores k and v at slots start[b] ..,
        returns q [B, S, n_heads, head_dim].  Rows behind counts[b] (int32 [B]; None: S) store nothing;
        their q is zero, or what `out` held (`out` shares nothing with qkv)."""
        D = self.head_dim
        if (qkv.dim() != 3 or qkv.dtype is not torch.bfloat16 or qkv.device != self.device or n_heads < 1 or
                qkv.shape[2] != (n_heads + 2 * self.n_kv) * D):
            raise ValueError("qkv: bf16 [B, S, (n_heads + 2 n_kv) * head_dim]")
        B, S, _ = qkv.shape
        s0, s1, s2 = qkv.stride()
        if s2 != 1 or (B > 1 and S > 1 and s0 != S * s1):
            raise ValueError("qkv: rows one stride apart")
        ld = s1 if S > 1 else s0
        if out is None:
            out = (torch.empty if counts is None else torch.zeros)((B, S, n_heads, D), dtype=torch.bfloat16,
                                                                  device=self.device)
        elif (out.shape != (B, S, n_heads, D) or out.dtype is not torch.bfloat16 or not out.is_contiguous() or
              out.device != self.device):
            raise ValueError("out: contiguous bf16 [B, S, n_heads, head_dim]")
        p = qkv.data_ptr()
        self._append(p, p + 2 * n_heads * D, p + 2 * (n_heads + self.n_kv) * D, out, n_heads, ld, ld, ld, B, S, start, rope,
                     positions, counts, q_norm, k_norm, eps)
        return out

    def write(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, rope: Optional[Rope] = None,
              positions: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None) -> None:
        """k, v bf16 [B, S, n_kv, head_dim]: stored at slots start[b] .. (k rotated if `rope` is given)."""
        lds = []
        B, S = k.shape[:2]
        for t in (k, v):
            if t.dim() != 4 or t.dtype is not torch.bfloat16 or t.device != self.device or \
                    t.shape != (B, S, self.n_kv, self.head_dim):
                raise ValueError("k, v: bf16 [B, S, n_kv, head_dim]")
            s0, s1, s2, s3 = t.stride()
            if s3 != 1 or (self.n_kv > 1 and s2 != self.head_dim) or (B > 1 and S > 1 and s0 != S * s1):
                raise ValueError("k, v: heads side by side, rows one stride apart")
            lds.append(s1 if S > 1 else s0)
        self._append(None, k.data_ptr(), v.data_ptr(), None, 0, 0, lds[0], lds[1], B, S, start, rope, positions, counts, None,
                     None, 0.0)

    def read(self, n: int, start: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
             rows: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Slots start[b] (None: 0) .. + n - 1 of the first `rows` rows (default: start's, or all) as bf16
        (k, v), each [rows, n_kv, n, head_dim]; rows behind counts[b] and slots past the end are zeros."""
        B = rows if rows is not None else self.rows if start is None else start.shape[0]
        if n < 0 or not 0 <= B <= self.rows:
            raise ValueError(f"read: {n} slots of {B} rows, of a cache of {self.rows}")
        k = torch.empty((B, self.n_kv, n, self.head_dim), dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        _call("read", self._f_read, self._index, self._ref, k.data_ptr(), v.data_ptr(),
              None if start is None else self._start(start, B), self._counts(counts, B), B, n)
        return k, v

    def compact(self, start: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor) -> None:
        """Keeps the accepted path of a drafted tree: slot start[b] + i takes what slot start[b] +
        path[b, i] holds, for i < accepted[b] (path int32 [B, P], P <= 64; accepted int32 [B])."""
        if path.dim() != 2:
            raise ValueError("path: int32 [B, P]")
        B, P = path.shape
        _call("compact", self._f_compact, self._index, self._ref, self._start(start, B),
              _i32(path, (B, P), self.device, "path"), _i32(accepted, (B,), self.device, "accepted"), B, P)

    def attend(self, q: torch.Tensor, start: torch.Tensor, tree: Optional[torch.Tensor] = None,
               counts: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
               max_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q bf16 [B, T, n_heads, head_dim] of tokens whose keys stand in slots start[b] .. (appended
        before): softmax(scale q . k) v over the context slots that mask (uint8 / bool [B, slots], 1 =
        attend) keeps and the new tokens that tree (int64 [B, T], `tree_masks`; None: a chain) shows.
        A token that sees nothing gets zeros; rows behind counts[b] are zero, or what `out` held
        (`out` is q itself or shares nothing with it).
        max_len: an upper bound of `start` known to the caller, for the shape of the launch.  The same
        call gives the same bits; a long row's rounding may differ beside rows of other lengths, or with
        another max_len."""
        if q.dim() != 4 or q.dtype is not torch.bfloat16 or q.shape[3] != self.head_dim or q.device != self.device:
            raise ValueError("q: bf16 [B, T, n_heads, head_dim]")
        B, T, H, D = q.shape
        s0, s1, s2, s3 = q.stride()
        if s3 != 1 or (H > 1 and s2 != D) or (B > 1 and T > 1 and s0 != T * s1):
            raise ValueError("q: heads side by side, rows one stride apart")
        tp = mp = None
        if tree is not None:
            if tree.dtype is not torch.int64 or tree.shape != (B, T) or not tree.is_contiguous() or tree.device != self.device:
                raise ValueError("tree: contiguous int64 [B, T]")
            tp = tree.data_ptr()
        if mask is not None:
            if mask.dtype not in (torch.uint8, torch.bool) or mask.shape != (B, self.slots) or not mask.is_contiguous() or \
                    mask.device != self.device:
                raise ValueError(f"mask: contiguous uint8 [B, {self.slots}]")
            mp = mask.data_ptr()
        if out is None:
            out = (torch.empty if counts is None else torch.zeros)((B, T, H, D), dtype=torch.bfloat16, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != self.device:
            raise ValueError("out: contiguous, like q")
        if scale is None:
            scale = 0.0
        elif not scale > 0:
            raise ValueError("scale > 0")
        ld = s1 if T > 1 else s0 if B > 1 else H * D  # (a single token has no stride)
        n = 0 if max_len is None else max(1, int(max_len))
        need = self._f_ws(B, T, H, self.n_kv, D, self.slots, n)
        # (scratch of this call alone, from torch's allocator: in order on this stream, a graph's own in a capture)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        _call("attend", self._f_attn, self._index, self._ref, q.data_ptr(), ld, out.data_ptr(), H * D, H,
              self._start(start, B), self._counts(counts, B), tp, mp, B, T, scale, n, None if ws is None else ws.data_ptr())
        return out
