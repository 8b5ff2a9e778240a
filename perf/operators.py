"""Decoding with drafted tokens over an 8-bit key / value cache: the operators, their cases and their
plain forms.

  rope      rotary positions of packed heads at explicit positions: half or interleaved pairs, all or
            part of the head, unscaled or stretched for long contexts
  append    the q / k norm and rotation of new tokens, with their keys and values quantised into the
            cache, and those slots read back
  read      a row of the quantised cache read back
  compact   the accepted path of a drafted tree moved to the front of its slots
  attend    attention of new tokens (one, a chain, a tree) over a cache of bf16, e4m3 or int8

`own` false: `run` computes them with elementary torch operations in 32 bits (angles in 64).  `own`
true: it calls `moss_tts_amd.kvcache`.  Caches hold `slots` positions a row; a row's context is its
first `start` slots and its new tokens take the slots behind them.
"""
import math
import random

import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
DEV = "cuda"


def listed():
    q8 = dict(n_heads=32, n_kv=8, head_dim=128)
    return [
        # one decode step of four sequences: rotation alone, bound by the launch
        dict(name="rope_step", op="rope", tokens=4, heads=40, head_dim=128, rotary=128, interleaved=False,
             scaling="none", far=1800),
        # a long script as one prompt, positions stretched to four times the trained length
        dict(name="rope_prompt_yarn", op="rope", tokens=6001, heads=40, head_dim=128, rotary=128,
             interleaved=False, scaling="yarn", far=131071),
        # one sequence's next token into the cache
        dict(name="append_step_e4m3", op="append", kind="e4m3", rows=1, tokens=1, slots=2048, norm=True,
             rotary=128, interleaved=False, scaling="none", **q8),
        # eight sequences' drafted trees of 17 tokens; pairs interleaved over half of the head
        dict(name="append_drafts_int8", op="append", kind="int8", rows=8, tokens=17, slots=4096, norm=False,
             rotary=64, interleaved=True, scaling="llama3", **q8),
        # three scripts of up to 2,117 tokens, padded to one batch
        dict(name="append_prompt_e4m3", op="append", kind="e4m3", rows=3, tokens=2117, slots=8192, norm=True,
             rotary=128, interleaved=False, scaling="yarn", **q8),
        # a long session's row of one layer, read back to move or to check it
        dict(name="read_row_int8", op="read", kind="int8", rows=1, tokens=65536, slots=65536, n_kv=8, head_dim=128),
        # the accepted path after one verification
        dict(name="compact_step_e4m3", op="compact", kind="e4m3", rows=1, tokens=16, slots=2048, n_kv=8, head_dim=128),
        # the same for a full batch of wide trees
        dict(name="compact_batch_int8", op="compact", kind="int8", rows=64, tokens=64, slots=2048, n_kv=8,
             head_dim=128),
        # one sequence, one token, a short clone prompt behind it: latency
        dict(name="attend_token_bf16", op="attend", kind="bf16", rows=1, tokens=1, context=389, slots=2048,
             tree=False, pads=False, **q8),
        # four left-padded sequences verify trees of 16 tokens
        dict(name="attend_tree_e4m3", op="attend", kind="e4m3", rows=4, tokens=16, context=7500, slots=8192,
             tree=True, pads=True, **q8),
        # an hour-long session: 33 drafted tokens against the longest context
        dict(name="attend_long_int8", op="attend", kind="int8", rows=1, tokens=33, context=130001, slots=131072,
             tree=True, pads=False, **q8),
        # a full batch verifies wide trees: bound by the products
        dict(name="attend_batch_bf16", op="attend", kind="bf16", rows=16, tokens=64, context=4000, slots=4096,
             tree=True, pads=False, **q8),
    ]


def _log(rng, lo, hi):
    """a whole number from lo to hi, spread over its logarithm"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "append", "read", "compact", "attend", "attend", "attend"])
    n_kv, group, head_dim = rng.choice([(8, 4, 128), (8, 3, 128), (4, 4, 64), (6, 4, 64), (2, 7, 128), (4, 1, 128)])
    rotary = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
    turn = dict(rotary=rotary, interleaved=rng.random() < 0.4, scaling=rng.choice(["none", "linear", "ntk", "yarn", "llama3"]))
    kind = rng.choice(["e4m3", "int8"])
    if op == "rope":
        return dict(op=op, tokens=_log(rng, 1, 6000), heads=n_kv * (group + 1), head_dim=head_dim, far=_log(rng, 512, 131071),
                    **turn)
    if op == "append":
        rows = _log(rng, 1, 8)
        tokens = _log(rng, 1, 6000 // rows)
        return dict(op=op, kind=kind, rows=rows, tokens=tokens, slots=_slots(tokens + _log(rng, 16, 2000)),
                    norm=rng.random() < 0.5, n_heads=n_kv * group, n_kv=n_kv, head_dim=head_dim, **turn)
    if op == "read":
        rows = _log(rng, 1, 8)
        tokens = _log(rng, 1, 60000 // rows)
        return dict(op=op, kind=kind, rows=rows, tokens=tokens, slots=_slots(tokens), n_kv=n_kv, head_dim=head_dim)
    if op == "compact":
        return dict(op=op, kind=kind, rows=_log(rng, 1, 64), tokens=_log(rng, 1, 64), slots=_slots(_log(rng, 128, 2000)),
                    n_kv=n_kv, head_dim=head_dim)
    rows = _log(rng, 1, 16)
    tokens = _log(rng, 1, 64)
    context = _log(rng, 1, min(130000 // rows, 4000 * 16 * 64 // (rows * tokens)))
    return dict(op=op, kind=rng.choice(["bf16", "e4m3", "int8"]), rows=rows, tokens=tokens, context=context,
                slots=_slots(context + tokens), tree=rng.random() < 0.7, pads=rng.random() < 0.4, n_heads=n_kv * group,
                n_kv=n_kv, head_dim=head_dim)


def _slots(n):
    return (n + 63) // 64 * 64


def _starts(case):
    """each row's context: ragged, the same for every seed"""
    rows, room = case["rows"], case["slots"] - case["tokens"]
    top = min(room, case["context"]) if "context" in case else room
    return [top - (top * b) // (2 * rows) for b in range(rows)]


def _counts(case):
    """new tokens of each row of a padded batch"""
    t = case["tokens"]
    return [max(1, t - (t * b) // (3 * case["rows"])) for b in range(case["rows"])]


def _scaling(name):
    return {"none": None,
            "linear": dict(rope_type="linear", factor=4.0),
            "ntk": dict(rope_type="ntk", factor=4.0),
            "yarn": dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768),
            "llama3": dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                           original_max_position_embeddings=8192)}[name]


THETA = 1000000.0


def _frequencies(name, rot):
    """(radians per position of each pair, factor on the rotated values)"""
    p, f = _scaling(name), [THETA ** (-2.0 * i / rot) for i in range(rot // 2)]
    if name == "none":
        return f, 1.0
    s = p["factor"]
    if name == "linear":
        return [x / s for x in f], 1.0
    if name == "ntk":
        base = THETA * s ** (rot / (rot - 2.0))
        return [base ** (-2.0 * i / rot) for i in range(rot // 2)], 1.0
    old = p["original_max_position_embeddings"]
    if name == "llama3":
        lo, hi = p["low_freq_factor"], p["high_freq_factor"]
        m = [min(1.0, max(0.0, (old * x / (2 * math.pi) - lo) / (hi - lo))) for x in f]
        return [(1 - a) * x / s + a * x for a, x in zip(m, f)], 1.0

    def at(turns):
        return rot * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(THETA))
    lo, hi = max(0, math.floor(at(32.0))), min(rot - 1, math.ceil(at(1.0)))
    r = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(rot // 2)]
    return [a * x / s + (1 - a) * x for a, x in zip(r, f)], 0.1 * math.log(s) + 1.0


def _tree(case, seed):
    """drafted trees: each token's parent is one of the eight before it; bit u of a token's mask says
    that it sees drafted token u.  ([rows, tokens] masks, depths)"""
    r = random.Random(seed)
    masks, depth = [], []
    for _ in range(case["rows"]):
        m, d = [1], [0]
        for t in range(1, case["tokens"]):
            p = r.randint(max(0, t - 8), t - 1)
            m.append(m[p] | 1 << t)
            d.append(d[p] + 1)
        masks.append([x - (1 << 64) if x >> 63 else x for x in m])
        depth.append(d)
    return masks, depth


def _quantise(x, kind):
    """codes (as values) and scales of rows of 32-bit values"""
    a = x.abs().amax(-1, keepdim=True)
    live = a >= 2.0 ** -100
    c = (x * QMAX[kind] / torch.where(live, a, torch.ones_like(a))).clamp(-QMAX[kind], QMAX[kind])
    c = torch.where(live, c, torch.zeros_like(c))
    c = c.to(torch.float8_e4m3fn) if kind == "e4m3" else c.round().to(torch.int8)
    return c, torch.where(live, a / QMAX[kind], torch.zeros_like(a))[..., 0]


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _keys(g, *shape):
    """keys as a trained model makes them: some of the dims much larger than the others"""
    w = 0.6 + 2.5 * torch.rand(shape[-1], generator=g, device=DEV) ** 6
    return (_randn(g, *shape) * w).to(torch.bfloat16)


def _rope_handle(case):
    from moss_tts_amd import kvcache
    return kvcache.Rope(case["head_dim"], theta=THETA, rotary_dim=case["rotary"], interleaved=case["interleaved"],
                        scaling=_scaling(case["scaling"]), device=DEV)


def _cache_handle(case, k=None, v=None):
    from moss_tts_amd import kvcache
    c = kvcache.KVCache(case["rows"], case["n_kv"], case["slots"], case["head_dim"], case["kind"], device=DEV)
    if k is not None:
        c.write(k, v, torch.zeros(case["rows"], dtype=torch.int32, device=DEV))
    return c


def prepare(case, seed):
    """The inputs, and the cache and the frequencies that a program keeps.  The plain form's cache is
    rows of codes with their scales; the framework's is its own handle with the same values."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=case)
    if "rotary" in case:
        f, s["factor"] = _frequencies(case["scaling"], case["rotary"])
        s["freq"] = torch.tensor(f, dtype=torch.float64, device=DEV)
        if own:
            s["rope"] = _rope_handle(case)
    if case["op"] == "rope":
        n = case["tokens"]
        s["x"] = _randn(g, n, case["heads"], case["head_dim"]).to(torch.bfloat16)
        lo = torch.randint(0, case["far"] - min(n, case["far"]) + 1, (1,), generator=g, device=DEV)
        s["pos"] = ((lo + torch.arange(n, device=DEV)) % (case["far"] + 1)).to(torch.int32)
        return s
    B, T, Hkv, D = case["rows"], case["tokens"], case["n_kv"], case["head_dim"]
    if case["op"] == "append":
        H = case["n_heads"]
        s["qkv"] = torch.cat([_keys(g, B, T, H + Hkv, D), _randn(g, B, T, Hkv, D).to(torch.bfloat16)], 2).view(B, T, -1)
        s["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEV)
        s["start"] = torch.tensor(_starts(case), dtype=torch.int32, device=DEV)
        s["pos"] = s["start"][:, None] + torch.arange(T, dtype=torch.int32, device=DEV)
        s["q_norm"] = (0.5 + torch.rand(D, generator=g, device=DEV)).to(torch.bfloat16) if case["norm"] else None
        s["k_norm"] = (0.5 + torch.rand(D, generator=g, device=DEV)).to(torch.bfloat16) if case["norm"] else None
        s["q"] = torch.zeros(B, T, H, D, dtype=torch.bfloat16, device=DEV)
        if own:
            s["cache"] = _cache_handle(case)
        return s
    if case["op"] == "attend":
        s["q"] = _keys(g, B, T, case["n_heads"], D)
        if case["tree"]:
            s["tree"] = torch.tensor(_tree(case, seed)[0], dtype=torch.int64, device=DEV)
        if case["pads"]:  # left pads: up to a fifth of a row's context
            pad = torch.tensor([n * b // (5 * B) for b, n in enumerate(_starts(case))], device=DEV)
            s["mask"] = (torch.arange(case["slots"], device=DEV)[None] >= pad[:, None]).to(torch.uint8)
    n = T if case["op"] == "read" else case["slots"]
    k, v = _keys(g, B, n, Hkv, D), _randn(g, B, n, Hkv, D).to(torch.bfloat16)
    s["start"] = torch.tensor([0] * B if case["op"] == "read" else _starts(case), dtype=torch.int32, device=DEV)
    if case["op"] == "compact":  # the accepted tokens: some path down the tree, the root first
        masks, depth = _tree(case, seed)
        path, took = [], []
        for m, d in zip(masks, depth):
            leaf = max(range(T), key=lambda t: (d[t], t))
            p = [t for t in range(T) if m[leaf] >> t & 1]
            path.append(p + [0] * (T - len(p)))
            took.append(len(p))
        s["path"] = torch.tensor(path, dtype=torch.int32, device=DEV)
        s["took"] = torch.tensor(took, dtype=torch.int32, device=DEV)
    if own:
        s["cache"] = _cache_handle(case, k, v)
    else:
        k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
        if case["kind"] == "bf16":
            s["k"], s["v"] = (k, None), (v, None)
        else:
            s["k"], s["v"] = _quantise(k.float(), case["kind"]), _quantise(v.float(), case["kind"])
    return s


# ---- plain forms -----------------------------------------------------------------------------------

def _rotate(x, pos, s, rot, interleaved):
    """x [..., heads, head_dim] in 32 bits, pos [...]"""
    a = pos.double()[..., None] * s["freq"]
    c, n = (a.cos() * s["factor"]).float()[..., None, :], (a.sin() * s["factor"]).float()[..., None, :]
    y = x.clone()
    if interleaved:
        u, v = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = u * c - v * n, v * c + u * n
    else:
        u, v = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = u * c - v * n, v * c + u * n
    return y


def _values(code, scale):
    x = code.float()
    return x if scale is None else x * scale[..., None]


def _normed(x, w):
    if w is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()


def _plain_append(s):
    case = s["case"]
    H, Hkv, D, kind = case["n_heads"], case["n_kv"], case["head_dim"], case["kind"]
    B, T = case["rows"], case["tokens"]
    x = s["qkv"].view(B, T, H + 2 * Hkv, D).float()
    q, k, v = _normed(x[:, :, :H], s["q_norm"]), _normed(x[:, :, H:H + Hkv], s["k_norm"]), x[:, :, H + Hkv:]
    q = _rotate(q, s["pos"], s, case["rotary"], case["interleaved"])
    k = _rotate(k, s["pos"], s, case["rotary"], case["interleaved"])
    live = (torch.arange(T, device=DEV)[None] < s["counts"][:, None])[..., None, None]
    k, v = (_values(*_quantise(y.transpose(1, 2), kind)).to(torch.bfloat16) for y in (k, v))
    zero = torch.zeros((), dtype=torch.bfloat16, device=DEV)
    return [torch.where(live, q.to(torch.bfloat16), s["q"]), *(torch.where(live.transpose(1, 2), y, zero) for y in (k, v))]


def _plain_compact(s):
    case = s["case"]
    T = case["tokens"]
    i = torch.arange(T, device=DEV)
    new = s["start"][:, None].long() + i  # [rows, T]
    old = s["start"][:, None].long() + torch.where(i < s["took"][:, None], s["path"].long(), i)
    rows = torch.arange(case["rows"], device=DEV)[:, None]
    out = []
    for code, scale in (s["k"], s["v"]):
        raw = code.view(torch.int8)
        raw[rows, :, new] = raw[rows, :, old]
        scale[rows, :, new] = scale[rows, :, old]
        out.append(_values(code[rows, :, new].float(), scale[rows, :, new]).transpose(1, 2).to(torch.bfloat16))
    return out


def _plain_attend(s):
    case = s["case"]
    B, T, H, Hkv, D = case["rows"], case["tokens"], case["n_heads"], case["n_kv"], case["head_dim"]
    n = min(case["slots"], max(_starts(case)) + T)
    k, v = (_values(c[:, :, :n], e if e is None else e[:, :, :n]) for c, e in (s["k"], s["v"]))
    q = s["q"].view(B, T, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D).float()
    z = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(D ** -0.5).view(B, Hkv, H // Hkv, T, n)
    j = torch.arange(n, device=DEV)
    u = j[None] - s["start"][:, None]  # [B, n]: which drafted token a slot holds
    sees = u < 0
    if case["pads"]:
        sees = sees & (s["mask"][:, :n] != 0)
    t = torch.arange(T, device=DEV)
    if case["tree"]:
        bit = (s["tree"][:, :, None] >> u.clamp(0, 63)[:, None, :]) & 1 != 0
    else:
        bit = u[:, None, :] <= t[None, :, None]
    sees = sees[:, None, :] | (bit & (u >= 0)[:, None, :] & (u < T)[:, None, :])  # [B, T, n]
    z = z.masked_fill_(~sees[:, None, None], -math.inf)
    z = torch.exp(z.sub_(z.amax(-1, keepdim=True)))
    o = torch.matmul(z.view(B, Hkv, -1, n), v) / z.sum(-1).view(B, Hkv, -1, 1)
    return o.view(B, Hkv, H // Hkv, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(torch.bfloat16)


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        if op == "rope":
            return s["rope"].apply(s["x"], s["pos"])
        cache = s["cache"]
        if op == "append":
            q = cache.append(s["qkv"], s["start"], n_heads=case["n_heads"], rope=s["rope"], positions=s["pos"],
                             counts=s["counts"], q_norm=s["q_norm"], k_norm=s["k_norm"], out=s["q"])
            return [q, *cache.read(case["tokens"], start=s["start"], counts=s["counts"])]
        if op == "read":
            return list(cache.read(case["tokens"]))
        if op == "compact":
            cache.compact(s["start"], s["path"], s["took"])
            return list(cache.read(case["tokens"], start=s["start"]))
        return cache.attend(s["q"], s["start"], tree=s.get("tree"), mask=s.get("mask"), max_len=case["context"])
    if op == "rope":
        return _rotate(s["x"].float(), s["pos"], s, case["rotary"], case["interleaved"]).to(torch.bfloat16)
    if op == "append":
        return _plain_append(s)
    if op == "read":
        return [_values(*s[x]).to(torch.bfloat16) for x in ("k", "v")]
    if op == "compact":
        return _plain_compact(s)
    return _plain_attend(s)


def work(case):
    D = case["head_dim"]
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 4 * n * D, "flops": 3 * n * case["rotary"]}
    slot = 2 * case["n_kv"] * (2 * D if case.get("kind") == "bf16" else D + 4)  # keys and values of one position
    plain = 2 * case["n_kv"] * 2 * D  # the same in bf16
    if case["op"] == "append":
        n, q = sum(_counts(case)), case["n_heads"] * D
        return {"bytes": n * (2 * q + plain + 2 * q + 2 * slot + plain), "flops": n * (6 * q + 8 * case["n_kv"] * D)}
    n = case["rows"] * case["tokens"]
    if case["op"] == "read":
        return {"bytes": n * (slot + plain), "flops": 2 * n * case["n_kv"] * D}
    if case["op"] == "compact":  # about half of a tree's tokens move
        return {"bytes": n * (slot + slot + plain), "flops": 2 * n * case["n_kv"] * D}
    keys = sum(_starts(case)) + n
    return {"bytes": keys * slot + n * case["n_heads"] * D * 4,
            "flops": 4 * D * case["n_heads"] * case["tokens"] * keys}


# ---- the definitions in 64 bits --------------------------------------------------------------------

def _to_e4m3(x):
    """the nearest e4m3 value, ties to the even one"""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _stored(x, kind):
    """the values that a quantised row stands for"""
    a = x.abs().max(-1, keepdim=True).values
    y = torch.where(a > 0, x * QMAX[kind] / a, torch.zeros_like(x))  # (a tie stays one: x is exact, so is the product)
    return (_to_e4m3(y) if kind == "e4m3" else torch.round(y)) * a / QMAX[kind]


def _spun(x, pos, case):
    """rotation of the pairs as a product of complex numbers"""
    rot = case["rotary"]
    f, m = _frequencies(case["scaling"], rot)
    a = torch.outer(pos.reshape(-1).double(), torch.tensor(f, dtype=torch.float64, device=DEV)).view(*pos.shape, 1, rot // 2)
    turn = torch.polar(torch.full_like(a, m), a)
    head, tail = x[..., :rot], x[..., rot:]
    if case["interleaved"]:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * turn
        return torch.cat([torch.view_as_real(z).flatten(-2), tail], -1)
    z = torch.complex(*(y.contiguous() for y in head.chunk(2, -1))) * turn
    return torch.cat([z.real, z.imag, tail], -1)


def exact(case, seed):
    s = _plain_inputs(case, seed)
    if case["op"] == "rope":
        return _spun(s["x"].double(), s["pos"], case)
    B, T, Hkv, D = case["rows"], case["tokens"], case["n_kv"], case["head_dim"]
    if case["op"] == "append":
        H = case["n_heads"]
        x = s["qkv"].view(B, T, -1, D).double()
        q, k, v = x.split([H, Hkv, Hkv], 2)
        if case["norm"]:
            q, k = (y / (y.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * s[w].double() for y, w in ((q, "q_norm"), (k, "k_norm")))
        q, k = _spun(q, s["pos"], case), _stored(_spun(k, s["pos"], case), case["kind"])
        v = _stored(v, case["kind"])
        for b, n in enumerate(_counts(case)):
            for y in (q, k, v):
                y[b, n:] = 0
        return [q, k.transpose(1, 2), v.transpose(1, 2)]
    k, v = (c.double() if e is None else c.double() * e.double()[..., None] for c, e in (s["k"], s["v"]))
    if case["op"] == "read":
        return [k, v]
    if case["op"] == "compact":
        out = []
        for y in (k, v):
            rows = []
            for b, n in enumerate(_starts(case)):
                took = s["path"][b, :int(s["took"][b])].long()
                new = y[b, :, n:n + T]
                rows.append(torch.cat([new[:, took], new[:, len(took):]], 1))
            out.append(torch.stack(rows))
        return out
    out = torch.zeros(B, T, case["n_heads"], D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_starts(case)):
        sees = torch.zeros(T, n + T, dtype=torch.bool, device=DEV)
        sees[:, :n] = True if not case["pads"] else s["mask"][b, :n] != 0
        for t in range(T):
            m = int(s["tree"][b, t]) if case["tree"] else (2 << t) - 1
            sees[t, n:] = torch.tensor([m >> u & 1 for u in range(T)], device=DEV, dtype=torch.bool)
        for h in range(Hkv):
            for i in range(case["n_heads"] // Hkv):
                x = h * (case["n_heads"] // Hkv) + i
                z = s["q"][b, :, x].double() @ k[b, h, :n + T].T / math.sqrt(D)
                out[b, :, x] = torch.softmax(z.masked_fill(~sees, -math.inf), -1) @ v[b, h, :n + T]
    return out


def _plain_inputs(case, seed):
    """the inputs without the framework's handles, whatever `own` says"""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was
