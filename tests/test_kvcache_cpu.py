"""Drafted-token operators, host side: rotary frequencies against their formulas, tree masks, and the
refusals of the C entry points (every check comes before any device call)."""
import ctypes
import math
import os
import random

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def kv():
    from moss_tts_amd import _native, kvcache
    if not os.path.exists(_native.lib_path()):
        pytest.skip("libmtts.so not built")
    _native.load()
    return kvcache


@pytest.fixture(scope="module")
def N(kv):
    from moss_tts_amd import _native
    return _native


def formula(rot, theta, sc):
    """radians per position, from the definitions"""
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    kind = sc.get("rope_type", "default")
    s = sc.get("factor", 1.0)
    if kind == "linear":
        return [x / s for x in f], 1.0
    if kind == "ntk":
        return [(theta * s ** (rot / (rot - 2.0))) ** (-2.0 * i / rot) for i in range(rot // 2)], 1.0
    if kind == "default":
        return f, 1.0
    old = sc["original_max_position_embeddings"]
    if kind == "llama3":
        lo, hi = sc.get("low_freq_factor", 1.0), sc.get("high_freq_factor", 4.0)
        out = []
        for x in f:
            turns = old * x / (2 * math.pi)
            w = (turns - lo) / (hi - lo)
            out.append(x / s if turns < lo else x if turns > hi else (1 - w) * x / s + w * x)
        return out, 1.0
    at = lambda b: rot * math.log(old / (b * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    lo, hi = max(math.floor(at(sc.get("beta_fast", 32))), 0), min(math.ceil(at(sc.get("beta_slow", 1))), rot - 1)
    hi = hi + 0.001 if hi == lo else hi
    out = []
    for i, x in enumerate(f):
        r = min(1.0, max(0.0, (i - lo) / (hi - lo)))
        out.append(x / s * r + x * (1 - r))
    return out, sc.get("attention_factor", 0.1 * math.log(s) + 1.0)


@pytest.mark.parametrize("rot", [2, 10, 64, 128])
@pytest.mark.parametrize("sc", [{}, dict(rope_type="linear", factor=4.0), dict(rope_type="ntk", factor=8.0),
                                dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768),
                                dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096, beta_fast=24,
                                     beta_slow=2, attention_factor=1.5),
                                dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                     original_max_position_embeddings=8192)])
def test_rope_turns(kv, rot, sc):
    if sc.get("rope_type") == "ntk" and rot == 2:
        pytest.skip("refused, below")
    turns, factor = kv.rope_turns(rot, 1e6, sc or None)
    want, m = formula(rot, 1e6, sc)
    got = turns * 2 * math.pi
    # 64-bit powers and logarithms: a few steps of 2^-53
    assert torch.allclose(got, torch.tensor(want, dtype=torch.float64), rtol=1e-13, atol=0)
    assert abs(factor - m) <= 2.0 ** -24 * m


@pytest.mark.parametrize("rot,theta,sc", [(3, 1e4, None), (0, 1e4, None), (64, 1.0, None), (64, float("nan"), None),
                                          (64, 1e4, dict(rope_type="linear", factor=0.5)),
                                          (64, 1e4, dict(rope_type="yarn", factor=4.0)),
                                          (64, 1e4, dict(rope_type="llama3", factor=8.0, low_freq_factor=4.0,
                                                         high_freq_factor=4.0, original_max_position_embeddings=8192)),
                                          (2, 1e4, dict(rope_type="ntk", factor=2.0)),
                                          (64, 1e4, dict(rope_type="longer"))])
def test_rope_turns_refusals(kv, rot, theta, sc):
    with pytest.raises(ValueError):
        kv.rope_turns(rot, theta, sc)


@pytest.mark.parametrize("extra", [dict(mscale=0.7), dict(truncate=False), dict(partial_rotary_factor=0.5), dict(rope_theta=5e5),
                                   dict(short_factor=[1.0])])
def test_rope_scaling_keys(kv, extra):
    """a key that the frequencies would not follow is refused, not ignored; one that says the same is fine"""
    sc = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)
    with pytest.raises(ValueError, match="not supported"):
        kv.rope_turns(64, 1e4, {**sc, **extra})
    a, b = kv.rope_turns(64, 1e4, sc), kv.rope_turns(64, 1e4, {**sc, "rope_theta": 10000, "truncate": True, "mscale": None})
    assert torch.equal(a[0], b[0]) and a[1] == b[1]


NAN, INF = float("nan"), float("inf")
YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)
LLAMA3 = dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192)


@pytest.mark.parametrize("sc", [
    dict(rope_type="linear"), dict(rope_type="ntk"), dict(rope_type="ntk", factor=None), {**YARN, "factor": None},
    dict(rope_type="yarn", original_max_position_embeddings=4096), dict(rope_type="llama3", original_max_position_embeddings=8192),
    dict(factor=4.0), dict(rope_type="default", factor=4.0), dict(rope_type="default", attention_factor=1.2), dict(original_max_position_embeddings=4096),
    dict(type="ntk", rope_type="linear", factor=2.0), {**YARN, "beta_fast": 0}, {**YARN, "beta_slow": 0},
    {**YARN, "beta_slow": -1.0}, {**YARN, "beta_fast": 1, "beta_slow": 32}, {**YARN, "attention_factor": 0},
    {**YARN, "attention_factor": -1.0}, {**YARN, "attention_factor": NAN}, {**YARN, "attention_factor": INF},
    {**YARN, "factor": INF}, {**YARN, "factor": NAN}, {**YARN, "beta_fast": NAN}, {**YARN, "beta_fast": INF},
    {**YARN, "original_max_position_embeddings": INF}, {**YARN, "original_max_position_embeddings": None},
    {**YARN, "original_max_position_embeddings": 0}, dict(rope_type="linear", factor=INF), {**LLAMA3, "high_freq_factor": INF},
    {**LLAMA3, "low_freq_factor": NAN}, {**LLAMA3, "low_freq_factor": 5.0}])
def test_rope_scaling_is_never_made_up(kv, sc):
    """what a scaling needs has to be there, and a value that is there is used or refused"""
    with pytest.raises(ValueError):
        kv.rope_turns(64, 1e4, sc)


@pytest.mark.parametrize("theta", [INF, 1.0, 0.5, NAN])
def test_rope_base_refused(kv, theta):
    with pytest.raises(ValueError):
        kv.rope_turns(64, theta)


@pytest.mark.parametrize("sc", [dict(rope_type="linear", factor=2.0), dict(rope_type="ntk", factor=2.0), YARN, LLAMA3,
                                dict(rope_type="default"), {}])
def test_rope_scaling_none_is_absent(kv, sc):
    """a key that holds None is as one that is not there, every key alike"""
    keys = ("type", "beta_fast", "beta_slow", "attention_factor", "low_freq_factor", "high_freq_factor", "factor",
            "original_max_position_embeddings", "rope_theta", "rope_type")
    a, b = kv.rope_turns(64, 1e4, sc), kv.rope_turns(64, 1e4, {**{k: None for k in keys}, **sc})
    assert torch.equal(a[0], b[0]) and a[1] == b[1]
    if "rope_type" in sc:  # the older name of the key; both, if they agree
        old = {"type" if k == "rope_type" else k: v for k, v in sc.items()}
        for other in (old, {**old, "rope_type": None}, {**old, "rope_type": sc["rope_type"]}):
            c = kv.rope_turns(64, 1e4, other)
            assert torch.equal(a[0], c[0]) and a[1] == c[1]


def test_rope_explicit_values_are_used(kv):
    plain = kv.rope_turns(64, 1e4)[0]
    assert torch.equal(kv.rope_turns(64, 1e4, dict(rope_type="default", factor=1.0, original_max_position_embeddings=4096))[0], plain)
    for sc in ({**LLAMA3, "low_freq_factor": 0}, {**LLAMA3, "low_freq_factor": 2.0, "high_freq_factor": 3.0},
               {**YARN, "beta_fast": 8, "beta_slow": 0.5, "attention_factor": 1e-3}):
        turns, factor = kv.rope_turns(64, 1e4, sc)
        want, m = formula(64, 1e4, sc)
        assert torch.allclose(turns * 2 * math.pi, torch.tensor(want, dtype=torch.float64), rtol=1e-13, atol=0)
        assert abs(factor - m) <= 2.0 ** -24 * m


@pytest.mark.parametrize("kw", [dict(factor=2.0), dict(factor=2.0, scaling=YARN), dict(factor=NAN)])
def test_rope_factor_without_frequencies(kv, kw):
    """a factor that would not be applied is refused (before a device is looked for)"""
    with pytest.raises(ValueError, match="factor"):
        kv.Rope(64, **kw)


def test_tree_masks(kv):
    masks, depth = kv.tree_masks([[-1, 0, 0, 1, 3], [-1, -1, 1, 2, 0]])
    assert masks.tolist() == [[1, 3, 5, 11, 27], [1, 2, 6, 14, 17]]
    assert depth.tolist() == [[0, 1, 1, 2, 3], [0, 0, 1, 2, 1]] and depth.dtype == torch.int32
    chain, _ = kv.tree_masks([list(range(-1, 63))])
    assert chain[0, 63].item() == -1 and chain[0, 62].item() == (1 << 63) - 1
    for bad in ([[0]], [[-1, 2]], [[-1], [-1, 0]], [[-1] + list(range(64))]):
        with pytest.raises(ValueError):
            kv.tree_masks(bad)


FAKE = 1 << 20  # an aligned address that no check follows


def cache(N, **kw):
    f = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, type=1, rows=2, n_kv=2, head_dim=64, slots=64)
    f.update(kw)
    return N.MttsKvCache(*(f[n] for n, _ in N.MttsKvCache._fields_))


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(type=3), dict(type=-1), dict(rows=0), dict(n_kv=0),
              dict(slots=0), dict(slots=48), dict(k=FAKE + 8), dict(v_scale=FAKE + 4)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches(N, bad):
    c = ctypes.byref(cache(N, **bad))
    with pytest.raises(ValueError):
        N.call("mtts_k_kv_append", c, None, 0, FAKE, 128, FAKE, 128, None, 0, 0, None, None, 0.0, None, None, FAKE, None, 1, 1,
               None)
    with pytest.raises(ValueError):
        N.call("mtts_k_kv_read", c, FAKE, FAKE, None, None, 1, 1, None)
    with pytest.raises(ValueError):
        N.call("mtts_k_kv_compact", c, FAKE, FAKE, FAKE, 1, 1, None)
    with pytest.raises(ValueError):
        N.call("mtts_k_attn_kv", c, FAKE, 256, FAKE, 256, 4, FAKE, None, None, None, 1, 1, 0.0, 0, FAKE, None)


@pytest.mark.parametrize("D", [16, 96, 256])
def test_head_dims_refused(N, D):
    with pytest.raises(RuntimeError, match="head_dim"):
        N.call("mtts_k_attn_kv", ctypes.byref(cache(N, head_dim=D)), FAKE, 4 * D, FAKE, 4 * D, 4, FAKE, None, None, None, 1, 1,
               0.0, 0, FAKE, None)


def test_attention_refusals(N):
    c = ctypes.byref(cache(N))
    ok = dict(q=FAKE, ldq=256, out=FAKE, ldo=256, H=4, start=FAKE, counts=None, tree=None, mask=None, B=1, T=1, scale=0.0,
              max_len=0, ws=FAKE)

    def call(**kw):
        N.call("mtts_k_attn_kv", c, *{**ok, **kw}.values(), None)
    for bad in (dict(q=None), dict(out=None), dict(start=None), dict(H=3), dict(H=0), dict(B=3), dict(B=-1), dict(T=-1),
                dict(q=FAKE + 2), dict(ldq=260), dict(out=FAKE + 4), dict(ldo=258), dict(mask=FAKE + 4), dict(ws=FAKE + 8)):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(RuntimeError, match="at most 64"):
        call(T=65, tree=FAKE)
    long = ctypes.byref(cache(N, slots=8192))
    assert N.load().mtts_k_attn_kv_ws_bytes(1, 1, 4, 2, 64, 8192, 0) > 0
    with pytest.raises(ValueError, match="workspace"):
        N.call("mtts_k_attn_kv", long, *{**ok, "ws": None}.values(), None)
    call(B=0), call(T=0)  # nothing to do: no launch


def test_append_and_move_refusals(N):
    c = ctypes.byref(cache(N))
    rope = N.MttsRope(FAKE, 64, 0, 1.0)

    def app(q=None, k=FAKE, v=FAKE, q_out=None, H=0, rope=None, start=FAKE, B=1, S=1):
        N.call("mtts_k_kv_append", c, q, 256, k, 128, v, 128, q_out, 256, H, None, None, 0.0,
               None if rope is None else ctypes.byref(rope), None, start, None, B, S, None)
    for bad in (dict(k=None), dict(v=None), dict(start=None), dict(q=FAKE, H=4), dict(q=FAKE, q_out=FAKE), dict(B=3),
                dict(S=-1), dict(rope=N.MttsRope(FAKE, 66, 0, 1.0)), dict(rope=N.MttsRope(FAKE, 3, 0, 1.0)),
                dict(rope=N.MttsRope(None, 64, 0, 1.0))):
        with pytest.raises(ValueError):
            app(**bad)
    app(B=0), app(S=0)
    for bad in ((None, FAKE, None, None, 1, 1), (FAKE, FAKE + 8, None, None, 1, 1), (FAKE, FAKE, None, None, 3, 1),
                (FAKE, FAKE, None, None, 1, -1)):
        with pytest.raises(ValueError):
            N.call("mtts_k_kv_read", c, *bad, None)
    for bad in ((None, FAKE, FAKE, 1, 1), (FAKE, None, FAKE, 1, 1), (FAKE, FAKE, None, 1, 1), (FAKE, FAKE, FAKE, 3, 1)):
        with pytest.raises(ValueError):
            N.call("mtts_k_kv_compact", c, *bad, None)
    with pytest.raises(RuntimeError, match="at most 64"):
        N.call("mtts_k_kv_compact", c, FAKE, FAKE, FAKE, 1, 65, None)
    for bad in (dict(x=None), dict(pos=None), dict(D=63), dict(M=-1), dict(ldy=256), dict(hs=32), dict(rope=None)):
        f = dict(x=FAKE, ldx=128, hs=64, ldy=128, pos=FAKE, M=2, D=64, rope=ctypes.byref(rope))
        f.update(bad)
        with pytest.raises(ValueError):
            N.call("mtts_k_rope", f["x"], f["ldx"], f["hs"], FAKE, f["ldy"], f["hs"], f["pos"], f["M"], 2, f["D"], f["rope"],
                   None)


@pytest.mark.parametrize("y,ldy,hsy,M,H", [(FAKE + 64, 128, 64, 2, 2), (FAKE - 126, 128, 64, 2, 2), (FAKE + 4096, 0, 64, 2, 2),
                                           (FAKE + 4096, 64, 64, 2, 2), (FAKE + 4096, 128, 0, 1, 2),
                                           (FAKE + 4096, 32, 0, 2, 1), (FAKE + 4096, 96, 64, 3, 2)])
def test_rope_outputs_that_overlap(N, y, ldy, hsy, M, H):
    r = N.MttsRope(FAKE, 64, 0, 1.0)
    with pytest.raises(ValueError, match="overlap"):
        N.call("mtts_k_rope", FAKE, 128, 64, y, ldy, hsy, FAKE, M, H, 64, ctypes.byref(r), None)


def heads_of(base, ld, hs, M, H, D):
    """every element that a layout touches"""
    return {base + m * ld + h * hs + d for m in range(M) for h in range(H) for d in range(D)}


def rope_accepts(N, x, ldx, hsx, y, ldy, hsy, M, H, D):
    """whether the overlap checks let a call through (elements from FAKE on); a rotary dim that is refused
    behind them keeps it from a launch"""
    with pytest.raises(ValueError) as e:
        N.call("mtts_k_rope", FAKE + 2 * x, ldx, hsx, FAKE + 2 * y, ldy, hsy, FAKE, M, H, D, ctypes.byref(N.MttsRope(FAKE, 3, 0, 1.0)),
               None)
    assert "overlap" in str(e.value) or "arguments" in str(e.value)
    return "overlap" not in str(e.value)


@pytest.mark.parametrize("x,ldx,hsx,y,ldy,hsy,M,H,ok", [
    (0, 256, 64, 64, 256, 64, 2, 2, False),       # by a whole head
    (0, 128, 64, 128, 128, 64, 4, 2, False),      # by a whole token
    (128, 128, 64, 0, 128, 64, 4, 2, False),      # the other way
    (0, 128, 64, 3 * 128, 128, 64, 4, 2, False),  # the last token alone
    (0, 128, 64, 4 * 128, 128, 64, 4, 2, True),   # behind it
    (0, 256, 64, 128, 256, 64, 3, 2, True),       # between the heads of packed rows
    (0, 256, 0, 128, 256, 64, 3, 2, True),        # one head at every place
    (0, 0, 0, 128, 256, 64, 3, 2, True), (130, 0, 0, 0, 128, 64, 3, 2, False),
    (0, 128, 64, 0, 128, 64, 4, 2, True),         # in place
    (0, 128, 64, 0, 64, 128, 2, 2, False),        # the same elements in another order
    (0, 999, 64, 0, 7, 64, 1, 2, True),           # in place: the stride of a single token is no stride
    (0, 128, 64, 0, 128, 999, 2, 1, True), (0, 128, 64, 0, 192, 64, 2, 2, False)])
def test_rope_output_shares_no_head(N, x, ldx, hsx, y, ldy, hsy, M, H, ok):
    assert rope_accepts(N, x, ldx, hsx, y, ldy, hsy, M, H, 64) == ok


def test_rope_overlap_is_exact(N):
    """random layouts against every element that they touch"""
    r = random.Random(5)
    seen = [0, 0]
    for _ in range(3000):
        D, M, H = r.choice([2, 4, 6]), r.randint(1, 5), r.randint(1, 5)
        ldx, hsx = (r.choice([0, D, H * D, M * D, r.randint(0, 40), 2 * H * D]) for _ in range(2))
        ldy, hsy = r.choice([(H * D, D), (D, M * D), (2 * H * D, D), (2 * H * D + 3, 2 * D), (ldx, hsx), (D + 1, M * (D + 1))])
        x, y = r.randint(0, 60), r.randint(0, 60)
        tok, head = (M, ldy), (H, hsy)
        if not any(
                (na == 1 or sa >= D) and (nb == 1 or sb >= (na - 1) * (sa if na > 1 else 0) + D)
                for (na, sa), (nb, sb) in ((tok, head), (head, tok))):
            continue  # (the output's own heads overlap, or its tokens interlock)
        ey = heads_of(y, ldy, hsy, M, H, D)
        same = x == y and (ldx == ldy or M == 1) and (hsx == hsy or H == 1)
        ok = same or not ey & heads_of(x, ldx, hsx, M, H, D)
        assert rope_accepts(N, x, ldx, hsx, y, ldy, hsy, M, H, D) == ok, (x, ldx, hsx, y, ldy, hsy, M, H, D)
        seen[ok] += 1
    assert min(seen) > 300, seen


def append_accepts(N, q, k, v, out, ldq, ldkv, ldo, B, S, H):
    """as rope_accepts; 2 KV heads of 64"""
    with pytest.raises(ValueError) as e:
        N.call("mtts_k_kv_append", ctypes.byref(cache(N, k=FAKE << 8, v=FAKE << 9)), FAKE + 2 * q, ldq, FAKE + 2 * k, ldkv, FAKE + 2 * v, ldkv, FAKE + 2 * out,
               ldo, H, None, None, 0.0, ctypes.byref(N.MttsRope(FAKE, 3, 0, 1.0)), None, FAKE, None, B, S, None)
    assert "overlap" in str(e.value) or "rotary" in str(e.value)
    return "overlap" not in str(e.value)


@pytest.mark.parametrize("q,k,v,out,ldq,ldkv,ldo,B,S,ok", [
    (0, 256, 384, 0, 512, 512, 512, 2, 3, True),      # packed rows, q in place
    (0, 256, 384, 4096, 512, 512, 256, 2, 3, True),
    (0, 256, 384, 512, 512, 512, 512, 1, 2, False),   # the next token's q
    (0, 256, 384, 64, 512, 512, 512, 1, 1, False),    # by a head
    (0, 256, 384, 256, 512, 512, 512, 1, 1, False),   # k
    (0, 256, 384, 384, 512, 512, 512, 1, 1, False),   # v, and what is behind it
    (0, 256, 384, 512, 512, 512, 256, 1, 1, True), (0, 256, 384, 0, 512, 512, 256, 1, 2, False),
    (0, 256, 384, 0, 512, 512, 256, 1, 1, True),      # one token: no stride
    (0, 256, 384, 512, 768, 768, 768, 1, 3, True),    # between the rows' q|k|v
    (0, 256, 384, 513, 768, 768, 768, 1, 3, False), (0, 256, 384, 513, 768, 768, 768, 1, 1, True)])
def test_append_output_is_apart(N, q, k, v, out, ldq, ldkv, ldo, B, S, ok):
    assert append_accepts(N, q, k, v, out, ldq, ldkv, ldo, B, S, 4) == ok


@pytest.mark.parametrize("q,ldq,out,ldo,B,T,ok", [
    (0, 256, 0, 256, 2, 3, True), (0, 512, 0, 512, 2, 3, True),  # in place
    (0, 256, 256, 256, 2, 3, False), (256, 256, 0, 256, 2, 3, False), (0, 256, 5 * 256, 256, 2, 3, False),
    (0, 256, 6 * 256, 256, 2, 3, True), (0, 512, 256, 512, 2, 3, True), (0, 512, 128, 512, 2, 3, False),
    (0, 512, 0, 256, 1, 2, False), (0, 512, 0, 256, 1, 1, True), (0, 256, 64, 256, 1, 1, False),
    (0, 0, 256, 256, 2, 1, True), (256, 0, 0, 256, 2, 1, False)])
def test_attention_output_is_apart(N, q, ldq, out, ldo, B, T, ok):
    """(a workspace that is refused behind the overlap checks keeps the calls from a launch)"""
    with pytest.raises(ValueError) as e:
        N.call("mtts_k_attn_kv", ctypes.byref(cache(N)), FAKE + 2 * q, ldq, FAKE + 2 * out, ldo, 4, FAKE, None, None, None, B, T, 0.0, 0,
               FAKE + 8, None)
    assert ("workspace" in str(e.value)) == ok and ("overlap" in str(e.value)) != ok


BIG = 2 ** 31 - 1


@pytest.mark.parametrize("n", [BIG, BIG - 30, (1 << 25) + 1])
def test_sizes_that_pass_the_index_range(N, n):
    """token and slot counts near 2^31, where rounding up to tiles would pass it"""
    c = ctypes.byref(cache(N))
    with pytest.raises(ValueError, match="2\\^25"):
        N.call("mtts_k_kv_read", c, FAKE, FAKE << 24, None, None, 1, n, None)
    with pytest.raises(ValueError, match="2\\^25"):
        N.call("mtts_k_kv_append", c, None, 0, FAKE, 128, FAKE, 128, None, 0, 0, None, None, 0.0, None, None, FAKE, None, 1, n, None)


def test_tokens_that_pass_the_index_range(N):
    many = ctypes.byref(cache(N, rows=128))
    with pytest.raises(ValueError, match="too many tokens"):
        N.call("mtts_k_kv_append", many, None, 0, FAKE, 128, FAKE, 128, None, 0, 0, None, None, 0.0, None, None, FAKE, None, 128,
               1 << 25, None)
    with pytest.raises(ValueError, match="too many tokens"):
        N.call("mtts_k_attn_kv", many, FAKE, 256, FAKE, 256, 4, FAKE, None, None, None, 128, 1 << 25, 0.0, 0, FAKE + 8, None)


@pytest.mark.parametrize("k,v,ld,ok", [(0, 1 << 20, 128, False), (1 << 20, 0, 128, False), (32767, 1 << 20, 128, False),
                                       (1 << 20, 49151, 128, False), (49152, 16384, 128, True), (65536, 1 << 20, 128, True),
                                       (-256, 1 << 20, 128, True), (-255, 1 << 20, 128, False), (-128, 1 << 20, 20000, True)])
def test_append_from_the_cache_itself(N, k, v, ld, ok):
    """keys or values that lie in the cache would be read while their slots are written; 2 rows x 2 heads x
    64 slots x 64 bf16: K's 16,384 values at 0, V's at 32,768"""
    c = cache(N, type=0, k=FAKE << 8, v=(FAKE << 8) + 65536, k_scale=None, v_scale=None)
    with pytest.raises(ValueError) as e:
        N.call("mtts_k_kv_append", ctypes.byref(c), None, 0, (FAKE << 8) + 2 * k, ld, (FAKE << 8) + 2 * v, ld, None, 0, 0, None, None, 0.0,
               ctypes.byref(N.MttsRope(FAKE, 3, 0, 1.0)), None, FAKE, None, 1, 2, None)
    assert ("rotary" in str(e.value)) == ok and ("cache" in str(e.value)) != ok


def test_output_rows_that_overlap(N):
    c = ctypes.byref(cache(N))
    with pytest.raises(ValueError, match="overlap"):
        N.call("mtts_k_attn_kv", c, FAKE, 256, FAKE, 252, 4, FAKE, None, None, None, 1, 2, 0.0, 0, FAKE, None)
    with pytest.raises(ValueError, match="overlap"):
        N.call("mtts_k_kv_append", c, FAKE, 256, FAKE, 128, FAKE, 128, FAKE, 128, 4, None, None, 0.0, None, None, FAKE, None, 2, 1,
               None)


def test_workspace_bytes(N):
    L = N.load()
    assert L.mtts_k_attn_kv_ws_bytes(64, 64, 32, 8, 128, 2048, 0) == 0  # one block a row and KV head: no partials
    one = L.mtts_k_attn_kv_ws_bytes(1, 1, 32, 8, 128, 131072, 0)
    assert one > 0 and L.mtts_k_attn_kv_ws_bytes(1, 1, 32, 8, 128, 131072, 100) == 0 and one % 4 == 0
    assert L.mtts_kv_bytes(0, 2, 8, 128, 4096) == 2 * L.mtts_kv_bytes(1, 2, 8, 128, 4096) == 2 * 2 * 8 * 128 * 4096


def test_layout_is_a_permutation(kv):
    """the tile layout as the header states it: every (slot, dim) has a byte of its own"""
    for D in (32, 64, 128):
        from tests.kv_layout import k_bytes, v_bytes
        for f in (k_bytes, v_bytes):
            assert sorted(f(D).reshape(-1).tolist()) == list(range(32 * D))
