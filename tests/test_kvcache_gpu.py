"""Drafted-token operators on the GPU against plain implementations in 64 bits.

Tolerances.  Half a bf16 step is 2^-8 of the value, half an e4m3 step 2^-4 (2^-10 of the scale below its
normal range), half an int8 step half the scale; fp32 sums of n terms are off by n 2^-24 of the sum of
their magnitudes.  Each bound below is built from these."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8


@pytest.fixture(scope="module")
def kv():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from moss_tts_amd import _native, kvcache
    _native.load()
    return kvcache


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rnd(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16)


# ---- rope ------------------------------------------------------------------------------------------

def turned(x, pos, turns, factor, rot, interleaved):
    """x [..., H, D] float64, pos [...]: the rotation in 64 bits, and the pairs' |a| + |b|"""
    a = 2 * math.pi * torch.remainder(pos.double()[..., None] * turns, 1.0)[..., None, :]
    c, s = a.cos() * factor, a.sin() * factor
    ii = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    jj = ii + 1 if interleaved else ii + rot // 2
    y, mag = x.clone(), torch.zeros_like(x)
    u, v = x[..., ii], x[..., jj]
    y[..., ii], y[..., jj] = u * c - v * s, v * c + u * s
    mag[..., ii] = mag[..., jj] = (u.abs() + v.abs()) * factor
    return y, mag


# the angle is rounded to 2^-25 of a turn (2^-22.3 rad), its sine and cosine and the two products and
# the sum to a few 2^-24: under 2^-21 of the pair's magnitude; then once to bf16
def rope_close(got, want, mag):
    tol = BF * want.abs() + 2.0 ** -21 * (1 + BF) * mag
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err - tol).max()


YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)


@pytest.mark.parametrize("M,H,D,rot,inter,sc,far", [
    (1, 1, 2, 2, False, None, 10), (1, 40, 128, 128, False, None, 4096), (3, 5, 128, 64, True, None, 131071),
    (17, 9, 64, 16, False, YARN, 131071), (5, 3, 80, 32, True, YARN, 5000), (4, 2, 96, 90, False, None, 70000),
    (2, 3, 128, 10, True, None, 1 << 30), (1000, 7, 128, 128, True, YARN, 131071), (9, 2, 256, 250, False, None, 3000),
    (700, 33, 32, 32, False, dict(rope_type="linear", factor=2.0), 900)])
@pytest.mark.parametrize("where", ["new", "in place", "strided"])
def test_rope(kv, M, H, D, rot, inter, sc, far, where):
    g = torch.Generator().manual_seed(M * 7 + H + D + rot)
    x = rnd(g, M, H, D)
    pos = torch.randint(0, far + 1, (M,), generator=g, dtype=torch.int32)
    pos[0] = far
    r = kv.Rope(D, theta=1e4, rotary_dim=rot, interleaved=inter, scaling=sc)
    turns, factor = kv.rope_turns(rot, 1e4, sc)
    want, mag = turned(x.double(), pos, turns, factor, rot, inter)
    if where == "strided":  # heads inside packed rows, at an odd place
        row = torch.full((M, (H + 2) * D + 3), 7.0, dtype=torch.bfloat16, device="cuda")
        xs = row[:, 1 + D:1 + D + H * D].unflatten(1, (H, D))
        xs.copy_(x)
        keep = row.clone()
        got = r.apply(xs, pos.cuda())
        assert torch.equal(row, keep)
        rope_close(got.cpu(), want, mag)
        r.apply(xs, pos.cuda(), out=xs)
        assert torch.equal(xs, got)
        keep[:, 1 + D:1 + D + H * D] = got.flatten(1)
        assert torch.equal(row, keep)
        return
    xd = x.cuda()
    got = r.apply(xd, pos.cuda(), out=xd if where == "in place" else None)
    rope_close(got.cpu(), want, mag)
    if where == "new":
        assert torch.equal(xd.cpu(), x)


def test_rope_step_equals_prompt_and_undoes(kv):
    """a token alone gives the bits it gives in a prompt; explicit frequencies of opposite sign turn back"""
    g = torch.Generator().manual_seed(2)
    x = rnd(g, 50, 6, 128).cuda()
    pos = torch.arange(90000, 90050, dtype=torch.int32, device="cuda")
    r = kv.Rope(128)
    y = r.apply(x, pos)
    for m in (0, 31, 49):
        assert torch.equal(r.apply(x[m:m + 1], pos[m:m + 1]), y[m:m + 1])
    f = kv.rope_turns(128, 1e6)[0] * 2 * math.pi
    back = kv.Rope(128, inv_freq=-f).apply(y, pos).double()
    pair = x.double()[..., :64].abs() + x.double()[..., 64:].abs()
    # two roundings to bf16 of values no larger than the pair's magnitude
    assert ((back - x.double()).abs() <= 2 * (BF + 2.0 ** -20) * torch.cat([pair, pair], -1)).all()


def test_rope_refusals(kv):
    r = kv.Rope(64)
    x, p = torch.zeros(2, 3, 64, dtype=torch.bfloat16, device="cuda"), i32([0, 1])
    for bad in (lambda: r.apply(x.float(), p), lambda: r.apply(x[..., :32], p), lambda: r.apply(x, p.long()),
                lambda: r.apply(x, i32([0])), lambda: r.apply(x, p.cpu()), lambda: r.apply(x.cpu(), p),
                lambda: r.apply(x, p, out=x[:1]), lambda: kv.Rope(63), lambda: kv.Rope(64, rotary_dim=66),
                lambda: r.apply(x.transpose(1, 2).contiguous().transpose(1, 2), p),
                lambda: kv.Rope(64, inv_freq=torch.ones(3))):
        with pytest.raises(ValueError):
            bad()
    assert r.apply(x[:0], p[:0]).shape == (0, 3, 64)


# ---- the cache -------------------------------------------------------------------------------------

QMAX = {"e4m3": 448.0, "int8": 127.0}


def stored(x, kind):
    """bf16 values as the cache holds them: the definition in 32 bits (exact for bf16 x, see the
    quantiser's comment), as 64-bit values of code * scale, and the scales"""
    if kind == "bf16":
        return x.double(), None
    x = x.float()
    a = x.abs().amax(-1, keepdim=True)
    sh = torch.where(a > 2.0 ** 100, 2.0 ** -64, 1.0)
    live = (a >= 2.0 ** -100) & torch.isfinite(a)
    y = torch.where(live, x * (QMAX[kind] * sh) / torch.where(live, a * sh, 1.0), 0.0).clamp(-QMAX[kind], QMAX[kind])
    c = y.to(torch.float8_e4m3fn).double() if kind == "e4m3" else y.round().double()
    scale = torch.where(live, a / QMAX[kind], torch.where(a < 2.0 ** -100, 0.0, float("nan")))
    return c * scale.double(), scale[..., 0]


def fresh(kv, rows, n_kv, slots, D, kind, fill=0xFF):
    """a cache whose bytes are all `fill` (NaN in every type)"""
    c = kv.KVCache(rows, n_kv, slots, D, kind)
    for t in (c.k, c.v, c.k_scale, c.v_scale):
        if t is not None:
            t.view(torch.uint8).fill_(fill)
    return c


def raw(c):
    return [t.view(torch.uint8).cpu().clone() for t in (c.k, c.v, c.k_scale, c.v_scale) if t is not None]


KINDS = ["bf16", "e4m3", "int8"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,S,starts,counts", [(1, 1, [0], None), (1, 1, [63], None), (2, 5, [30, 31], None),
                                               (3, 70, [0, 33, 100], [70, 0, 41]), (2, 32, [32, 96], None),
                                               (2, 9, [250, 256], [9, 3]), (1, 3, [-1], [7])])
def test_write_and_read(kv, kind, D, B, S, starts, counts):
    """keys and values without rotation are stored to the bit, where they belong and nowhere else"""
    from tests.kv_layout import contents
    g = torch.Generator().manual_seed(D + S)
    Hkv, slots = 3, 256
    k, v = rnd(g, B, S, Hkv, D, scale=3.0), rnd(g, B, S, Hkv, D, scale=0.01)
    c = fresh(kv, B + 1, Hkv, slots, D, kind, fill=0x11)
    before = contents(c)
    c.write(k.cuda(), v.cuda(), i32(starts), counts=None if counts is None else i32(counts))
    after = contents(c)
    for x, was, got in zip((k, v), before, after):
        want = was.clone()
        val, _ = stored(x, kind)
        for b in range(B):
            n = S if counts is None else min(S, counts[b])
            for t in range(n):
                if 0 <= starts[b] + t < slots:
                    want[b, :, starts[b] + t] = val[b, t]
        assert torch.equal(got, want)
    n = S + 3
    for got, held in zip(c.read(n, start=i32(starts), counts=None if counts is None else i32(counts)), after):
        want = torch.zeros(B, Hkv, n, D, dtype=torch.bfloat16)
        for b in range(B):
            for t in range(n if counts is None else min(n, counts[b])):
                if 0 <= starts[b] + t < slots:
                    # (value = code * scale rounded to 32 bits, then to bf16, as the kernel's product)
                    want[b, :, t] = held[b, :, starts[b] + t].float().to(torch.bfloat16)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_every_code_comes_back(kv, kind):
    """all finite codes, through the quantiser and back"""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn if kind == "e4m3" else torch.int8).float()
    codes = codes[codes.isfinite() & (codes.abs() <= QMAX[kind])]
    D = 128
    rows = torch.nn.functional.pad(codes, (0, -codes.numel() % (D - 1))).view(-1, D - 1)
    rows = torch.cat([torch.full((rows.shape[0], 1), QMAX[kind]), rows], 1)  # the row's largest sets the scale to 1
    x = rows.to(torch.bfloat16)[None, :, None]
    assert torch.equal(x.float()[0, :, 0], rows)
    c = kv.KVCache(1, 1, 64, D, kind)
    c.write(x.cuda(), x.cuda(), i32([0]))
    for got in c.read(rows.shape[0]):
        assert torch.equal(got.cpu()[0, 0].float(), rows)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_odd_rows(kv, kind):
    """zeros, rows below 2^-100, rows near the type's largest, NaN and infinities: the row's own affair"""
    from tests.kv_layout import codes, contents
    g = torch.Generator().manual_seed(4)
    D = 64
    x = rnd(g, 1, 9, 2, D)
    x[0, 1] = 0
    x[0, 2] *= 2.0 ** -101
    x[0, 2] = x[0, 2].clamp(-2.0 ** -101, 2.0 ** -101)
    x[0, 3] *= 2.0 ** -90
    x[0, 4] *= 2.0 ** 120
    x[0, 4, :, 7] = torch.finfo(torch.bfloat16).max
    x[0, 5, :, 3] = float("nan")
    x[0, 6, :, 60] = float("-inf")
    c = fresh(kv, 1, 2, 64, D, kind)
    c.write(x.cuda(), x.cuda(), i32([0]))
    want, _ = stored(x, kind)
    for got, code in zip(contents(c), codes(c)):
        got, code = got[0, :, :9].transpose(0, 1), code[0, :, :9].transpose(0, 1)
        assert got[5:7].isnan().all() and (code[5:7] == 0).all() and (got[1:3] == 0).all()
        keep = [0, 1, 2, 3, 4, 7, 8]
        assert torch.equal(got[keep], want[0, keep])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_heads,n_kv,D,rot,inter,norm,B,S", [(4, 1, 128, 128, False, True, 1, 1), (8, 2, 64, 32, True, True, 2, 3),
                                                              (14, 2, 128, 64, False, False, 2, 37), (3, 3, 32, 10, True, True, 2, 5),
                                                              (6, 2, 64, 64, False, True, 1, 300)])
def test_append(kv, kind, n_heads, n_kv, D, rot, inter, norm, B, S):
    """norm, rotation at explicit positions, quantisation: q and the keys within the roundings' bounds, the
    values to the bit"""
    from tests.kv_layout import contents
    g = torch.Generator().manual_seed(n_heads + S)
    heads = n_heads + 2 * n_kv
    qkv = rnd(g, B, S, heads * D)
    qn, kn = ((0.5 + torch.rand(2, D, generator=g)).to(torch.bfloat16)) if norm else (None, None)
    starts, counts = [7 * b + 3 for b in range(B)], [S - b for b in range(B)]
    pos = torch.randint(0, 100000, (B, S), generator=g, dtype=torch.int32)
    r = kv.Rope(D, theta=1e6, rotary_dim=rot, interleaved=inter, scaling=YARN)
    turns, factor = kv.rope_turns(rot, 1e6, YARN)
    c = fresh(kv, B, n_kv, 512, D, kind)
    q = torch.full((B, S, n_heads, D), 9.0, dtype=torch.bfloat16, device="cuda")
    got = c.append(qkv.cuda(), i32(starts), n_heads, rope=r, positions=pos.cuda(), counts=i32(counts),
                   q_norm=None if qn is None else qn.cuda(), k_norm=None if kn is None else kn.cuda(), out=q)
    assert got is q
    x = qkv.double().view(B, S, heads, D)

    def normed(y, w):
        return y if w is None else y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    wq, mq = turned(normed(x[:, :, :n_heads], qn), pos, turns, factor, rot, inter)
    wk, mk = turned(normed(x[:, :, n_heads:-n_kv], kn), pos, turns, factor, rot, inter)
    # the norm's sum of squares is off by D 2^-24, its root and products by a few steps: under 2^-16 of a
    # value for D <= 128; the rotation as above
    fp = 2.0 ** -16
    ck, cv = contents(c)
    for b in range(B):
        n = counts[b]
        err = (q[b, :n].cpu().double() - wq[b, :n]).abs()
        assert (err <= BF * wq[b, :n].abs() + fp * (wq[b, :n].abs() + mq[b, :n])).all()
        assert (q[b, n:] == 9.0).all()
        held, want = ck[b, :, starts[b]:starts[b] + n].transpose(0, 1), wk[b, :n]
        a = want.abs().amax(-1, keepdim=True)
        step = BF * want.abs() if kind == "bf16" else (0.5 * a / 127 if kind == "int8" else
                                                       torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * a / 448))
        err = (held - want).abs()
        assert (err <= (step + fp * (a + mk[b, :n])) * (1 + fp)).all(), (err - step).max()
        sv, _ = stored(x[b, :n, -n_kv:].to(torch.bfloat16), kind)
        assert torch.equal(cv[b, :, starts[b]:starts[b] + n].transpose(0, 1), sv)
    # positions left out are the slots
    p2 = (torch.tensor(starts)[:, None] + torch.arange(S)).to(torch.int32).cuda()
    one, two = fresh(kv, B, n_kv, 512, D, kind), fresh(kv, B, n_kv, 512, D, kind)
    q1 = one.append(qkv.cuda(), i32(starts), n_heads, rope=r)
    q2 = two.append(qkv.cuda(), i32(starts), n_heads, rope=r, positions=p2)
    assert torch.equal(q1, q2) and all(torch.equal(u, w) for u, w in zip(raw(one), raw(two)))


def test_append_strided_rows(kv):
    """a packed row wider than q|k|v, and one that is not 16-byte aligned, give the same bits"""
    g = torch.Generator().manual_seed(8)
    B, S, H, Hkv, D = 2, 6, 4, 2, 64
    W = (H + 2 * Hkv) * D
    qkv = rnd(g, B, S, W).cuda()
    r = kv.Rope(D, rotary_dim=32)
    want = None
    for off, pad in ((0, 0), (8, 16), (1, 3)):
        row = torch.zeros(B * S, off + W + pad, dtype=torch.bfloat16, device="cuda")
        row[:, off:off + W] = qkv.view(-1, W)
        c = fresh(kv, B, Hkv, 64, D, "e4m3")
        q = c.append(row.view(B, S, -1)[..., off:off + W], i32([0, 40]), H, rope=r)
        now = [q.cpu().view(torch.uint8), *raw(c)]
        want = want or now
        assert all(torch.equal(a, b) for a, b in zip(now, want))


@pytest.mark.parametrize("B,S", [(1, 1), (2, 5)])
def test_append_outputs_that_share(kv, B, S):
    """q rotated where it lies is as into a new tensor; an output elsewhere inside qkv is refused"""
    import ctypes
    from moss_tts_amd import _native as N
    g = torch.Generator().manual_seed(9)
    H, Hkv, D = 4, 2, 64
    W = (H + 2 * Hkv) * D
    qkv, qn = rnd(g, B, S, W).cuda(), rnd(g, D).cuda()
    r, at = kv.Rope(D, rotary_dim=32), i32([3] * B)
    one, two = (fresh(kv, B, Hkv, 64, D, "int8") for _ in range(2))
    want = one.append(qkv, at, H, rope=r, q_norm=qn)
    for off in (D, W - H * D):
        flat = qkv.view(-1)[off:]
        if flat.numel() >= B * S * H * D:
            with pytest.raises(ValueError, match="overlap"):
                two.append(qkv, at, H, rope=r, q_norm=qn, out=flat[:B * S * H * D].view(B, S, H, D))
    p = qkv.data_ptr()
    N.call("mtts_k_kv_append", two._ref, p, W, p + 2 * H * D, W, p + 2 * (H + Hkv) * D, W, p, W, H, qn.data_ptr(), None, 1e-6,
           ctypes.byref(r._c), None, at.data_ptr(), None, B, S, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(qkv.view(B, S, -1, D)[:, :, :H], want)
    assert all(torch.equal(x, y) for x, y in zip(raw(one), raw(two)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("P,path,took,start", [(1, [[0]], [1], [3]), (5, [[0, 2, 4, 1, 1], [1, 0, 3, 3, 2]], [3, 5], [30, 0]),
                                               (64, None, [64, 20], [1, 190]), (4, [[0, 63, -1, 64], [2, 1, 0, 3]], [4, -2], [60, 5]),
                                               (3, [[1, 2, 3], [4, 5, 6]], [9, 2], [254, 255])])
def test_compact(kv, kind, P, path, took, start):
    from tests.kv_layout import contents
    g = torch.Generator().manual_seed(P)
    B, Hkv, slots, D = len(took), 2, 256, 64
    path = path or torch.stack([torch.randperm(64, generator=g) for _ in range(B)]).tolist()
    c = kv.KVCache(B + 1, Hkv, slots, D, kind)
    c.write(rnd(g, B + 1, slots, Hkv, D).cuda(), rnd(g, B + 1, slots, Hkv, D).cuda(), i32([0] * (B + 1)))
    want = [x.clone() for x in contents(c)]
    old = contents(c)
    for b in range(B):
        for i in range(max(0, min(took[b], P))):
            f, t = start[b] + path[b][i], start[b] + i
            if 0 <= path[b][i] < 64 and f < slots and t < slots:
                for w, o in zip(want, old):
                    w[b, :, t] = o[b, :, f]
    c.compact(i32(start), i32(path), i32(took))
    for w, o in zip(want, contents(c)):
        assert torch.equal(o, w)


# ---- attention -------------------------------------------------------------------------------------

def sees(B, T, slots, start, counts, tree, mask):
    """[B, T, slots] truth values from the definition"""
    out = torch.zeros(B, T, slots, dtype=torch.bool)
    for b in range(B):
        n = T if counts is None else counts[b]
        for t in range(n):
            for j in range(min(start[b], slots)):
                out[b, t, j] = mask is None or bool(mask[b, j])
            for u in range(n):
                if 0 <= start[b] + u < slots:
                    out[b, t, start[b] + u] = (u <= t) if tree is None else bool(tree[b][t] >> u & 1)
    return out


def attend64(q, k, v, see, scale):
    """the definition in 64 bits; what is not seen does not exist.  Also the bound's parts: sum p |v| and
    the largest sum |q| |k| of a token"""
    B, T, H, D = q.shape
    G = H // k.shape[1]
    o, pv, qk = (torch.zeros(B, T, H, D, dtype=torch.float64) for _ in range(3))
    for b in range(B):
        for t in range(T):
            j = see[b, t].nonzero()[:, 0]
            if len(j) == 0:
                continue
            kk, vv = k[b][:, j], v[b][:, j]  # [Hkv, n, D]
            x = q[b, t].double().view(-1, G, D)
            p = torch.softmax(scale * x @ kk.transpose(1, 2), -1)
            o[b, t] = (p @ vv).view(H, D)
            pv[b, t] = (p @ vv.abs()).view(H, D)
            qk[b, t] = (x.abs() @ kk.abs().transpose(1, 2)).amax(-1).view(H, 1) * scale
    return o, pv, qk


# Each p is rounded to bf16 (BF of it); a score is off by the products' sum (D + 8 steps of 2^-24 of sum
# |q||k|), the rounded factor log2(e) * scale and the power of two (2^-21 of a score and 2^-20 beside
# it), twice: above and below the line; the result is rounded once.
def attention_close(got, o, pv, qk, D, live=None):
    d = (D + 8) * 2.0 ** -24 * qk + 2.0 ** -21 * qk + 2.0 ** -20
    tol = BF * o.abs() + (BF + 2.5 * d) * (1 + BF) * pv
    err = (got.double() - o).abs()
    ok = (err <= tol) if live is None else (err <= tol) | ~live
    assert ok.all(), float((err - tol).max())


def trees(g, B, T):
    out = []
    for _ in range(B):
        m = [1]
        for t in range(1, T):
            p = int(torch.randint(max(0, t - 4), t, (1,), generator=g))
            m.append(m[p] | 1 << t)
        out.append(m)
    return out


def signed(tree):
    return torch.tensor([[x - (1 << 64) if x >> 63 else x for x in r] for r in tree], dtype=torch.int64, device="cuda")


def attend_case(kv, kind, B, T, H, Hkv, D, start, tree=False, masked=False, counts=None, max_len=None, scale=None, seed=0,
                spread=1.5):
    from tests.kv_layout import contents
    g = torch.Generator().manual_seed(seed + B * 1000 + T * 10 + H + D)
    slots = (max(start) + T + 63) // 64 * 64
    c = fresh(kv, B, Hkv, slots, D, kind)  # what is not written is NaN
    S = max(start) + T
    lens = [s + (T if counts is None else counts[b]) for b, s in enumerate(start)]
    c.write(rnd(g, B, S, Hkv, D, scale=spread).cuda(), rnd(g, B, S, Hkv, D).cuda(), i32([0] * B), counts=i32(lens))
    q = rnd(g, B, T, H, D, scale=spread)
    tr = trees(g, B, T) if tree else None
    mask = None
    if masked:
        mask = torch.rand(B, slots, generator=g) < 0.7
        mask[0, :start[0]] = False  # one row's context is all padding
        for t in (c.k, c.v):  # and padded places hold NaN in the bf16 cache
            if kind == "bf16" and t is c.k:
                t.masked_fill_(~mask.cuda()[:, None, :, None] & _context(start, slots)[:, None, :, None], float("nan"))
            elif kind == "bf16":
                t.masked_fill_(~mask.cuda()[:, None, None, :] & _context(start, slots)[:, None, None, :], float("nan"))
    out = torch.full((B, T, H, D), 5.0, dtype=torch.bfloat16, device="cuda")
    got = c.attend(q.cuda(), i32(start), tree=signed(tr) if tree else None, counts=None if counts is None else i32(counts),
                   mask=None if mask is None else mask.cuda(), max_len=max_len, scale=scale, out=out)
    k, v = contents(c)
    see = sees(B, T, slots, start, counts, tr, mask)
    o, pv, qk = attend64(q, k, v, see, scale or D ** -0.5)
    got = got.cpu()
    for b in range(B):
        n = T if counts is None else counts[b]
        assert (got[b, n:] == 5.0).all()
        got[b, n:] = 0
        empty = ~see[b].any(-1)
        assert (got[b][empty] == 0).all()
    attention_close(got, o, pv, qk, D)


def _context(start, slots):
    return torch.arange(slots, device="cuda")[None] < i32(start)[:, None]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,T,H,Hkv,start,kw", [
    (1, 1, 1, 1, [0], {}), (1, 1, 4, 1, [31], {}), (1, 1, 8, 2, [32], {}), (2, 1, 8, 2, [700, 1], {}),
    (1, 2, 2, 2, [63], {}), (2, 7, 8, 2, [65, 0], dict(tree=True)), (1, 64, 4, 1, [40], dict(tree=True)),
    (3, 17, 6, 2, [200, 33, 0], dict(tree=True, masked=True)), (2, 33, 7, 1, [100, 31], dict(masked=True)),
    (3, 12, 4, 2, [50, 64, 10], dict(tree=True, counts=[12, 0, 5])), (1, 150, 4, 2, [70], {}),
    (2, 90, 2, 1, [0, 5], dict(counts=[1, 90]))])
def test_attend(kv, kind, D, B, T, H, Hkv, start, kw):
    attend_case(kv, kind, B, T, H, Hkv, D, start, **kw)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T,H,Hkv,start,kw", [
    (1, 1, 4, 1, [9000], {}), (3, 5, 4, 2, [6000, 0, 1234], dict(tree=True)), (2, 20, 8, 2, [3000, 2999], dict(tree=True, masked=True)),
    (2, 1, 4, 2, [4000, 17], dict(max_len=10)), (1, 1, 4, 1, [2500], dict(max_len=100000, scale=0.5)),
    (2, 40, 4, 1, [5000, 130], dict(counts=[40, 3])), (70, 1, 2, 1, [(97 * b) % 640 for b in range(70)], dict(max_len=8000))])
def test_attend_split(kv, kind, B, T, H, Hkv, start, kw):
    """long and ragged contexts, worked on by several blocks a row"""
    attend_case(kv, kind, B, T, H, Hkv, 128, start, **kw)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,T,H,Hkv,start,kw", [
    (1, 1, 32, 1, [300], dict(masked=True)), (2, 1, 33, 1, [40, 900], {}), (1, 1, 32, 1, [3500], {}),
    (2, 12, 8, 2, [2100, 40], dict(tree=True, masked=True)), (2, 64, 8, 2, [1500, 2050], dict(tree=True, masked=True, counts=[64, 40])),
    (1, 64, 16, 2, [1800], dict(tree=True)), (1, 150, 4, 2, [1700], {}), (3, 70, 4, 1, [31, 900, 0], dict(masked=True)),
    (70, 12, 4, 1, [(97 * b) % 640 for b in range(70)], dict(max_len=2000, counts=[b % 13 for b in range(70)]))])
def test_attend_groups_and_forms(kv, kind, D, B, T, H, Hkv, start, kw):
    """groups of a tile of rows and one more; one, two, four and more tiles of rows, split and not"""
    attend_case(kv, kind, B, T, H, Hkv, D, start, **kw)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T,H,Hkv", [(130, 10, 16, 2), (130, 24, 8, 2), (65, 33, 16, 4)])
def test_attend_many_short_rows(kv, kind, B, T, H, Hkv):
    """more rows and heads than the card has compute units: three row tiles a block, and others"""
    attend_case(kv, kind, B, T, H, Hkv, 32, [(7 * b) % 90 for b in range(B)], tree=True,
                counts=[T - b % 3 if b % 11 else 0 for b in range(B)])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,H,split", [(1, 8, False), (12, 8, False), (30, 8, False), (64, 8, False), (1, 8, True), (12, 8, True),
                                       (64, 8, True)])
def test_rows_beside_other_rows(kv, kind, T, H, split):
    """A row beside others of other lengths and contents.  Without a workspace its bits are the same; with one,
    long rows are cut where the lengths of all rows put the cuts: the same within rounding, and the same bits for
    the same call"""
    from moss_tts_amd import _native as N
    g = torch.Generator().manual_seed(T)
    Hkv, D, B, slots, n = 2, 64, 3, 6080 if split else 512, 5000 if split else 400
    assert (N.load().mtts_k_attn_kv_ws_bytes(B, T, H, Hkv, D, slots, 0) > 0) == split
    k, v, q = rnd(g, B, slots, Hkv, D).cuda(), rnd(g, B, slots, Hkv, D).cuda(), rnd(g, B, T, H, D).cuda()
    outs = []
    for other in ([0, 0], [17, 33], [slots - T, 100], [40, slots]):
        c = fresh(kv, B, Hkv, slots, D, kind)
        c.write(k, v, i32([0] * B))
        for max_len in (None, slots):
            outs.append(c.attend(q, i32([other[0], n, other[1]]), max_len=max_len)[1].clone())
        assert torch.equal(outs[-1], c.attend(q, i32([other[0], n, other[1]]), max_len=slots)[1])
        k[[0, 2]], v[[0, 2]], q[[0, 2]] = -k[[0, 2]] * 3, v[[0, 2]] + 1, q[[2, 0]]
    if not split:
        assert all(torch.equal(x, outs[0]) for x in outs)
    see = sees(B, T, slots, [0, n, 0], None, None, None)[1:2]
    from tests.kv_layout import contents
    ck, cv = (x[1:2] for x in contents(c))
    for x in outs:
        attention_close(x[None].cpu(), *attend64(q[1:2].cpu(), ck, cv, see, D ** -0.5), D)


def test_two_streams_at_once(kv):
    """calls of two streams over one cache, each with a workspace of its own, as one after the other"""
    g = torch.Generator().manual_seed(11)
    c = fresh(kv, 2, 2, 4096, 128, "int8")
    c.write(rnd(g, 2, 4000, 2, 128).cuda(), rnd(g, 2, 4000, 2, 128).cuda(), i32([0, 0]))
    qs = [rnd(g, 2, T, 8, 128).cuda() for T in (1, 8, 30, 64)]
    at = i32([3900, 2500])
    want = [c.attend(q, at) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append([c.attend(q, at) for q in (qs if i else qs[::-1])])
    torch.cuda.synchronize()
    for run in got[0]:
        assert all(torch.equal(x, y) for x, y in zip(run[::-1], want))
    for run in got[1]:
        assert all(torch.equal(x, y) for x, y in zip(run, want))


@pytest.mark.parametrize("kind", KINDS)
def test_attend_large_scores(kv, kind):
    """scores of hundreds: one key takes nearly all, the running maximum moves"""
    attend_case(kv, kind, 1, 9, 4, 1, 128, [500], tree=True, spread=5.0)


FAR = 2 ** 31 - 1


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,G", [(3, 2), (40, 4), (64, 4)])
@pytest.mark.parametrize("slots", [64, 4096])
@pytest.mark.parametrize("tree", [False, True])
def test_starts_outside_the_cache(kv, kind, T, G, slots, tree):
    """new tokens before slot 0 or behind the last have no slot: nothing is stored for them, read from them or
    moved to them, and attention sees those tokens that have one"""
    from tests.kv_layout import contents
    g = torch.Generator().manual_seed(T + G + slots)
    start = [-2, 5 - T, -T - 40, slots - 2, slots, FAR, FAR - 7, -FAR - 1]
    B, D, n_kv = len(start), 64, 2
    c = fresh(kv, B, n_kv, slots, D, kind)
    c.write(rnd(g, B, slots, n_kv, D).cuda(), rnd(g, B, slots, n_kv, D).cuda(), i32([0] * B))
    before = [t.clone() for t in contents(c)]
    new = rnd(g, B, T, n_kv, D)
    c.write(new.cuda(), new.cuda(), i32(start))
    want = stored(new, kind)[0]
    for x, y in zip(contents(c), before):
        for b in range(B):
            for u in range(T):
                if 0 <= start[b] + u < slots:
                    y[b, :, start[b] + u] = want[b, u]
        assert torch.equal(x, y)
    q = rnd(g, B, T, G * n_kv, D)
    tr = trees(g, B, T) if tree else None
    got = c.attend(q.cuda(), i32(start), tree=signed(tr) if tree else None).cpu()
    o, pv, qk = attend64(q, *before, sees(B, T, slots, start, None, tr, None), D ** -0.5)
    attention_close(got, o, pv, qk, D)
    for r in c.read(T, start=i32(start)):
        for b in range(B):
            for u in range(T):
                if not 0 <= start[b] + u < slots:
                    assert (r[b, :, u] == 0).all()
    path = torch.arange(T, dtype=torch.int32).repeat(B, 1).flip(1).cuda()
    c.compact(i32(start), path, i32([T] * B))
    for x, y in zip(contents(c), before):
        for b in range(B):
            old = y[b].clone()
            for i in range(T):
                t, f = start[b] + i, start[b] + T - 1 - i
                if 0 <= t < slots and 0 <= f < slots:
                    y[b, :, t] = old[:, f]
        assert torch.equal(x, y)


def test_rope_broadcast_and_gaps(kv):
    """one head's values at every token and head; an output between the input's heads"""
    g = torch.Generator().manual_seed(1)
    r, pos = kv.Rope(64, theta=1e4), i32([3, 70, 9])
    x = rnd(g, 1, 1, 64).cuda()
    assert torch.equal(r.apply(x.expand(3, 5, 64), pos), r.apply(x.repeat(3, 5, 1), pos))
    rows = rnd(g, 3, 4, 64).cuda()
    want = r.apply(rows[:, :2].contiguous(), pos)
    kept = rows[:, :2].clone()
    r.apply(rows[:, :2], pos, out=rows[:, 2:])
    assert torch.equal(rows[:, 2:], want) and torch.equal(rows[:, :2], kept)
    for bad in (x.expand(3, 5, 64), rows.view(-1)[64 + 32:64 + 32 + 3 * 128].view(3, 2, 64)):
        with pytest.raises(ValueError, match="overlap"):
            r.apply(rows.view(-1)[64:64 + 3 * 128].view(3, 2, 64) if bad.shape[1] == 2 else rows[:, :1].expand(3, 5, 64), pos, out=bad)


def test_rope_outputs_that_share_heads(kv):
    """an output shifted by a head or a token is refused, and nothing is written; one between the input's heads
    or behind its tokens is as a new one"""
    g = torch.Generator().manual_seed(3)
    r, pos = kv.Rope(64, theta=1e4), i32([3, 70, 9])
    buf = rnd(g, 6, 4, 64).cuda()
    keep = buf.clone()
    for x, out in ((buf[:3, :2], buf[:3, 1:3]), (buf[:3], buf[1:4]), (buf[1:4], buf[:3]), (buf[:3], buf[2:5]),
                   (buf[:3, 1:3], buf[:3, :2]), (buf[1:2].expand(3, 4, 64), buf[:3])):
        with pytest.raises(ValueError, match="overlap"):
            r.apply(x, pos, out=out)
        assert torch.equal(buf, keep)
    for x, out in ((buf[:3], buf[3:]), (buf[:3, :1].expand(3, 2, 64), buf[:3, 2:]), (buf[5:, 1:2].expand(3, 3, 64), buf[:3, :3]),
                   (buf[:3, ::2], buf[:3, 1::2])):
        buf.copy_(keep)
        want = r.apply(x.contiguous(), pos)
        r.apply(x, pos, out=out)
        assert torch.equal(out, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T,H,start", [(1, 1, 4, [300]), (2, 6, 4, [9000, 50]), (3, 20, 8, [40, 1300, 0]), (2, 40, 8, [5000, 4000]),
                                         (2, 150, 6, [90, 600])])
def test_attend_in_place(kv, kind, B, T, H, start):
    """out = q is as a new output, in every form, split and not; an output shifted inside q is refused"""
    g = torch.Generator().manual_seed(T)
    Hkv, D, S = 2, 64, max(start) + T
    c = fresh(kv, B, Hkv, S, D, kind)
    c.write(rnd(g, B, S, Hkv, D).cuda(), rnd(g, B, S, Hkv, D).cuda(), i32([0] * B))
    buf = rnd(g, B * T * H * D + D).cuda()
    q, at = buf[:-D].view(B, T, H, D), i32(start)
    want = c.attend(q, at)
    with pytest.raises(ValueError, match="overlap"):
        c.attend(q, at, out=buf[D:].view(B, T, H, D))
    assert c.attend(q, at, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("kind", KINDS)
def test_attend_single_token_of_an_odd_row(kv, kind):
    """one token out of rows of odd length: its address is what counts, there is no next one"""
    g = torch.Generator().manual_seed(3)
    c = fresh(kv, 1, 2, 64, 64, kind)
    c.write(rnd(g, 1, 41, 2, 64).cuda(), rnd(g, 1, 41, 2, 64).cuda(), i32([0]))
    q = torch.empty(1, 1, 4, 64, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, 4, 64), (259, 259, 64, 1))
    q.copy_(rnd(g, 1, 1, 4, 64))
    want = c.attend(q.as_strided((1, 1, 4, 64), (256, 256, 64, 1)), i32([40]))
    assert q.stride(0) == 259 and torch.equal(c.attend(q, i32([40])), want)


@pytest.mark.parametrize("kind", KINDS)
def test_nothing_seen_is_zero(kv, kind):
    c = fresh(kv, 2, 1, 256, 64, kind)
    q = torch.ones(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    mask = torch.zeros(2, 256, dtype=torch.uint8, device="cuda")
    got = c.attend(q, i32([200, 0]), tree=torch.zeros(2, 3, dtype=torch.int64, device="cuda"), mask=mask)
    assert (got == 0).all()
    got = c.attend(q[:, :1], i32([256, 300]), mask=mask)  # the new tokens have no slot
    assert (got == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("long", [0, 1300])
def test_what_is_not_seen_never_reaches(kv, kind, what, long):
    """a drafted token whose key or value is not finite: the rows that do not see it are as without it"""
    g = torch.Generator().manual_seed(6)
    T, H, Hkv, D, n = 6, 4, 2, 64, 37 + long
    k, v, q = rnd(g, 1, n + T, Hkv, D), rnd(g, 1, n + T, Hkv, D), rnd(g, 1, T, H, D).cuda()
    tree = signed([[1, 3, 5, 11, 21, 35]])  # token 2 and 4 see token 2; token 3 and 5 see token 1
    outs = []
    for bad in (False, True):
        if bad:
            v[0, n + 1, 1, 5] = what
            k[0, n + 2, 0, 9] = what
        c = fresh(kv, 1, Hkv, n + T, D, kind)
        c.write(k.cuda(), v.cuda(), i32([0]))
        outs.append(c.attend(q, i32([n]), tree=tree).cpu()[0])
    good, got = outs
    see_v, see_k = [1, 3, 5], [2, 4]
    for t in range(T):
        for h in range(H):
            hk = h // (H // Hkv)
            if hk == 1 and t in see_v:
                assert not got[t, h, 5].isfinite()
                if kind == "bf16":
                    assert got[t, h, 5].isnan() if math.isnan(what) else got[t, h, 5] == what
                    assert torch.equal(got[t, h, :5], good[t, h, :5]) and torch.equal(got[t, h, 6:], good[t, h, 6:])
                else:
                    assert got[t, h].isnan().all()
            elif hk == 0 and t in see_k:
                if math.isnan(what) or kind != "bf16":
                    assert got[t, h].isnan().all()
            else:
                assert torch.equal(got[t, h], good[t, h]), (t, h)


def test_same_bits_every_time(kv):
    g = torch.Generator().manual_seed(1)
    c = kv.KVCache(2, 2, 8192, 128, "e4m3")
    c.write(rnd(g, 2, 8192, 2, 128).cuda(), rnd(g, 2, 8192, 2, 128).cuda(), i32([0, 0]))
    q = rnd(g, 2, 16, 8, 128).cuda()
    first = c.attend(q, i32([8000, 4001]))
    for _ in range(5):
        assert torch.equal(c.attend(q, i32([8000, 4001])), first)


def test_long_cache_offsets(kv):
    """a cache of more than 2^31 values: the last row, slot and head"""
    from moss_tts_amd import _native as N
    rows, Hkv, slots, D = 17, 8, 131072, 128
    g = torch.Generator().manual_seed(3)
    c = kv.KVCache(rows, Hkv, slots, D, "e4m3")
    assert c.k.numel() > 1 << 31
    n = 40
    k, v = rnd(g, rows, n, Hkv, D).cuda(), rnd(g, rows, n, Hkv, D).cuda()
    at = i32([slots - n] * rows)
    c.write(k, v, at)
    gk, gv = c.read(n, start=at)
    for x, got in ((k, gk), (v, gv)):
        val, _ = stored(x.cpu(), "e4m3")
        assert torch.equal(got.cpu(), val.float().to(torch.bfloat16).transpose(1, 2))
    mask = torch.zeros(rows, slots, dtype=torch.uint8, device="cuda")
    mask[:, slots - n:] = 1
    q = rnd(g, rows, 1, 16, D)
    got = c.attend(q.cuda(), i32([slots - 1] * rows), mask=mask).cpu()
    o, pv, qk = attend64(q[-1:], stored(k.cpu(), "e4m3")[0].transpose(1, 2)[-1:], stored(v.cpu(), "e4m3")[0].transpose(1, 2)[-1:],
                         torch.ones(1, 1, n, dtype=torch.bool), D ** -0.5)
    attention_close(got[-1:], o, pv, qk, D)
    c.compact(i32([slots - n] * rows), i32([[n - 1, n - 2]] * rows), i32([2] * rows))
    assert torch.equal(c.read(2, start=at)[0][-1, -1], gk[-1, -1, [n - 1, n - 2]])


def test_attend_refusals(kv):
    c = kv.KVCache(2, 2, 64, 64, "int8")
    q, s = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, device="cuda"), i32([0, 0])
    z = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    for bad in (lambda: c.attend(q.float(), s), lambda: c.attend(q[:, :, :3], s), lambda: c.attend(q, s[:1]),
                lambda: c.attend(q, s.long()), lambda: c.attend(q, s, tree=z.int()), lambda: c.attend(q, s, tree=z[:, :2]),
                lambda: c.attend(q, s, mask=torch.ones(2, 63, dtype=torch.uint8, device="cuda")),
                lambda: c.attend(q, s, mask=torch.ones(2, 64, device="cuda")), lambda: c.attend(q, s, scale=-1.0),
                lambda: c.attend(q, s, out=q[:1]), lambda: c.attend(q.transpose(1, 2), s), lambda: c.attend(q, s.cpu()),
                lambda: c.attend(torch.zeros(3, 1, 4, 64, dtype=torch.bfloat16, device="cuda"), i32([0, 0, 0])),
                lambda: c.attend(q, s, counts=s.long()), lambda: kv.KVCache(1, 1, 64, 48), lambda: kv.KVCache(1, 1, 64, 64, "fp4"),
                lambda: c.write(q[:, :, :2].float(), q[:, :, :2], s), lambda: c.write(q, q, s), lambda: c.read(-1),
                lambda: c.read(1, rows=3), lambda: c.compact(s, i32([0, 1]), s),
                lambda: c.append(q.flatten(2), s, 4), lambda: c.append(torch.zeros(2, 1, 512, dtype=torch.bfloat16, device="cuda"),
                                                                     s, 4, rope=kv.Rope(32))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        c.attend(torch.zeros(1, 65, 4, 64, dtype=torch.bfloat16, device="cuda"), s[:1],
                 tree=torch.zeros(1, 65, dtype=torch.int64, device="cuda"))
    assert c.attend(q[:, :0], s).shape == (2, 0, 4, 64)


# ---- the operators together ------------------------------------------------------------------------

def test_engine_layout(kv):
    """the bf16 cache is the engine's: a prompt appended here, the next token decoded by the engine's own
    fused decode attention, and the same token attended here"""
    import ctypes
    from moss_tts_amd import _native as N
    g = torch.Generator().manual_seed(5)
    H, Hkv, D, slots, n = 8, 2, 128, 256, 77
    W = (H + 2 * Hkv) * D
    qkv = rnd(g, 1, n + 1, W).cuda()
    qn, kn = (0.5 + torch.rand(2, D, generator=g)).to(torch.bfloat16).cuda()
    r = kv.Rope(D, theta=1e4)
    c = fresh(kv, 1, Hkv, slots, D, "bf16", fill=0)
    c.append(qkv[:, :n], i32([0]), H, rope=r, q_norm=qn, k_norm=kn)
    cs, sn = (torch.empty(slots, D, dtype=torch.bfloat16) for _ in range(2))
    N.call("mtts_rope_table", ctypes.c_float(1e4), D, slots, cs.data_ptr(), sn.data_ptr())
    cs, sn = cs.cuda(), sn.cuda()
    mask = torch.ones(1, slots, dtype=torch.uint8, device="cuda")
    ws = torch.zeros(N.load().mtts_k_attn_decode_ws_bytes(1, H, Hkv, D, slots), dtype=torch.uint8, device="cuda")
    out = torch.empty(1, H * D, dtype=torch.bfloat16, device="cuda")
    k2, v2 = c.k.clone(), c.v.clone()
    pos = i32([n])
    N.call("mtts_k_attn_decode", *(t.data_ptr() for t in (qkv[:, n], qn, kn, cs, sn, k2, v2, mask, pos, out, ws)), 1, H, Hkv, D,
           slots, 1e-6, None)
    q = c.append(qkv[:, n:], i32([n]), H, rope=r, q_norm=qn, k_norm=kn)
    got = c.attend(q, i32([n])).view(1, -1).float()
    # the engine rounds its table, its norm and its rotation to bf16, five roundings of q and of k, each BF:
    # scores off by up to 10 BF of sum |q||k| / sqrt(D) (under 12 here), so p by that share, and V exact
    assert torch.equal(v2, c.v)
    rel = ((got - out.float()).norm() / out.float().norm()).item()
    assert rel < 0.05, rel  # (independent roundings: far under the bound of 10 BF * 12)


@pytest.mark.parametrize("kind", KINDS)
def test_a_run_of_steps(kv, kind):
    """a prompt in pieces, a drafted tree, its accepted path compacted, then a next token: equal to a 64-bit
    attention over what the cache holds, and the compacted cache holds what a plain chain would"""
    from tests.kv_layout import contents
    g = torch.Generator().manual_seed(12)
    B, H, Hkv, D = 2, 8, 2, 64
    r = kv.Rope(D, theta=1e5, scaling=YARN)
    W = (H + 2 * Hkv) * D
    lens, S = [90, 41], 48
    c, plain = (kv.KVCache(B, Hkv, 192, D, kind) for _ in range(2))
    prompt = rnd(g, B, 96, W).cuda()
    start = i32([0, 0])
    for lo in (0, S):  # two pieces of a padded batch
        counts = i32([max(0, min(S, n - lo)) for n in lens])
        q = c.append(prompt[:, lo:lo + S].contiguous(), start, H, rope=r, counts=counts)
        out = c.attend(q, start, counts=counts)
        plain.append(prompt[:, lo:lo + S].contiguous(), start, H, rope=r, counts=counts)
        k, v = contents(c)
        see = sees(B, S, 192, start.tolist(), counts.tolist(), None, None)
        attention_close(out.cpu(), *attend64(q.cpu(), k, v, see, D ** -0.5), D)
        start = start + counts
    assert start.tolist() == lens
    parents = [[-1, 0, 0, 2, 1, 3, 3], [-1, 0, 1, 0, 3, 4, 5]]
    tree, depth = kv.tree_masks(parents)
    draft = rnd(g, B, 7, W).cuda()
    pos = (start[:, None] + depth.cuda()).contiguous()
    q = c.append(draft, start, H, rope=r, positions=pos)
    out = c.attend(q, start, tree=tree.cuda())
    k, v = contents(c)
    see = sees(B, 7, 192, lens, None, [[x for x in row] for row in tree.tolist()], None)
    attention_close(out.cpu(), *attend64(q.cpu(), k, v, see, D ** -0.5), D)
    paths, took = [[0, 2, 3, 6], [0, 3, 4, 0]], [4, 3]
    c.compact(start, i32(paths), i32(took))
    for b in range(B):  # the same tokens, one after the other
        idx = torch.tensor(paths[b][:took[b]], device="cuda")
        st = start.clone()
        st[1 - b] = 192  # (the other row's have no slot)
        plain.append(draft[:, idx].contiguous() if b == 0 else draft[:, idx].contiguous(), st, H, rope=r,
                     positions=(st[:, None] + torch.arange(took[b], dtype=torch.int32, device="cuda")).contiguous())
    start = start + i32(took)
    for x, y in zip(c.read(96), plain.read(96)):
        for b in range(B):
            assert torch.equal(x[b, :, :int(start[b])], y[b, :, :int(start[b])])
    q = c.append(rnd(g, B, 1, W).cuda(), start, H, rope=r)
    out = c.attend(q, start)
    k, v = contents(c)
    attention_close(out.cpu(), *attend64(q.cpu(), k, v, sees(B, 1, 192, start.tolist(), None, None, None), D ** -0.5), D)


def test_streams_and_graphs(kv):
    """another stream, and two captured steps that replay with eager work between, against eager results"""
    g = torch.Generator().manual_seed(13)
    B, H, Hkv, D, slots = 2, 8, 2, 128, 4096
    W = (H + 2 * Hkv) * D
    r = kv.Rope(D)
    k, v = rnd(g, B, slots, Hkv, D).cuda(), rnd(g, B, slots, Hkv, D).cuda()
    tree, depth = kv.tree_masks([[-1, 0, 0, 1]] * B)
    tree, depth = tree.cuda(), depth.cuda()

    def step(c, qkv, start):
        q = c.append(qkv, start, H, rope=r, positions=(start[:, None] + depth).contiguous())
        out = c.attend(q, start, tree=tree)
        c.compact(start, path, took)
        return out, *c.read(4, start=start)
    path, took = i32([[0, 2, 0, 0]] * B), i32([2] * B)

    def new():
        c = kv.KVCache(B, Hkv, slots, D, "int8")
        c.write(k, v, i32([0] * B))
        return c
    inputs = [(rnd(g, B, 4, W).cuda(), i32([s, s // 3])) for s in (100, 1111, 3999, 5)]
    eager = [[x.clone() for x in step(new(), *x)] for x in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = new()
        got = step(c, *inputs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, eager[1]))
    graphs = []
    for _ in range(2):
        c, qkv, start = new(), inputs[0][0].clone(), inputs[0][1].clone()
        step(c, qkv, start)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step(c, qkv, start)
        graphs.append((gr, c, qkv, start, outs))
    for n in range(3):
        for i, (qkv_i, start_i) in enumerate(inputs):
            gr, c, qkv, start, outs = graphs[(n + i) % 2]
            c.write(k, v, i32([0] * B))
            qkv.copy_(qkv_i)
            start.copy_(start_i)
            gr.replay()
            eager_now = step(new(), qkv_i, start_i)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager[i]))
            assert all(torch.equal(a, b) for a, b in zip(eager_now, eager[i]))
