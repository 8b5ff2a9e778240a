"""The 8-bit cache's 32-slot tiles, restated from their definition (csrc/kvq.h), and a cache's contents
as 64-bit values [rows, n_kv, slots, D]."""
import numpy as np
import torch


def k_bytes(D):
    """[32, D]: the byte of (slot, dim) in a K tile"""
    s, d = np.arange(32)[:, None], np.arange(D)[None]
    u, h, i = s // 16, s // 8 % 2, s % 8
    return (d // 16 * 32 + 16 * u + 8 * (i // 4) + 4 * h + i % 4) * 16 + d % 16


def v_bytes(D):
    s, d = np.arange(32)[:, None], np.arange(D)[None]
    u, h, i = s // 16, s // 8 % 2, s % 8
    return (d // 32 * 64 + 32 * h + d % 32) * 16 + 8 * u + i


def codes(c):
    """(k, v) as the values of their codes, [rows, n_kv, slots, D]"""
    out = []
    for buf, at in ((c.k, k_bytes(c.head_dim)), (c.v, v_bytes(c.head_dim))):
        t = buf.cpu().view(c.rows, c.n_kv, c.slots // 32, 32 * c.head_dim)[..., torch.from_numpy(at)]
        t = t.view(torch.float8_e4m3fn if c.dtype == "e4m3" else torch.int8)
        out.append(t.double().view(c.rows, c.n_kv, c.slots, c.head_dim))
    return out


def contents(c):
    if c.dtype == "bf16":
        return c.k.cpu().double(), c.v.cpu().double().transpose(2, 3)
    k, v = codes(c)
    return k * c.k_scale.cpu().double()[..., None], v * c.v_scale.cpu().double()[..., None]
