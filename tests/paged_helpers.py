"""Inputs and 64-bit references of the serving-step operator tests (torch, on the GPU)."""
import math

import torch

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
UNIT = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}  # half a unit in the last place of 1


def tables(n_pos, rot, dev="cuda"):
    half = rot // 2
    a = torch.arange(n_pos, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(half, device=dev, dtype=torch.float64) / half)[None]
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def rotate64(x, pos, cos, sin, axis, interleaved, inverse=False):
    """(rotated, |a| + |b| of each value's pair), both in 64 bits; pos [axes, tokens], axis [half] or None."""
    x = x.double()
    half = cos.shape[1]
    rot = 2 * half
    ax = torch.zeros(half, dtype=torch.long, device=x.device) if axis is None else axis.long()
    p = pos.long()[ax].T
    at = torch.arange(half, device=x.device)
    c, s = cos[p, at].double()[:, None], sin[p, at].double()[:, None]
    if inverse:
        s = -s
    u = torch.arange(0, rot, 2, device=x.device) if interleaved else torch.arange(half, device=x.device)
    v = u + 1 if interleaved else u + half
    a, b = x[..., u], x[..., v]
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., u], y[..., v] = a * c - b * s, b * c + a * s
    mag[..., u] = mag[..., v] = a.abs() + b.abs()
    return y, mag


def assert_rotated(got, x, pos, cos, sin, axis, interleaved, dtype, inverse=False):
    """Two FP32 products and a sum (each within 2^-24 of its own size, so 2^-22 (|a| + |b|) covers them), then
    one rounding to the type (FP16: subnormal results within 2^-25); values past the rotation are copied."""
    want, mag = rotate64(x, pos, cos, sin, axis, interleaved, inverse)
    tol = UNIT[dtype] * want.abs() + (1 + UNIT[dtype]) * 2.0 ** -22 * mag + (2.0 ** -25 if dtype == "fp16" else 2.0 ** -134)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} values off, worst {float((err - tol).max()):.3e} over the bound"
    rot = 2 * cos.shape[1]
    assert torch.equal(got[..., rot:], x[..., rot:])


class Paged:
    """A batch with a shared prefix and ragged tails in pages whose unused places hold NaN, infinities and the
    type's lowest value."""

    def __init__(self, batch, hq, hkv, dim, prefix, lens, page, layout="nhd", dtype="bf16", seed=0, paged_prefix=True,
                 q_scale=1.2):
        dev = "cuda"
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        dt = TYPES[dtype]
        self.dtype, self.page, self.prefix_len = dtype, page, prefix
        self.lens_host = list(lens)
        self.max_len = max(lens) if lens else 0
        n_table = max(1, -(-self.max_len // page))
        n_prefix = -(-prefix // page) if paged_prefix else 0
        n_pages = n_prefix + batch * n_table + 3
        perm = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
        self.prefix_table = perm[:n_prefix].contiguous()
        self.table = perm[n_prefix:n_prefix + batch * n_table].reshape(batch, n_table).contiguous()
        self.lens = torch.tensor(self.lens_host, dtype=torch.int32, device=dev)
        bad = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dt).min], device=dev, dtype=dt)
        shape = (n_pages, hkv, page, dim) if layout == "hnd" else (n_pages, page, hkv, dim)

        def pool():
            x = bad[torch.randint(0, 4, shape, generator=g, device=dev)]
            return x.transpose(1, 2) if layout == "hnd" else x

        self.k_pool, self.v_pool = pool(), pool()
        scale = torch.exp2(torch.randint(-2, 3, (1, hkv, dim), generator=g, device=dev).float() / 2)

        def values(n):
            return ((torch.randn((n, hkv, dim), generator=g, device=dev) * scale).to(dt),
                    torch.randn((n, hkv, dim), generator=g, device=dev).to(dt))

        self.prefix = values(prefix)
        if paged_prefix:
            self._store(self.prefix_table, *self.prefix)
        self.tails = [values(n) for n in lens]
        for b, (k, v) in enumerate(self.tails):
            self._store(self.table[b], k, v)
        # queries are a strided view of a wider tensor, as behind a fused projection
        self.q = (torch.randn((batch, hq + 2 * hkv, dim), generator=g, device=dev) * q_scale).to(dt)[:, :hq]
        self.scale = dim ** -0.5

    def _store(self, table, k, v):
        t = torch.arange(k.shape[0], device=k.device)
        page = table.long()[t // self.page]
        self.k_pool[page, t % self.page], self.v_pool[page, t % self.page] = k, v

    def truth(self, scale=None):
        """(out, lse, tolerance of out, tolerance of lse) in 64 bits."""
        return attention64(self.q, [(torch.cat([self.prefix[0], k]), torch.cat([self.prefix[1], v])) for k, v in self.tails],
                           self.scale if scale is None else scale, self.dtype)


def attention64(q, kv, scale, dtype):
    """Attention of q [batch, hq, dim] over kv[b] = (K, V) [tokens, hkv, dim], and how far an FP32 evaluation whose
    softmax weights and output are rounded to the type may be off.

    With w the weights, u the type's unit: the output's rounding u |out|; the weights' rounding u sum w |v|; a score is a
    dim-term FP32 sum, off by at most (dim + 2) 2^-23 scale sum |q k| =: e (tensor-core sums may truncate: 2^-23 a
    term), which moves weights by a factor of 1 + 2 e after normalising; 2^x by the SFU, the sums over n tokens and the
    folds of partial states n 2^-23 + 2^-18 together."""
    q = q.double()
    batch, hq, dim = q.shape
    out = torch.zeros_like(q)
    lse = torch.full((batch, hq), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.full_like(out, 1e-30), torch.full_like(lse, 1e-30)
    u = UNIT[dtype]
    for b, (k, v) in enumerate(kv):
        if k.shape[0] == 0:
            continue
        k, v = k.double(), v.double()
        g = hq // k.shape[1]
        kh, vh = k.repeat_interleave(g, 1).transpose(0, 1), v.repeat_interleave(g, 1).transpose(0, 1)
        s = (kh @ q[b][:, :, None])[..., 0] * scale
        e = (dim + 2) * 2.0 ** -23 * scale * (kh.abs() @ q[b].abs()[:, :, None])[..., 0].amax(1)
        w = torch.softmax(s, 1)
        out[b] = (w[:, None] @ vh)[:, 0]
        lse[b] = torch.logsumexp(s, 1)
        mass = (w[:, None] @ vh.abs())[:, 0]
        acc = k.shape[0] * 2.0 ** -23 + 2.0 ** -18
        tol[b] = u * out[b].abs() + (1 + u) * (u + 2 * e + acc)[:, None] * mass + (2.0 ** -24 if dtype == "fp16" else 1e-30)
        tol_lse[b] = e + acc + 2.0 ** -22 * (1 + lse[b].abs() + s.abs().amax(1))
    return out, lse, tol, tol_lse


def assert_attends(out, lse, truth):
    want, want_lse, tol, tol_lse = truth
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), (
        f"{int((~(err <= tol)).sum())} of {err.numel()} outputs off; worst error {float(err.max()):.3e}, "
        f"over its bound by {float((err - tol).max()):.3e}")
    if lse is not None:
        empty = want_lse == -math.inf
        assert torch.equal(lse.double() == -math.inf, empty)
        d = (lse.double() - want_lse)[~empty].abs()
        assert bool((d <= tol_lse[~empty]).all()), f"lse off by {float(d.max()):.3e}"
