"""GPU tests of the serving-step operators (kvx_batch_*): position rotation, append to a paged cache and attention
over a shared prefix and paged tails, against 64-bit evaluations of their formulas (paged_helpers)."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def H(cuda):
    import paged_helpers
    return paged_helpers


def _axis(torch, half, n_axes, mixed):
    """Axis of each pair: runs of pairs, or changing from pair to pair."""
    at = torch.arange(half, device="cuda")
    return ((at % n_axes) if mixed else at * n_axes // half).to(torch.uint8)


# ---- rotation -------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,heads,dim,rot,axes,interleaved,dtype", [
    (1, 1, 64, 64, 1, False, "bf16"), (1, 14, 64, 64, 1, False, "bf16"), (3, 2, 32, 32, 1, True, "fp16"),
    (257, 5, 128, 64, 1, False, "bf16"), (1000, 3, 128, 96, 1, True, "bf16"), (77, 7, 256, 256, 3, False, "fp16"),
    (130, 2, 64, 64, 3, True, "bf16"), (33, 4, 32, 24, 2, False, "bf16"),   # 24: not whole 16-value pieces
    (19, 3, 80, 80, 3, False, "fp16"), (5, 3, 6, 2, 1, False, "bf16"),
])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotate(kvx, cuda, H, tokens, heads, dim, rot, axes, interleaved, dtype, inverse):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens * 7 + dim)
    cos, sin = H.tables(300, rot)
    x = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(H.TYPES[dtype])
    pos = torch.randint(0, 300, (axes, tokens), generator=g, device="cuda").to(torch.int32)
    for mixed in ([False, True] if axes > 1 else [False]):
        axis = _axis(torch, rot // 2, axes, mixed) if axes > 1 else None
        b = kvx.Batch(1, heads, heads, dim, dtype=dtype)
        rope = kvx.Rope(cos, sin, axis=axis, n_axes=axes, interleaved=interleaved)
        out = torch.full_like(x, 7.0)
        b.rotate(x, pos, rope, out, inverse=inverse)
        b.check()
        H.assert_rotated(out, x, pos, cos, sin, axis, interleaved, dtype, inverse)
        y = x.clone()
        b.rotate(y, pos, rope, y, inverse=inverse)  # in place
        assert torch.equal(y, out)


@pytest.mark.parametrize("tokens,heads,dim,rot,axes,interleaved,dtype", [
    (4500, 40, 128, 128, 1, False, "bf16"), (9001, 17, 128, 96, 2, True, "fp16"), (2100, 33, 256, 64, 3, False, "bf16"),
    (33000, 3, 224, 192, 1, True, "bf16"), (2500, 300, 32, 32, 1, False, "bf16"),
])
def test_rotate_many(kvx, cuda, H, tokens, heads, dim, rot, axes, interleaved, dtype):
    """Over a million pieces: the kernel that turns several heads a thread."""
    test_rotate(kvx, cuda, H, tokens, heads, dim, rot, axes, interleaved, dtype, False)


@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (8, 8), (0, 1), (0, 4)])
def test_rotate_strides_and_alignment(kvx, cuda, H, offset, pad):
    """Rows anywhere: odd starts and odd strides take the general kernel, with the same values."""
    torch = cuda
    tokens, heads, dim = 37, 3, 64
    cos, sin = H.tables(64, dim)
    base = torch.randn(tokens * (heads * (dim + pad) + 5 * pad) + 64, device="cuda").to(torch.bfloat16)
    x = torch.as_strided(base, (tokens, heads, dim), (heads * (dim + pad) + 5 * pad, dim + pad, 1), offset)
    y = torch.zeros_like(base)
    out = torch.as_strided(y, x.shape, x.stride(), offset)
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32)
    b = kvx.Batch(1, heads, heads, dim)
    b.rotate(x, pos, kvx.Rope(cos, sin), out)
    H.assert_rotated(out, x, pos[None], cos, sin, None, False, "bf16")
    untouched = torch.ones_like(y, dtype=torch.bool)
    torch.as_strided(untouched, x.shape, x.stride(), offset).fill_(False)
    assert not bool(y[untouched].any())


def test_rotate_gradient(kvx, cuda, H):
    """The opposite rotation of an upstream gradient is the gradient: against the formula's, and against central
    differences of a loss of the kernel's own outputs (their rounding, at most u |out| a value, over the step)."""
    torch = cuda
    tokens, heads, dim = 4, 2, 32
    g = torch.Generator(device="cuda").manual_seed(5)
    cos, sin = H.tables(50, dim)
    pos = torch.randint(0, 50, (tokens,), generator=g, device="cuda").to(torch.int32)
    x = torch.randn((tokens, heads, dim), generator=g, device="cuda").half()
    w = torch.randn((tokens, heads, dim), generator=g, device="cuda").half()
    b, rope = kvx.Batch(1, heads, heads, dim, dtype="fp16"), kvx.Rope(cos, sin)
    grad = torch.empty_like(w)
    b.rotate(w, pos, rope, grad, inverse=True)
    xd = x.double().requires_grad_()
    (H.rotate64(xd, pos[None], cos, sin, None, False)[0] * w.double()).sum().backward()
    assert bool(((grad.double() - xd.grad).abs() <= 2.0 ** -11 * xd.grad.abs() + 2.0 ** -20 + 2.0 ** -25).all())

    def loss(v):
        o = torch.empty_like(v)
        b.rotate(v, pos, rope, o)
        return float((o.double() * w.double()).sum()), o

    step = 0.5
    for t, h, d in [(0, 0, 0), (1, 1, 5), (3, 0, 16), (2, 1, 31)]:
        up, dn = x.clone(), x.clone()
        up[t, h, d] += step
        dn[t, h, d] -= step
        (a, oa), (c, oc) = loss(up), loss(dn)
        slack = float(((oa.double().abs() + oc.double().abs()) * w.double().abs())[t, h].sum()) * 2.0 ** -11
        moved = float(up[t, h, d].double() - dn[t, h, d].double())
        assert abs((a - c) / moved - float(grad[t, h, d])) <= slack / moved + 2.0 ** -10 * abs(float(grad[t, h, d])) + 1e-5


# ---- append -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,axes,page,layout,dtype", [
    (1, 14, 2, 64, 64, 1, 16, "nhd", "bf16"), (1, 1, 1, 32, 32, 1, 1, "hnd", "fp16"),
    (300, 8, 2, 128, 128, 1, 16, "hnd", "bf16"), (123, 6, 3, 64, 32, 3, 48, "nhd", "fp16"),
    (61, 4, 4, 256, 256, 1, 7, "nhd", "bf16"), (40, 3, 1, 32, 24, 2, 5, "hnd", "bf16"),
    (9, 2, 2, 64, 0, 1, 16, "nhd", "bf16"),
    (4097, 32, 4, 128, 64, 1, 16, "hnd", "bf16"), (9000, 9, 9, 128, 128, 1, 48, "nhd", "fp16"),  # over a million pieces
])
def test_append(kvx, cuda, H, tokens, hq, hkv, dim, rot, axes, page, layout, dtype):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    dt = H.TYPES[dtype]
    n_pages = -(-tokens // page) + 4
    shape = (n_pages, hkv, page, dim) if layout == "hnd" else (n_pages, page, hkv, dim)
    kp, vp = (torch.randn(shape, generator=g, device="cuda").to(dt) for _ in range(2))
    if layout == "hnd":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    k0, v0 = kp.clone(), vp.clone()
    qkv = torch.randn((tokens, hq + 2 * hkv, dim), generator=g, device="cuda").to(dt)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:tokens].to(torch.int64)
    if tokens > 3:
        slots[2], slots[-1] = -1, -(1 << 40)  # padding tokens
    out = torch.empty((tokens, hq, dim), device="cuda", dtype=dt)
    b = kvx.Batch(1, hq, hkv, dim, dtype=dtype)
    if rot:
        cos, sin = H.tables(200, rot)
        pos = torch.randint(0, 200, (axes, tokens), generator=g, device="cuda").to(torch.int32)
        axis = _axis(torch, rot // 2, axes, False) if axes > 1 else None
        rope = kvx.Rope(cos, sin, axis=axis, n_axes=axes)
    else:
        pos = rope = None
    b.append(q, k, v, pos, rope, slots, kvx.Pages(kp, vp), out)
    b.check()
    keep = slots >= 0
    at = (slots[keep] // page, slots[keep] % page)
    if rot:
        H.assert_rotated(out, q, pos, cos, sin, axis, False, dtype)
        H.assert_rotated(kp[at], k[keep], pos[:, keep], cos, sin, axis, False, dtype)
    else:
        assert torch.equal(out, q) and torch.equal(kp[at], k[keep])
    assert torch.equal(vp[at], v[keep])
    k0[at], v0[at] = kp[at], vp[at]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)  # nothing else was written
    # without queries
    k1, v1 = kp.clone(), vp.clone()
    kp[at], vp[at] = 0, 0
    b.append(None, k, v, pos, rope, slots, kvx.Pages(kp, vp), None)
    assert torch.equal(kp, k1) and torch.equal(vp, v1)


@pytest.mark.parametrize("tokens,hkv,dim,rot", [(1, 2, 64, 64), (300, 2, 128, 64), (9000, 16, 128, 128), (40, 1, 32, 24)])
def test_padding_tokens_have_no_position(kvx, cuda, H, tokens, hkv, dim, rot):
    """A padding token's position is a filler: in an append without queries it is not looked at, however many tokens the
    call has (9000 of 2 x 16 heads of 128 are over a million pieces); where a query is rotated by it, it is reported."""
    torch = cuda
    cos, sin = H.tables(50, rot)
    rope = kvx.Rope(cos, sin)
    k, v = (torch.randn((tokens, hkv, dim), device="cuda").to(torch.bfloat16) for _ in range(2))
    kp, vp = (torch.zeros((tokens, 1, hkv, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    pad = torch.arange(tokens, device="cuda") % 3 == 0
    slots = torch.where(pad, -1, torch.arange(tokens, device="cuda"))
    pos = torch.where(pad, -1, torch.arange(tokens, device="cuda") % 50).to(torch.int32)
    b = kvx.Batch(1, hkv, hkv, dim)
    b.append(None, k, v, pos, rope, slots, kvx.Pages(kp, vp), None)
    b.check()
    H.assert_rotated(kp[~pad, 0], k[~pad], pos[None, ~pad], cos, sin, None, False, "bf16")
    assert torch.equal(vp[~pad, 0], v[~pad]) and not bool(kp[pad].any()) and not bool(vp[pad].any())
    b.append(k, k, v, pos, rope, slots, kvx.Pages(kp, vp), torch.empty_like(k))
    with pytest.raises(RuntimeError, match="position outside the rotation tables"):
        b.check()


def test_append_past_32_bits(kvx, cuda, H):
    """Elements whose offset in the pool passes 2^32."""
    torch = cuda
    page, hkv, dim = 128, 8, 256
    n_pages = (1 << 32) // (page * hkv * dim) + 40
    kp = torch.zeros((n_pages, page, hkv, dim), device="cuda", dtype=torch.bfloat16)
    vp = torch.zeros_like(kp)
    k = torch.randn((3, hkv, dim), device="cuda").to(torch.bfloat16)
    slots = torch.tensor([(n_pages - 1) * page + 127, 5, (n_pages - 3) * page], device="cuda")
    b = kvx.Batch(2, 8, 8, dim)
    pages = kvx.Pages(kp, vp)
    b.append(None, k, k, None, None, slots, pages, None)
    b.check()
    at = (slots // page, slots % page)
    assert torch.equal(kp[at], k) and torch.equal(vp[at], k)
    assert int(torch.count_nonzero(kp[:, :, 0, 0])) == int(torch.count_nonzero(k[:, 0, 0]))
    # and attention reads them: one token of each sequence, so out is its V
    table = torch.tensor([[n_pages - 3], [n_pages - 1]], dtype=torch.int32, device="cuda")
    vp[n_pages - 1, 0], kp[n_pages - 1, 0] = k[1], k[1]
    q = torch.randn((2, 8, dim), device="cuda").to(torch.bfloat16)
    out = torch.empty_like(q)
    b.attend(q, out, pages, table, torch.ones(2, dtype=torch.int32, device="cuda"), 1)
    b.check()
    assert torch.equal(out[0], k[2]) and torch.equal(out[1], k[1])


# ---- attention --------------------------------------------------------------------------------------

def _attend(kvx, torch, H, c, hq, hkv, dim, **kw):
    b = kvx.Batch(len(c.lens_host), hq, hkv, dim, dtype=c.dtype)
    out = torch.full((len(c.lens_host), hq, dim), 7.0, device="cuda", dtype=c.q.dtype)
    lse = torch.full((len(c.lens_host), hq), 7.0, device="cuda")
    b.attend(c.q, out, kvx.Pages(c.k_pool, c.v_pool), c.table, c.lens, c.max_len, prefix_table=c.prefix_table,
             prefix_len=c.prefix_len, lse=lse, **kw)
    b.check()
    return out, lse


CASES = [
    # hq, hkv, dim, prefix, lens, page, layout, dtype
    (1, 1, 64, 1, [0], 16, "nhd", "bf16"),
    (1, 1, 32, 0, [1], 16, "nhd", "bf16"),
    (2, 1, 64, 0, [0, 3], 16, "nhd", "bf16"),              # a row with nothing at all
    (14, 2, 64, 300, [17, 0], 16, "nhd", "bf16"),
    (14, 2, 64, 129, [64, 1, 0, 33, 128, 5, 250, 16, 15], 16, "hnd", "bf16"),
    (32, 8, 128, 1000, [100, 0, 257], 64, "nhd", "bf16"),
    (8, 8, 128, 63, [64, 65], 32, "hnd", "fp16"),
    (20, 2, 128, 500, [40] * 13, 48, "nhd", "bf16"),       # 10 heads a group, 130 rows
    (16, 1, 64, 777, [9] * 17, 7, "nhd", "fp16"),          # 272 rows, odd pages
    (4, 4, 256, 200, [0, 300], 128, "nhd", "bf16"),
    (12, 3, 256, 321, [31] * 7, 16, "hnd", "fp16"),
    (5, 5, 32, 450, [12, 700], 1, "nhd", "bf16"),          # one token a page
    (9, 3, 32, 64, [2] * 50, 16, "nhd", "fp16"),
    (28, 4, 128, 4100, [1500, 2, 0, 0, 900], 16, "nhd", "bf16"),
    (64, 1, 64, 2000, [600] * 5, 16, "nhd", "bf16"),       # one KV head for 64
    (2, 2, 64, 20000, [0], 128, "nhd", "bf16"),
]


@pytest.mark.parametrize("hq,hkv,dim,prefix,lens,page,layout,dtype", CASES)
def test_attend(kvx, cuda, H, hq, hkv, dim, prefix, lens, page, layout, dtype):
    c = H.Paged(len(lens), hq, hkv, dim, prefix, lens, page, layout, dtype, seed=hq + dim + prefix)
    out, lse = _attend(kvx, cuda, H, c, hq, hkv, dim)
    H.assert_attends(out, lse, c.truth())
    again, _ = _attend(kvx, cuda, H, c, hq, hkv, dim)
    assert cuda.equal(out.view(cuda.int16), again.view(cuda.int16))  # no order of atomics in it


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 255, 256, 257, 383, 385])
@pytest.mark.parametrize("batch,hq,hkv,dim", [(5, 8, 2, 64), (37, 4, 1, 128)])
def test_attend_prefix_lengths(kvx, cuda, H, prefix, batch, hq, hkv, dim):
    lens = [(prefix + 3 * i) % 23 for i in range(batch)]
    c = H.Paged(batch, hq, hkv, dim, prefix, lens, 16, seed=prefix)
    out, lse = _attend(kvx, cuda, H, c, hq, hkv, dim)
    H.assert_attends(out, lse, c.truth())


@pytest.mark.parametrize("batch,hq,hkv,dim,dtype", [(7, 32, 8, 128, "fp16"), (9, 2, 2, 64, "bf16"), (40, 4, 1, 32, "bf16"),
                                                    (3, 16, 4, 256, "bf16")])
def test_attend_long_prefix_again_and_again(kvx, cuda, H, batch, hq, hkv, dim, dtype):
    """Many tiles an item and warps with no rows of their own: every run is the same, and no wait runs out."""
    torch = cuda
    c = H.Paged(batch, hq, hkv, dim, 40000, [5] * batch, 48, "hnd", dtype)
    b, pages = kvx.Batch(batch, hq, hkv, dim, dtype=dtype), kvx.Pages(c.k_pool, c.v_pool)
    outs = [torch.empty((batch, hq, dim), device="cuda", dtype=c.q.dtype) for _ in range(2)]
    for i in range(60):
        b.attend(c.q, outs[i % 2], pages, c.table, c.lens, 5, prefix_table=c.prefix_table, prefix_len=40000)
    b.check()
    assert torch.equal(outs[0], outs[1])
    H.assert_attends(outs[0], None, c.truth())


@pytest.mark.parametrize("dim,dtype", [(32, "fp16"), (64, "bf16"), (128, "bf16"), (256, "bf16")])
def test_attend_peaked_and_rising_scores(kvx, cuda, H, dim, dtype):
    """Scores that rise along the prefix (every tile raises the maximum) and differ by hundreds."""
    torch = cuda
    c = H.Paged(9, 4, 1, dim, 700, [30] * 9, 16, dtype=dtype, q_scale=1.0)
    k, v = c.prefix
    k = k * 0.1
    k[:, :, 0] = (torch.arange(700, device="cuda") / 2.0).to(k.dtype)[:, None]
    c.prefix = (k, v)
    c._store(c.prefix_table, k, v)
    c.q = c.q.contiguous()
    c.q[:, :, 0] = torch.linspace(-3, 3, 36, device="cuda").reshape(9, 4).to(c.q.dtype)
    out, lse = _attend(kvx, cuda, H, c, 4, 1, dim, scale=0.9)
    H.assert_attends(out, lse, c.truth(scale=0.9))


def test_attend_prefix_is_the_sum_of_its_parts(kvx, cuda, H):
    """The same tokens as a prefix, or as tails of their own, give the same attention (within both bounds)."""
    torch = cuda
    c = H.Paged(20, 8, 2, 64, 500, [0] * 20, 16)
    out, _ = _attend(kvx, cuda, H, c, 8, 2, 64)
    b = kvx.Batch(20, 8, 2, 64)
    own = torch.empty_like(out)
    table = c.prefix_table[None].expand(20, -1).contiguous()
    b.attend(c.q, own, kvx.Pages(c.k_pool, c.v_pool), table, torch.full((20,), 500, dtype=torch.int32, device="cuda"), 500)
    want, _, tol, _ = c.truth()
    assert bool(((own.double() - want).abs() <= tol).all())
    assert bool(((own.double() - out.double()).abs() <= 2 * tol).all())


def test_attend_special_values(kvx, cuda, H):
    """A NaN or an infinity among the attended values reaches the rows that see it, and no others."""
    torch = cuda
    c = H.Paged(3, 4, 2, 64, 200, [20, 30, 0], 16)
    k, v = c.tails[1]
    v[5, 0, 3] = math.nan
    k[7, 1, 2] = math.nan
    c._store(c.table[1], k, v)
    out, lse = _attend(kvx, cuda, H, c, 4, 2, 64)
    assert bool(out[1, :2, 3].isnan().all()) and bool(out[1, 2:].isnan().all()) and bool(lse[1, 2:].isnan().all())
    assert bool(out[0].isfinite().all()) and bool(out[2].isfinite().all())
    assert int(out[1, :2].isnan().sum()) == 2


def test_attend_in_a_graph_on_a_stream(kvx, cuda, H):
    """Captured once with its append, replayed while the tails grow."""
    torch = cuda
    hq, hkv, dim, page, batch = 8, 2, 64, 16, 12
    c = H.Paged(batch, hq, hkv, dim, 300, [0] * batch, page)
    c.table = torch.arange(batch * 4, device="cuda", dtype=torch.int32).reshape(batch, 4)
    n = batch * 4
    kp = torch.full((n + c.prefix_table.numel(), page, hkv, dim), math.nan, device="cuda", dtype=torch.bfloat16)
    vp = kp.clone()
    c.prefix_table = torch.arange(n, kp.shape[0], device="cuda", dtype=torch.int32)
    c.k_pool, c.v_pool = kp, vp
    c._store(c.prefix_table, *c.prefix)
    b, pages = kvx.Batch(batch, hq, hkv, dim), kvx.Pages(kp, vp)
    new = torch.empty((batch, hq + 2 * hkv, dim), device="cuda", dtype=torch.bfloat16)
    slots = torch.full((batch,), -1, device="cuda", dtype=torch.int64)
    q, out = torch.empty((batch, hq, dim), device="cuda", dtype=torch.bfloat16), torch.empty(
        (batch, hq, dim), device="cuda", dtype=torch.bfloat16)
    lens = torch.zeros(batch, device="cuda", dtype=torch.int32)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()

    def step(stream):
        b.append(new[:, :hq], new[:, hq:hq + hkv], new[:, hq + hkv:], None, None, slots, pages, q, stream=stream)
        b.attend(q, out, pages, c.table, lens, 4 * page, prefix_table=c.prefix_table, prefix_len=300, stream=stream)

    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(s.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        step(s.cuda_stream)
    ks, vs = [], []
    for i in range(3):
        x = torch.randn((batch, hq + 2 * hkv, dim), device="cuda").to(torch.bfloat16)
        new.copy_(x)
        slots.copy_(torch.arange(batch, device="cuda") * 4 * page + i)
        lens.fill_(i + 1)
        graph.replay()
        torch.cuda.synchronize()
        ks.append(x[:, hq:hq + hkv])
        vs.append(x[:, hq + hkv:])
        kv = [(torch.cat([c.prefix[0], torch.stack([k[j] for k in ks])]), torch.cat([c.prefix[1], torch.stack([v[j] for v in vs])]))
              for j in range(batch)]
        H.assert_attends(out, None, H.attention64(x[:, :hq], kv, dim ** -0.5, "bf16"))
    b.check()


@pytest.mark.parametrize("batch,hq,hkv,dim,prefix,longest,page,dtype", [
    (129, 4, 2, 64, 0, 40, 16, "bf16"), (300, 2, 2, 128, 4000, 64, 16, "bf16"), (700, 2, 2, 256, 0, 33, 7, "fp16"),
    (1500, 8, 1, 64, 1000, 20, 16, "fp16"), (2048, 2, 1, 32, 300, 50, 16, "bf16"), (2048, 4, 2, 128, 100, 70, 32, "bf16"),
    (2048, 2, 2, 256, 100, 20, 16, "bf16"),
])
def test_attend_large_batches(kvx, cuda, H, batch, hq, hkv, dim, prefix, longest, page, dtype):
    """More sequences than a CTA has threads, up to the handle's bound; ragged, many of them empty."""
    lens = [(i * 7919) % (longest + 1) if i % 5 else 0 for i in range(batch)]
    lens[3] = longest
    c = H.Paged(batch, hq, hkv, dim, prefix, lens, page, dtype=dtype, seed=batch)
    out, lse = _attend(kvx, cuda, H, c, hq, hkv, dim)
    H.assert_attends(out, lse, c.truth())
    again, _ = _attend(kvx, cuda, H, c, hq, hkv, dim)
    assert cuda.equal(out.view(cuda.int16), again.view(cuda.int16))


@pytest.mark.parametrize("batch,hq,hkv,dim,prefix,page,dtype", [
    (3, 14, 2, 64, 0, 16, "bf16"), (1, 8, 8, 128, 500, 16, "bf16"), (20, 8, 2, 64, 3000, 16, "fp16"), (64, 8, 2, 128, 9000, 64, "bf16"),
    (40, 16, 16, 32, 900, 48, "bf16"), (5, 32, 8, 256, 700, 128, "bf16"),
])
def test_attend_lengths_far_below_max_len(kvx, cuda, H, batch, hq, hkv, dim, prefix, page, dtype):
    """max_len as a capacity: tables with room for 20000 tokens, of which a few are there."""
    torch = cuda
    lens = [(i * 31) % 90 for i in range(batch)]
    c = H.Paged(batch, hq, hkv, dim, prefix, lens, page, dtype=dtype)
    wide = torch.full((batch, -(-20000 // page)), -1, device="cuda", dtype=torch.int32)  # (never looked at)
    wide[:, :c.table.shape[1]] = c.table
    c.table, c.max_len = wide, 20000
    out, lse = _attend(kvx, torch, H, c, hq, hkv, dim)
    H.assert_attends(out, lse, c.truth())


def test_attend_on_two_streams(kvx, cuda, H):
    """Two handles of different shapes on two streams at once, each with its own scratch: the same bits as one after the
    other."""
    torch = cuda
    shapes = [(64, 32, 8, 128, 9000, 300, "bf16"), (20, 14, 2, 64, 5000, 900, "fp16")]
    made = []
    for batch, hq, hkv, dim, prefix, longest, dtype in shapes:
        c = H.Paged(batch, hq, hkv, dim, prefix, [(i * 37) % (longest + 1) for i in range(batch)], 16, dtype=dtype, seed=dim)
        b, pages = kvx.Batch(batch, hq, hkv, dim, dtype=dtype), kvx.Pages(c.k_pool, c.v_pool)

        def call(out, stream, b=b, c=c, pages=pages):
            b.attend(c.q, out, pages, c.table, c.lens, c.max_len, prefix_table=c.prefix_table, prefix_len=c.prefix_len, stream=stream)

        want = torch.empty((batch, hq, dim), device="cuda", dtype=c.q.dtype)
        call(want, None)
        b.check()
        H.assert_attends(want, None, c.truth())
        made.append((b, call, want, [torch.full_like(want, 7.0) for _ in range(40)], torch.cuda.Stream()))
    torch.cuda.synchronize()
    for i in range(40):
        for b, call, want, outs, stream in made:
            call(outs[i], stream.cuda_stream)
    for b, call, want, outs, stream in made:
        b.check()
        assert all(torch.equal(x, want) for x in outs)


# ---- a prefix kept as XKV blobs ---------------------------------------------------------------------

def _modes(torch, seq, heads, dim, block, seed, special=0.01):
    """[heads, seq, dim] BF16 whose blocks favour raw, 2-, 3- and 4-bit residuals in turn, with escapes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    spread = torch.tensor([3, 7, 15, 60], device="cuda")[(torch.arange(seq, device="cuda") // block + seed) % 4]
    e = 126 - (torch.rand((heads, seq, dim), generator=g, device="cuda") * spread[None, :, None]).long()
    far = torch.rand(e.shape, generator=g, device="cuda") < special
    e = torch.where(far, torch.randint(60, 127, e.shape, generator=g, device="cuda"), e)
    bits = (torch.randint(0, 2, e.shape, generator=g, device="cuda") << 15) | (e << 7) | torch.randint(
        0, 128, e.shape, generator=g, device="cuda")
    bits = torch.where(bits >= 32768, bits - 65536, bits).to(torch.int16)
    return bits.view(torch.bfloat16)


@pytest.mark.parametrize("hq,hkv,dim,seq,lens,block,bits", [
    (1, 1, 64, 1, [0], 128, 0x14), (14, 2, 64, 1000, [3, 0, 40], 128, 0x14), (14, 2, 64, 1000, [3, 0, 40], 128, 0x1C),
    (8, 2, 128, 700, [0] * 40, 128, 0x1C), (32, 8, 128, 2111, [100] * 9, 128, 0x14), (6, 3, 32, 999, [70] * 70, 128, 0x1C),
    (4, 2, 256, 515, [17, 0, 5], 128, 0x1C), (8, 4, 64, 777, [9] * 4, 32, 0x1C), (4, 1, 128, 900, [1] * 40, 255, 0x1C),
    (4, 4, 64, 300, [0] * 3, 7, 0x14), (12, 2, 64, 20000, [64] * 12, 128, 0x1C),
])
def test_attend_xkv(kvx, cuda, H, hq, hkv, dim, seq, lens, block, bits):
    torch = cuda
    k, v = _modes(torch, seq, hkv, dim, block, 0), _modes(torch, seq, hkv, dim, block, 1, special=0.1)
    c = H.Paged(len(lens), hq, hkv, dim, 0, lens, 16, paged_prefix=False, q_scale=0.7)
    c.prefix = (k.transpose(0, 1), v.transpose(0, 1))
    prefix = kvx.Prefix.encode(k, v, block_tokens=block, code_bits=bits)
    b, pages = kvx.Batch(len(lens), hq, hkv, dim), kvx.Pages(c.k_pool, c.v_pool)
    out = torch.full((len(lens), hq, dim), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((len(lens), hq), 7.0, device="cuda")
    for _ in range(2):
        b.attend(c.q, out, pages, c.table, c.lens, c.max_len, prefix=prefix, lse=lse)
    b.check()
    H.assert_attends(out, lse, c.truth())


@pytest.mark.parametrize("hq,hkv,dim,seq,batch,bits", [(14, 2, 64, 1000, 3, 0x1C), (8, 2, 128, 700, 40, 0x14),
                                                       (6, 3, 32, 999, 70, 0x1C), (4, 2, 256, 515, 5, 0x1C)])
def test_xkv_prefix_is_the_paged_prefix(kvx, cuda, H, hq, hkv, dim, seq, batch, bits):
    """The same tiles reach the tensor cores as from pages: the same bits where both are cut alike (a tile an item,
    as long as the items are no more than the SMs)."""
    torch = cuda
    k, v = _modes(torch, seq, hkv, dim, 128, 0), _modes(torch, seq, hkv, dim, 128, 1, special=0.1)
    assert -(-seq // 64) * hkv * -(-batch * (hq // hkv) // 128) <= 148
    c = H.Paged(batch, hq, hkv, dim, seq, [0] * batch, 16, q_scale=0.7)
    c.prefix = (k.transpose(0, 1), v.transpose(0, 1))
    c._store(c.prefix_table, *c.prefix)
    b, pages = kvx.Batch(batch, hq, hkv, dim), kvx.Pages(c.k_pool, c.v_pool)
    out, same = (torch.empty((batch, hq, dim), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    b.attend(c.q, out, pages, None, None, 0, prefix=kvx.Prefix.encode(k, v, code_bits=bits))
    b.attend(c.q, same, pages, None, None, 0, prefix_table=c.prefix_table, prefix_len=seq)
    b.check()
    assert torch.equal(out, same)


def test_xkv_prefix_special_values(kvx, cuda, H):
    """Every BF16 class goes through the decoder: V columns of zeros, subnormals and a NaN or infinity."""
    torch = cuda
    k, v = _modes(torch, 200, 1, 64, 128, 2), _modes(torch, 200, 1, 64, 128, 3)
    v[0, :, 0], v[0, :, 1], v[0, 150, 2], v[0, 20, 3] = 0.0, 1e-40, math.nan, math.inf
    c = H.Paged(10, 1, 1, 64, 0, [0] * 10, 16, paged_prefix=False)
    out = torch.empty((10, 1, 64), device="cuda", dtype=torch.bfloat16)
    b = kvx.Batch(10, 1, 1, 64)
    b.attend(c.q, out, kvx.Pages(c.k_pool, c.v_pool), None, None, 0, prefix=kvx.Prefix.encode(k, v))
    b.check()
    assert bool((out[..., 0] == 0).all()) and bool(out[..., 2].isnan().all()) and bool((out[..., 3] == math.inf).all())
    assert bool((out[..., 1].abs() < 1e-38).all()) and bool(out[..., 4:].isfinite().all())


def test_xkv_prefix_refusals(kvx, cuda, H):
    torch = cuda
    k = _modes(torch, 300, 2, 64, 128, 0)
    p = kvx.Prefix.encode(k, k)
    c = H.Paged(2, 4, 2, 64, 16, [4, 4], 16)
    pages, out = kvx.Pages(c.k_pool, c.v_pool), torch.empty((2, 4, 64), device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="one prefix"):
        kvx.Batch(2, 4, 2, 64).attend(c.q, out, pages, c.table, c.lens, 4, prefix=p, prefix_table=c.prefix_table, prefix_len=16)
    one = H.Paged(2, 4, 1, 64, 16, [4, 4], 16)
    with pytest.raises(ValueError, match="other heads"):
        kvx.Batch(2, 4, 1, 64).attend(one.q, out, kvx.Pages(one.k_pool, one.v_pool), one.table, one.lens, 4, prefix=p)
    half = H.Paged(2, 4, 2, 64, 16, [4, 4], 16, dtype="fp16")
    with pytest.raises(ValueError, match="BF16"):
        kvx.Batch(2, 4, 2, 64, dtype="fp16").attend(half.q, out.half(), kvx.Pages(half.k_pool, half.v_pool), half.table,
                                                    half.lens, 4, prefix=p)
    blobs, index = p._keep
    at = blobs.data_ptr()
    short = kvx.make_unit(at, at, None, None, k_index=index, v_index=index, k_bytes=100, v_bytes=100, n_blocks=3, seq=300)
    with pytest.raises(RuntimeError, match="xkv"):  # blobs shorter than their index says
        kvx.Prefix([short], 64)
    with pytest.raises(ValueError, match="index"):
        kvx.Prefix([kvx.make_unit(at, at, None, None, seq=300)], 64)
    with pytest.raises(ValueError, match="empty"):
        kvx.Prefix.encode(k[:, :0].contiguous(), k[:, :0].contiguous())


# ---- refusals and device-side reports ---------------------------------------------------------------

def test_reports(kvx, cuda, H):
    """Bad positions, slots, table entries and lengths are found on the device, touch nothing and are reported."""
    torch = cuda
    b = kvx.Batch(2, 4, 2, 64)
    cos, sin = H.tables(10, 64)
    rope = kvx.Rope(cos, sin)
    x = torch.randn((3, 4, 64), device="cuda").to(torch.bfloat16)
    out = torch.full_like(x, 7.0)
    b.rotate(x, torch.tensor([1, 10, -1], dtype=torch.int32, device="cuda"), rope, out)
    with pytest.raises(RuntimeError, match="position outside the rotation tables"):
        b.check()
    b.check()  # reported once
    assert bool((out[1:] == 7).all()) and not bool((out[0] == 7).all())

    c = H.Paged(2, 4, 2, 64, 0, [20, 20], 16)
    pages = kvx.Pages(c.k_pool, c.v_pool)
    k0 = c.k_pool.clone()
    kv = torch.zeros((1, 2, 64), device="cuda", dtype=torch.bfloat16)
    for slot in (c.k_pool.shape[0] * 16, 1 << 40, (1 << 62) + 5):
        b.append(None, kv, kv, None, None, torch.tensor([slot], device="cuda"), pages, None)
        with pytest.raises(RuntimeError, match="slot outside the page pools"):
            b.check()
    assert torch.equal(c.k_pool.view(torch.int16), k0.view(torch.int16))

    out = torch.empty((2, 4, 64), device="cuda", dtype=torch.bfloat16)
    c.table[0, 1], c.table[1, 1] = c.k_pool.shape[0], -1
    b.attend(c.q, out, pages, c.table, c.lens, 20)
    with pytest.raises(RuntimeError, match="page table entry outside the page pools"):
        b.check()
    c.tails = [(k[:16], v[:16]) for k, v in c.tails]
    H.assert_attends(out, None, c.truth())

    c = H.Paged(2, 4, 2, 64, 0, [20, 20], 16)
    pages = kvx.Pages(c.k_pool, c.v_pool)
    b.attend(c.q, out, pages, c.table, torch.tensor([25, -3], dtype=torch.int32, device="cuda"), 20)
    with pytest.raises(RuntimeError, match="sequence length"):
        b.check()
    c.tails[1] = tuple(x[:0] for x in c.tails[1])
    H.assert_attends(out, None, c.truth())


def test_refusals(kvx, cuda, H):
    torch = cuda
    b = kvx.Batch(2, 4, 2, 64)
    c = H.Paged(2, 4, 2, 64, 16, [4, 4], 16)
    pages = kvx.Pages(c.k_pool, c.v_pool)
    out = torch.empty((2, 4, 64), device="cuda", dtype=torch.bfloat16)

    def attend(**kw):
        a = dict(q=c.q, out=out, pages=pages, table=c.table, lens=c.lens, max_len=4, prefix_table=c.prefix_table,
                 prefix_len=16) | kw
        b.attend(a.pop("q"), a.pop("out"), a.pop("pages"), a.pop("table"), a.pop("lens"), a.pop("max_len"), **a)

    attend()
    b.check()
    for bad, what in [(dict(q=c.q.half()), "torch.bfloat16"), (dict(q=c.q[:, :3]), "must be"), (dict(q=c.q.cpu()), "CUDA"),
                      (dict(out=out.transpose(1, 2)), "contiguous|must be"), (dict(max_len=17), "fewer than max_len"),
                      (dict(prefix_len=17), "fewer than prefix_len"), (dict(lens=c.lens.long()), "int32"),
                      (dict(lens=c.lens[:1]), "one row"), (dict(scale=-1.0), "scale"), (dict(prefix_table=None), "prefix"),
                      (dict(lse=torch.empty((2, 3), device="cuda")), "lse"), (dict(max_len=-1), "bad argument")]:
        with pytest.raises(ValueError, match=what):
            attend(**bad)
    big = torch.empty((3, 4, 64), device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="bad argument"):  # more sequences than the handle's scratch is for
        b.attend(big, big, pages, None, None, 0, prefix_table=c.prefix_table, prefix_len=16)
    odd = torch.empty((2, 4, 66), device="cuda", dtype=torch.bfloat16)[:, :, 1:65]
    with pytest.raises(ValueError, match="16-byte aligned"):
        attend(q=odd)
    pool = torch.zeros((3, 16, 2, 66), device="cuda", dtype=torch.bfloat16)[..., :64]
    with pytest.raises(ValueError, match="16-byte aligned"):
        attend(pages=kvx.Pages(pool, pool))
    with pytest.raises(ValueError, match="other heads"):
        attend(pages=kvx.Pages(c.k_pool[:, :, :1], c.v_pool[:, :, :1]))
    with pytest.raises(NotImplementedError, match="head_dim"):
        n = kvx.Batch(1, 1, 1, 80)
        z = torch.zeros((1, 16, 1, 80), device="cuda", dtype=torch.bfloat16)
        n.attend(z[0, :1], z[0, :1].clone(), kvx.Pages(z, z), None, None, 0)
    with pytest.raises(ValueError, match="axis|axes"):
        kvx.Rope(*H.tables(4, 64), n_axes=3)
    # nothing to do is not an error
    none = torch.empty((0, 4, 64), device="cuda", dtype=torch.bfloat16)
    b.attend(none, none, pages, None, None, 0)
    b.rotate(none, torch.empty(0, dtype=torch.int32, device="cuda"), kvx.Rope(*H.tables(4, 64)), none)
    b.check()


# ---- waits that run out -----------------------------------------------------------------------------

@pytest.mark.parametrize("limit", [0, 1])
@pytest.mark.parametrize("hq,hkv,dim,prefix,batch,page,dtype,coded", [
    (14, 2, 64, 3000, 9, 16, "bf16", False), (32, 8, 128, 20000, 40, 64, "fp16", False), (4, 4, 32, 100, 11, 8, "bf16", False),
    (8, 4, 256, 2000, 10, 128, "bf16", False), (6, 2, 128, 5000, 7, 7, "fp16", False), (5, 1, 32, 700, 3, 20, "bf16", False),
    (8, 4, 256, 900, 6, 5, "bf16", False),
    (14, 2, 64, 4000, 9, 16, "bf16", True), (32, 8, 128, 6000, 20, 64, "bf16", True), (4, 4, 32, 100, 11, 8, "bf16", True),
    (8, 4, 256, 2000, 10, 128, "bf16", True),
])
def test_waits_that_run_out(kvx, cuda, H, hq, hkv, dim, prefix, batch, page, dtype, coded, limit):
    """With no time for its waits the prefix kernel gives up: the call reports it, and a row is right or NaN, never
    what an earlier call left in the scratch.  With its time back the handle works as before."""
    torch = cuda
    lens = [(7 * i) % 40 for i in range(batch)]
    c = H.Paged(batch, hq, hkv, dim, prefix, lens, page, dtype=dtype, paged_prefix=not coded)
    b, pages = kvx.Batch(batch, hq, hkv, dim, dtype=dtype), kvx.Pages(c.k_pool, c.v_pool)
    if coded:
        kept = {"prefix": kvx.Prefix.encode(*(x.transpose(0, 1).contiguous() for x in c.prefix))}
    else:
        kept = {"prefix_table": c.prefix_table, "prefix_len": prefix}
    want, want_lse, tol, _ = truth = c.truth()

    def attend(q):
        out = torch.full((batch, hq, dim), 7.0, device="cuda", dtype=c.q.dtype)
        lse = torch.full((batch, hq), 7.0, device="cuda")
        b.attend(q, out, pages, c.table, c.lens, c.max_len, lse=lse, **kept)
        return out, lse

    attend(c.q.flip(0))  # another call's rows are in the scratch
    b.check()
    b.wait_limit(limit)
    out, lse = attend(c.q)
    if limit == 0:
        with pytest.raises(kvx.DeviceTimeout, match="timed out"):
            b.check()
        assert bool(out.isnan().all()) and bool(lse.isnan().all())
    else:  # whether a wait takes longer is the device's affair
        try:
            b.check()
            late = False
        except kvx.DeviceTimeout:
            late = True
        gone = lse.isnan()
        assert late or not bool(gone.any())
        assert bool((out.isnan().all(-1) == gone).all())
        assert bool(((out.double() - want).abs() <= tol)[~gone].all())
    b.wait_limit(1000000)
    out, lse = attend(c.q)
    b.check()
    H.assert_attends(out, lse, truth)


def test_wait_limit_refuses(kvx, cuda):
    b = kvx.Batch(1, 1, 1, 64)
    with pytest.raises(ValueError, match="wait_limit"):
        b.wait_limit(-1)
