"""The serving-step operators together (serve.py): tokens generated behind a shared prompt, the prompt compressed or in
pages, against the same steps evaluated in 64 bits from the projections on."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _rotated(torch, x, pos, cos, sin):
    """x [tokens, heads, dim] turned in 64 bits and rounded once to BF16, as the cache keeps it."""
    half = cos.shape[1]
    x = x.double()
    c, s = cos[pos.long()].double()[:, None], sin[pos.long()].double()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c - b * s, b * c + a * s), -1).to(torch.bfloat16).double()


@pytest.mark.parametrize("compressed", [True, False])
@pytest.mark.parametrize("batch,hq,hkv,dim,prompt,steps", [(3, 4, 2, 64, 333, 19), (34, 8, 2, 128, 700, 33)])
def test_steps_behind_a_prompt(cuda, batch, hq, hkv, dim, prompt, steps, compressed):
    """Tolerance: the caches' values are the exact ones' nearest BF16 neighbours but for values that an FP32
    rotation moves across a rounding boundary (one unit, 2^-7 of a value, in a few of dim products of a score);
    the weights and the output are rounded to BF16 (2^-8 of the largest |v| each)."""
    import serve
    torch = cuda
    s = serve.Session(batch, hq, hkv, dim, prompt, steps, layers=2, compressed=compressed, seed=batch)
    s.run()
    cos, sin = serve.rope_tables(prompt + steps, dim)
    at = torch.arange(prompt, device="cuda")
    for layer in range(2):
        pk = _rotated(torch, s.prompts[layer][0], at, cos, sin)
        pv = s.prompts[layer][1].double()
        q = _rotated(torch, s.new_q[layer, -1], torch.full((batch,), prompt + steps - 1, device="cuda"), cos, sin)
        for b in range(batch):
            tk = _rotated(torch, s.new_k[layer, :, b], prompt + torch.arange(steps, device="cuda"), cos, sin)
            k, v = torch.cat((pk, tk)), torch.cat((pv, s.new_v[layer, :, b].double()))
            k, v = (x.repeat_interleave(hq // hkv, 1) for x in (k, v))
            score = torch.einsum("hd,thd->ht", q[b], k) / math.sqrt(dim)
            want = torch.einsum("ht,thd->hd", score.softmax(-1), v)
            tol = 3 * 2.0 ** -8 * v.abs().amax(0)
            assert bool(((s.out[layer, b].double() - want).abs() <= tol).all()), (layer, b)


def test_prompt_in_pages_and_compressed_agree(cuda):
    """The same tokens reach the softmax either way; only the cut of the prompt may differ."""
    import serve
    torch = cuda
    a, b = (serve.Session(5, 14, 2, 64, 2000, 20, compressed=c, seed=3) for c in (True, False))
    a.run(), b.run()
    assert bool(torch.isfinite(a.out.float()).all())
    tol = 3 * 2.0 ** -8 * max(x[1].abs().max().item() for x in a.prompts + [(None, a.new_v)])
    assert float((a.out.float() - b.out.float()).abs().max()) <= tol
    assert 0 < a.prompt_bytes < b.prompt_bytes


@pytest.mark.parametrize("compressed", [True, False])
@pytest.mark.parametrize("steps", [1, 17])
def test_a_session_runs_again(cuda, steps, compressed):
    """A second run begins again and gives the same outputs; a step past the last is refused on the host."""
    import serve
    torch = cuda
    s = serve.Session(3, 4, 2, 64, 100, steps, layers=2, compressed=compressed, seed=1)
    s.run()
    first = s.out.clone()
    s.run()
    assert torch.equal(s.out, first) and int(s.lens.min()) == int(s.lens.max()) == steps
    with pytest.raises(ValueError, match="steps have been taken"):
        s.step()
    s.rewind()
    for _ in range(steps):  # without the graph
        s.step()
    s.op.check()
    assert torch.equal(s.out, first)
    with pytest.raises(ValueError, match="steps have been taken"):
        s.capture()


def test_a_session_of_no_steps(cuda):
    import serve
    with pytest.raises(ValueError, match="steps have been taken"):
        serve.Session(3, 4, 2, 64, 100, 0).run()


@pytest.mark.parametrize("compressed", [True, False])
@pytest.mark.parametrize("batch,hq,hkv,dim,prompt,steps", [(3, 4, 2, 64, 333, 19), (34, 8, 2, 128, 700, 33), (2, 14, 2, 64, 2000, 1)])
def test_the_newest_and_the_first_own_token(cuda, batch, hq, hkv, dim, prompt, steps, compressed):
    """The last step's even heads look at its own token and its odd heads at the sequence's first, so that a length, a slot
    or a position that is off by one shows.  The cache is where the table says, K rotated and V as it was; the outputs are
    within attention64's bound of what 64 bits make of that cache, and outside of it without either token."""
    import paged_helpers as H
    import serve
    torch = cuda
    s = serve.Session(batch, hq, hkv, dim, prompt, steps, layers=2, compressed=compressed, seed=batch)
    cos, sin = serve.rope_tables(prompt + steps, dim)
    head = torch.arange(hq, device="cuda") // (hq // hkv)
    apart = torch.tensor([[steps - 1]], device="cuda")
    for layer in range(2):
        newest, first = s.new_k[layer, -1][:, head], s.new_k[layer, 0][:, head]
        # turned back by the places between them, the first token's key meets its own rotation
        first = H.rotate64(first.transpose(0, 1), apart.expand(1, hq), cos, sin, None, False, inverse=True)[0].transpose(0, 1)
        at = torch.where((torch.arange(hq, device="cuda") % 2 == 0)[:, None], newest.double(), first)
        s.new_q[layer, -1] = (at * 30.0 * dim ** 0.5 / at.square().sum(-1, keepdim=True)).to(torch.bfloat16)
    s.run()
    per = s.pages[0].page_tokens
    t = torch.arange(steps, device="cuda")
    pos = (prompt + t).to(torch.int32)
    last = torch.full((batch,), prompt + steps - 1, device="cuda", dtype=torch.int32)
    for layer in range(2):
        k, v = s.prompts[layer]
        turned, q = torch.empty_like(k), torch.empty_like(s.new_q[layer, -1])
        s.op.rotate(k, torch.arange(prompt, device="cuda", dtype=torch.int32), s.rope, turned)
        s.op.rotate(s.new_q[layer, -1], last, s.rope, q)
        kv = []
        for b in range(batch):
            page = s.table[b].long()[t // per]
            own_k, own_v = s.pages[layer].k[page, t % per], s.pages[layer].v[page, t % per]
            H.assert_rotated(own_k, s.new_k[layer, :, b], pos[None], cos, sin, None, False, "bf16")
            assert torch.equal(own_v, s.new_v[layer, :, b])
            kv.append((torch.cat((turned, own_k)), torch.cat((v, own_v))))
        truth = H.attention64(q, kv, dim ** -0.5, "bf16")
        H.assert_attends(s.out[layer], None, truth)
        even = torch.arange(hq, device="cuda") % 2 == 0
        for gone, heads in [(prompt + steps - 1, even), (prompt, ~even)]:
            less = [(torch.cat((a[:gone], a[gone + 1:])), torch.cat((c[:gone], c[gone + 1:]))) for a, c in kv]
            off = (H.attention64(q, less, dim ** -0.5, "bf16")[0] - truth[0]).abs() > 2 * truth[2]
            assert float(off[:, heads].double().mean()) > 0.9
