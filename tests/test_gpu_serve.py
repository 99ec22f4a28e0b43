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
