"""GPU tests of the tensor-core prefix kernel in its steady state: items of many tiles, so that each loader's ring (and a
coded prefix's staging slots) goes round many times, against the formula in 64 bits and run by run."""
import pytest

from long_cases import CASES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def H(cuda):
    import paged_helpers
    return paged_helpers


@pytest.mark.parametrize("hq,hkv,dim,batch,prefix,page,dtype", CASES)
def test_long_items(kvx, cuda, H, hq, hkv, dim, batch, prefix, page, dtype):
    """Coded prefixes have raw, 2-, 3- and 4-bit blocks and escapes."""
    from test_gpu_paged import _modes
    torch = cuda
    lens = [(5 * i) % 10 for i in range(batch)]
    if page == 0:
        k, v = _modes(torch, prefix, hkv, dim, 128, 0), _modes(torch, prefix, hkv, dim, 128, 1, special=0.05)
        c = H.Paged(batch, hq, hkv, dim, 0, lens, 16, paged_prefix=False, q_scale=0.7)
        c.prefix = (k.transpose(0, 1), v.transpose(0, 1))
        kept = {"prefix": kvx.Prefix.encode(k, v, code_bits=kvx.CODE_BITS_ALL)}
    else:
        c = H.Paged(batch, hq, hkv, dim, prefix, lens, page, "hnd" if batch % 2 else "nhd", dtype)
        kept = {"prefix_table": c.prefix_table, "prefix_len": prefix}
    b, pages = kvx.Batch(batch, hq, hkv, dim, dtype=dtype), kvx.Pages(c.k_pool, c.v_pool)
    out, lse = torch.full((batch, hq, dim), 7.0, device="cuda", dtype=c.q.dtype), torch.full((batch, hq), 7.0, device="cuda")
    b.attend(c.q, out, pages, c.table, c.lens, c.max_len, lse=lse, **kept)
    for _ in range(8):
        again, lse_again = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
        b.attend(c.q, again, pages, c.table, c.lens, c.max_len, lse=lse_again, **kept)
        assert torch.equal(out.view(torch.int16), again.view(torch.int16)) and torch.equal(lse, lse_again)
    b.check()
    kv = ((torch.cat([c.prefix[0], k]), torch.cat([c.prefix[1], v])) for k, v in c.tails)
    H.assert_attends(out, lse, H.attention64(c.q, kv, c.scale, dtype))


@pytest.mark.parametrize("hq,hkv,dim,batch,prefix,page,dtype", CASES)
def test_rows_that_look_at_one_token(kvx, cuda, H, hq, hkv, dim, batch, prefix, page, dtype):
    """Each query is a multiple of some prefix token's key, so that its output is that token's value: a tile that came from
    another place or another round of the ring changes it by as much as it is (an average over the prefix hides that)."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(dim + batch)
    lens = [i % 3 for i in range(batch)]
    c = H.Paged(batch, hq, hkv, dim, prefix, lens, page or 16, dtype=dtype, paged_prefix=page != 0)
    if page == 0:
        k, v = c.prefix
        far = torch.rand(v.shape, generator=g, device="cuda") < 0.01  # (some escapes)
        c.prefix = (k, torch.where(far, v / 1024, v))
        kept = {"prefix": kvx.Prefix.encode(*(x.transpose(0, 1).contiguous() for x in c.prefix), code_bits=kvx.CODE_BITS_ALL)}
    else:
        kept = {"prefix_table": c.prefix_table, "prefix_len": prefix}
    aim = torch.randint(0, prefix, (batch, hq), generator=g, device="cuda")
    head = torch.arange(hq, device="cuda") // (hq // hkv)
    key = c.prefix[0][aim, head].double()
    q = (key * 30.0 / (key.square().sum(-1, keepdim=True) * c.scale)).to(c.q.dtype)
    b, pages = kvx.Batch(batch, hq, hkv, dim, dtype=dtype), kvx.Pages(c.k_pool, c.v_pool)
    out, lse = torch.empty_like(q), torch.empty((batch, hq), device="cuda")
    b.attend(q, out, pages, c.table, c.lens, c.max_len, lse=lse, **kept)
    b.check()
    kv = ((torch.cat([c.prefix[0], k]), torch.cat([c.prefix[1], v])) for k, v in c.tails)
    truth = H.attention64(q, kv, c.scale, dtype)
    weight = ((key * q.double()).sum(-1) * c.scale - truth[1]).exp()
    assert float((weight > 0.9).double().mean()) > 0.3  # (they do look at it: half of them at dim 32, nearly all above)
    H.assert_attends(out, lse, truth)
