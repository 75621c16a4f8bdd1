"""The operators together: a small decoder that serves requests from a paged cache (``boostr_b200.paged_stack``)."""
import pytest

from boostr_b200 import ops

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SMALL = dict(layers=2, hidden=512, kv=256, ffn=1024, vocab=512, head_dim=64, max_pages=12, page_size=16)


def _stack(requests, **more):
    from boostr_b200.paged_stack import PagedStack

    return PagedStack(requests, pages=requests * 12, **{**SMALL, **more})


def _close(a, b):
    # two ways through the same model: products of other row counts round their activations and attention weights to 16 bits
    # (2^-8) in one of them, in each of 2 layers' 7 products and attentions, against logits of comparable size
    return float((a - b).norm() / b.norm()) < 16 * 2.0 ** -8 / 2


@pytest.mark.parametrize("more", [{}, dict(window=40, sinks=3), dict(head_norms=True, rope_scaling={"type": "linear", "factor": 2.0})])
def test_steps_continue_prompts(more):
    """A token served by a step, and the same token as the last of a longer prompt."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    lengths = [100, 37, 1]
    x = [torch.randn(n + 2, 512, device="cuda", generator=g) for n in lengths]
    a, b = _stack(3, **more), _stack(3, **more)
    a.prompt(torch.cat([y[:-2] for y in x]), lengths)
    a.step(torch.stack([y[-2] for y in x]))
    got = a.step(torch.stack([y[-1] for y in x]))
    want = b.prompt(torch.cat(x), [n + 2 for n in lengths])
    assert a.ctx.tolist() == b.ctx.tolist() == [n + 2 for n in lengths]
    assert _close(got, want)
    # in chunks: the same keys, values and rows
    c = _stack(3, **more)
    c.prompt(torch.cat([x[0][:64], x[1][:5]]), [64, 5, 0])
    assert _close(c.prompt(torch.cat([x[0][64:], x[1][5:], x[2]]), [38, 34, 3]), want)
    assert int(a.missing) == int(b.missing) == int(c.missing) == 0
    ops.check_device_status()


def test_graph_advances_by_itself():
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x = torch.randn(9, 4, 512, device="cuda", generator=g)
    a, b = _stack(4), _stack(4)
    for s in (a, b):
        s.prompt(torch.cat([x[0], x[1]]), [3, 0, 1, 4])
    graph = a.capture()
    assert a.ctx.tolist() == [3, 0, 1, 4]  # capturing serves nothing
    for i in range(2, 9):
        got = graph.replay(hidden=x[i])["logits"]
        assert torch.equal(got, b.step(x[i])), i
    assert a.ctx.tolist() == b.ctx.tolist() == [10, 7, 8, 11] and torch.equal(a.table, b.table) and torch.equal(a.free_count, b.free_count)


def test_pool_that_runs_dry():
    """Requests beyond the last page: their tokens are not kept, the attention meets the hole and says so."""
    from boostr_b200._cabi import B200QError
    from boostr_b200.paged_stack import PagedStack

    s = PagedStack(2, pages=3, **{**SMALL, "max_pages": 4})
    s.prompt(torch.randn(50, 512, device="cuda"), [20, 30])
    assert int(s.missing) == 1 and int(s.free_count) == 0
    with pytest.raises(B200QError, match="out of range"):
        ops.check_device_status()
