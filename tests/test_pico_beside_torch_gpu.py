"""pico's launches between torch's: a layer of experts run on pico's own stream by a
program that has torch write the parameters before it and read the results behind it,
without waiting for the device."""
import pytest
import torch

import perf.operators as operators

pytestmark = pytest.mark.gpu

CASE = {"name": "layer", "kind": "moe", "tokens": 2048, "d": 256, "ff": 512, "experts": 8, "topk": 2}


@pytest.fixture
def own():
    operators.own = True
    yield
    operators.own = False


def test_the_layer_starts_behind_torchs_writes_and_torch_reads_behind_the_layer(dev, own):
    st = operators.prepare(CASE, 1)
    session, x = st["session"], st["leaves"]["x"]
    first = {k: t.clone() for k, t in operators.run(st).items()}
    torch.cuda.synchronize()
    values = torch.randn(CASE["tokens"], CASE["d"], device=dev, generator=torch.Generator(dev).manual_seed(2))
    out = operators.run(st)
    for t in out.values():
        t.fill_(7)  # what a read ahead of the layer would find
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)  # some ms, and only then the new tokens
    session.view(x).copy_(values)
    got = {k: t.clone() for k, t in operators.run(st).items()}
    torch.cuda.synchronize()
    for t in out.values():
        t.fill_(7)
    torch.cuda.synchronize()
    again = {k: t.clone() for k, t in operators.run(st).items()}  # (the clones are issued at once)
    torch.cuda.synchronize()
    for k, t in operators.run(st).items():
        torch.cuda.synchronize()
        assert torch.equal(again[k], t) and torch.equal(got[k], t), k
        assert not torch.equal(first[k], t), k


def test_an_error_leaves_no_arena_behind(dev, own):
    from pico_amd.pico import PicoError

    st = operators.prepare(CASE, 1)
    lib = st["session"].lib
    before = lib.arena_ctx_current()
    broken = dict(st, case=dict(CASE, topk=CASE["experts"] + 1))
    with pytest.raises(PicoError):
        operators.run(broken)
    assert lib.arena_ctx_current() == before
    operators.run(st)
