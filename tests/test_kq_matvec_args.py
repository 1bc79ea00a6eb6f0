"""Context.kq_matvec's checks of its tensors: what the library would read as something else is refused before the library is called
(CPU: tensors that say they are on a GPU, and a library that only counts its calls), and on the GPU."""
import pytest
import torch

import loki_amd
from loki_amd import FL_Q2K, FL_Q4K, FL_Q6K, KQ_BYTES, LokiError

R, K, N = 3, 512, 2


class On:
    """a CPU tensor that says it is on GPU `dev`"""

    def __init__(self, t, dev=0):
        self.t, self.dev, self.device = t, dev, "cuda:%d" % dev

    def get_device(self):
        return self.dev

    def __getattr__(self, name):
        return getattr(self.t, name)


class Lib:
    calls = 0

    def fl_kq_matvec_dev(self, *args):
        self.calls += 1
        return 0


@pytest.fixture
def made(monkeypatch):
    c = loki_amd.Context.__new__(loki_amd.Context)
    c.torch, c.ctx, c._device = torch, None, 0
    lib = Lib()
    monkeypatch.setattr(loki_amd, "lib", lambda: lib)
    return c, lib


def tensors(fmt=FL_Q4K):
    return {"w": torch.zeros(R * (K // 256) * KQ_BYTES[fmt], dtype=torch.uint8), "q": torch.zeros((N, K), dtype=torch.int8), "d": torch.zeros((N, K // 256))}


@pytest.mark.parametrize("fmt", [FL_Q2K, FL_Q4K, FL_Q6K])
def test_calls_that_go_through(made, fmt):
    c, lib = made
    t = tensors(fmt)
    call = lambda y=None, **k: c.kq_matvec(fmt, On(k.get("w", t["w"])), R, K, On(k.get("q", t["q"])), On(k.get("d", t["d"])), y)   # noqa: E731
    out = call()
    assert out.dtype is torch.float32 and out.shape == (N, R)
    for y in (torch.zeros((N, R)), torch.zeros(N * R)):
        y = On(y)
        assert call(y) is y
    call(q=t["q"].view(N, -1, 256), d=t["d"].view(-1), w=torch.cat([t["w"], t["w"]]))   # (the same bytes in another shape; more of them)
    call(w=t["w"].view(R, -1).view(torch.int8))
    assert lib.calls == 5
    assert c.kq_matvec(fmt, On(t["w"]), R, K, On(t["q"][:0]), On(t["d"][:0])).shape == (0, R)


@pytest.mark.parametrize("name,bad", [
    ("q", lambda t: t.to(torch.int16)), ("q", lambda t: t.view(torch.uint8)), ("q", lambda t: t[:, :256]), ("q", lambda t: t.t().contiguous().t()),
    ("q", lambda t: torch.zeros((2 * N, K), dtype=torch.int8)[::2]), ("q", lambda t: torch.zeros((1, K), dtype=torch.int8).expand(N, K)), ("q", lambda t: t.view(2 * N, K // 2)),
    ("d", lambda t: t.double()), ("d", lambda t: t.half()), ("d", lambda t: t[:, :1]), ("d", lambda t: t.t().contiguous().t()), ("d", lambda t: t[:1]),
    ("w", lambda t: t[:-1]), ("w", lambda t: torch.cat([t, t])[::2])])
@pytest.mark.parametrize("fmt", [FL_Q4K, FL_Q6K])
def test_refused_inputs(made, fmt, name, bad):
    c, lib = made
    t = tensors(fmt)
    t[name] = bad(t[name])
    with pytest.raises(LokiError, match="kq_matvec"):
        c.kq_matvec(fmt, On(t["w"]), R, K, On(t["q"]), On(t["d"]))
    assert lib.calls == 0


@pytest.mark.parametrize("y", [torch.zeros((N, R + 1)), torch.zeros((N, R), dtype=torch.float64), torch.zeros((R, N)).t(), torch.zeros((N, 2 * R))[:, ::2],
                               torch.zeros(1)])
def test_refused_outputs(made, y):
    c, lib = made
    t = tensors()
    with pytest.raises(LokiError, match="y must be"):
        c.kq_matvec(FL_Q4K, On(t["w"]), R, K, On(t["q"]), On(t["d"]), On(y))
    assert lib.calls == 0


@pytest.mark.parametrize("name", ["w", "q", "d", "y"])
@pytest.mark.parametrize("dev", [-1, 1])
def test_refused_devices(made, name, dev):
    c, lib = made
    t = dict(tensors(), y=torch.zeros((N, R)))
    g = {k: On(v, dev if k == name else 0) for k, v in t.items()}
    with pytest.raises(LokiError, match="context's GPU"):
        c.kq_matvec(FL_Q4K, g["w"], R, K, g["q"], g["d"], g["y"])
    assert lib.calls == 0


@pytest.mark.gpu
def test_on_the_gpu(ctx):
    t = {k: v.cuda() for k, v in tensors().items()}
    t["d"].fill_(1.0)
    y = torch.full((N, R), 7.0, device="cuda")
    ctx.kq_matvec(FL_Q4K, t["w"], R, K, t["q"], t["d"], y)
    ctx.sync()
    assert not torch.any(y)
    for bad in ({"q": torch.zeros((K, N), dtype=torch.int8, device="cuda").t()}, {"d": t["d"].double()}, {"q": t["q"].cpu()}, {"w": t["w"].cpu()}):
        a = dict(t, **bad)
        with pytest.raises(LokiError, match="kq_matvec"):
            ctx.kq_matvec(FL_Q4K, a["w"], R, K, a["q"], a["d"])
    with pytest.raises(LokiError, match="y must be"):
        ctx.kq_matvec(FL_Q4K, t["w"], R, K, t["q"], t["d"], torch.zeros((N, 2 * R), device="cuda")[:, ::2])
    ctx.sync()
