"""A tensor of another GPU, or a status word that is none, is refused on the host: its pointer would be used as one of this GPU's.
Stand-ins take the place of CUDA tensors, so that no GPU is needed."""
import pytest
import torch

from lfm3_kv800 import kv800, spec

HERE, THERE = torch.device("cuda:0"), torch.device("cuda:1")


class Fake(torch.Tensor):
    """A host tensor that says it lies on a GPU."""

    @staticmethod
    def make(t, device=HERE):
        f = t.as_subclass(Fake)
        f.where = device
        return f

    @property
    def is_cuda(self):
        return True

    @property
    def device(self):
        return self.where


def i32(*shape, device=HERE):
    return Fake.make(torch.zeros(*shape, dtype=torch.int32), device)


@pytest.fixture(autouse=True)
def no_call(monkeypatch):
    """Whatever is not refused ends here, before the library."""
    class Reached(Exception):
        pass

    def call(*a):
        raise Reached
    monkeypatch.setattr(kv800._lib, "call", call)
    monkeypatch.setitem(kv800._CHOSEN, "cuda", "cuda")
    for m in (kv800, spec):
        monkeypatch.setattr(m, "_raw_stream", lambda index: 0)
    return Reached


def pages(device=HERE):
    return [i32(2, 4, device=device), i32(8, device=device), Fake.make(torch.zeros(6, dtype=torch.int64), device)]


@pytest.mark.parametrize("which", ["qlen", "table", "ring", "state", "quant", "status"])
def test_step_tables_devices(which):
    there = lambda name: THERE if which == name else HERE  # noqa: E731
    own, other = pages(), pages(THERE)
    g = spec.Pages(*[other[i] if which == n else own[i] for i, n in enumerate(("table", "ring", "state"))], 64)
    with pytest.raises((RuntimeError, ValueError), match="cuda:1"):
        spec.step_tables(i32(2), i32(2, device=there("qlen")), 4, g, spec.Pages(*pages(there("quant")), 1280, "flushed"),
                         i32(1, device=there("status")))


@pytest.mark.parametrize("which", ["tokens", "query_start_loc", "uniform", "noise", "draft_probs", "temperature", "status"])
def test_verify_devices(which):
    f = lambda *s: Fake.make(torch.ones(*s))  # noqa: E731
    a = dict(logits=f(6, 9), tokens=i32(6), query_start_loc=i32(3), uniform=f(6), noise=f(2, 9), max_drafts=2, draft_probs=f(4, 9),
             temperature=f(2), status=i32(1))
    a[which] = Fake.make(a[which].as_subclass(torch.Tensor), THERE)
    with pytest.raises((RuntimeError, ValueError), match="cuda:1"):
        spec.verify(**a)


@pytest.mark.parametrize("which", ["cos_t", "sin_t", "epool", "qpool", "sk", "sv", "status"])
def test_extend_devices(which):
    bf = lambda *s: Fake.make(torch.zeros(*s, dtype=torch.bfloat16))  # noqa: E731
    win = 256 if which in ("sk", "sv") else 0
    off = Fake.make(torch.zeros(2, dtype=torch.int64))
    d = dict(qpool=Fake.make(torch.zeros(51200, dtype=torch.uint8)), boff=Fake.make(torch.zeros(2, 1, dtype=torch.int64)), epool=bf(65536),
             eoff=Fake.make(torch.zeros(2, 1, dtype=torch.int64)), ebs=64, e_hs=16384, e_ts=256, e_v=128, sk=bf(4096), sv=bf(4096),
             skoff=off, svoff=off, N=i32(2), NQ=i32(2), nqmax=1, win=win)
    c = dict(cos_t=bf(64, 32), sin_t=bf(64, 32), status=i32(1))
    for x in (d, c):
        if which in x:
            x[which] = Fake.make(x[which].as_subclass(torch.Tensor), THERE)
    with pytest.raises((RuntimeError, ValueError), match="cuda:1"):
        kv800.extend(kv800.Paged(**d), bf(6, 16, 128), i32(3), c["cos_t"], c["sin_t"], 3, c["status"])


@pytest.mark.parametrize("status", [torch.zeros(1, dtype=torch.int32), Fake.make(torch.zeros(1, dtype=torch.int64)), i32(0), 0])
def test_status_is_a_device_int32(status):
    f = lambda *s: Fake.make(torch.ones(*s))  # noqa: E731
    with pytest.raises((RuntimeError, ValueError), match="status"):
        spec.step_tables(i32(2), i32(2), 4, spec.Pages(*pages(), 64), None, status)
    with pytest.raises((RuntimeError, ValueError), match="status"):
        spec.verify(f(6, 9), i32(6), i32(3), f(6), f(2, 9), 2, status=status)
    bf = lambda *s: Fake.make(torch.zeros(*s, dtype=torch.bfloat16))  # noqa: E731
    P = kv800.Paged(epool=bf(65536), eoff=Fake.make(torch.zeros(2, 1, dtype=torch.int64)), ebs=64, e_hs=16384, e_ts=256, e_v=128,
                    N=i32(2), NQ=i32(2), nqmax=0, win=256)
    with pytest.raises((RuntimeError, ValueError), match="status"):
        kv800.extend(P, bf(6, 16, 128), i32(3), None, None, 3, status)


@pytest.mark.parametrize("short", ["eoff", "skoff", "svoff"])
def test_extend_short_tables(short):
    """A table with fewer rows than the batch would be read past its end."""
    bf = lambda *s: Fake.make(torch.zeros(*s, dtype=torch.bfloat16))  # noqa: E731
    n = lambda name: 1 if name == short else 2  # noqa: E731
    P = kv800.Paged(epool=bf(65536), eoff=Fake.make(torch.zeros(n("eoff"), 1, dtype=torch.int64)), ebs=64, e_hs=16384, e_ts=256, e_v=128,
                    sk=bf(4096), sv=bf(4096), skoff=Fake.make(torch.zeros(n("skoff"), dtype=torch.int64)),
                    svoff=Fake.make(torch.zeros(n("svoff"), dtype=torch.int64)), N=i32(2), NQ=i32(2), nqmax=0, win=256)
    with pytest.raises(ValueError, match=short):
        kv800.extend(P, bf(6, 16, 128), i32(3), None, None, 3)


def test_stand_ins_get_through(no_call):
    """What the other tests refuse is refused for its one wrong tensor: with all of them right the library is reached."""
    f = lambda *s: Fake.make(torch.ones(*s))  # noqa: E731
    with pytest.raises(no_call):
        spec.step_tables(i32(2), i32(2), 4, spec.Pages(*pages(), 64), spec.Pages(*pages(), 1280, "flushed"), i32(1))
    with pytest.raises(no_call):
        spec.verify(f(6, 9), i32(6), i32(3), f(6), f(2, 9), 2, f(4, 9), f(2), i32(1))
