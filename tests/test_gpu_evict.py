"""Eviction of cached rows on the GPU against a plain selection and gather."""
import math

import pytest
import torch

from tests import kv_util as U

pytestmark = pytest.mark.gpu


def plain_keep(x, n, budget, sink, recent):
    """Kept row numbers of one head, ascending (the definition, by sorting)."""
    if n <= budget:
        return list(range(n))
    w = [-math.inf if math.isnan(v) else v + 0.0 for v in x[:n].tolist()]
    free = sorted(range(sink, n - recent), key=lambda t: (-w[t], t))[:budget - sink - recent]
    return sorted(list(range(sink)) + free + list(range(n - recent, n)))


class Case:
    def __init__(self, lens, kvh, kv, seed, kind="heavy", extra=5, slots_extra=2):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.kvh, self.kv = lens, kvh, kv
        self.cap, self.row = max(max(lens), 1) + extra, U.row_bytes(kvh, kv)
        n_slots = len(lens) + slots_extra
        self.slots = torch.randperm(n_slots, generator=g)[:len(lens)]
        self.host = {n: torch.randint(0, 256, (n_slots, self.cap, self.row), generator=g, dtype=torch.uint8) for n in ("k", "v")}
        x = torch.randn(n_slots, kvh, self.cap, generator=g)
        if kind == "heavy":
            x = torch.exp(3 * x)
        elif kind == "ties":
            x = (x * 2).round() / 2
        elif kind == "odd":      # NaN, infinities, signed zeros, subnormals
            pool = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42, 1.0, -1.0, 3.4e38])
            x = pool[torch.randint(0, len(pool), x.shape, generator=g)]
        elif kind == "equal":
            x = torch.full_like(x, 0.25)
        self.scores = x
        self.k, self.v = self.host["k"].cuda(), self.host["v"].cuda()
        dev = lambda t: torch.tensor([t[i].data_ptr() for i in range(n_slots)], dtype=torch.int64).cuda()  # noqa: E731
        self.kt, self.vt = dev(self.k), dev(self.v)
        self.ids = self.slots.cuda()
        self.seq = torch.tensor(lens, dtype=torch.int32).cuda()

    def heads(self, rows):
        """Bytes of a head inside rows [..., row]: list of index tensors per head."""
        if self.kv == "int4":
            at, _, sc = U._int4_places(self.kvh)
            return [torch.cat([at[j], sc[j]]).unique() for j in range(self.kvh)]
        e = 256 if self.kv == "bf16" else 128
        return [torch.arange(j * e, (j + 1) * e) for j in range(self.kvh)]

    def check(self, budget, sink, recent, in_place):
        from glake_b200 import ops
        before = self.scores.cuda()
        out = before if in_place else torch.full_like(before, 7.0)
        first = out.cpu().clone()
        kept = ops.evict_rows(before, self.kt.data_ptr(), self.vt.data_ptr(), self.kvh, self.ids, self.seq, max(self.lens), budget, sink,
                              recent, self.kv if self.kv != "bf16" else "auto", scores_out=None if in_place else out)
        torch.cuda.synchronize()
        assert ops.attn_status() == 0
        kept, out = kept.cpu(), out.cpu()
        want_rows = {n: t.clone() for n, t in self.host.items()}
        want_scores = first.clone()
        for i, n in enumerate(self.lens):
            s = int(self.slots[i])
            for j, at in enumerate(self.heads(None)):
                keep = plain_keep(self.scores[s, j], n, budget, sink, recent)
                assert kept[i, j].tolist() == keep + [-1] * (budget - len(keep)), (i, j, n)
                idx = torch.tensor(keep, dtype=torch.long)
                want_scores[s, j, :n] = 0
                want_scores[s, j, :len(keep)] = self.scores[s, j, idx]
                if n > budget:
                    for name in ("k", "v"):
                        want_rows[name][s, :budget, at] = self.host[name][s, idx][:, at]
        assert torch.equal(out.nan_to_num(nan=123.0), want_scores.nan_to_num(nan=123.0))
        for name in ("k", "v"):
            assert torch.equal(getattr(self, name).cpu(), want_rows[name])


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3", "int4"])
@pytest.mark.parametrize("kvh", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("in_place", [True, False])
def test_shapes(kv, kvh, in_place):
    Case([0, 1, 63, 64, 65, 130, 700, 333], kvh, kv, 1).check(64, 4, 16, in_place)
    Case([257, 300, 256, 1000], kvh, kv, 2).check(256, 0, 0, in_place)
    Case([9, 5], kvh, kv, 3).check(1, 0, 1, in_place)


@pytest.mark.parametrize("kind", ["heavy", "ties", "odd", "equal"])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (1, 1, 0), (7, 0, 7), (100, 100, 0), (99, 50, 49), (500, 4, 33), (1999, 0, 0), (2000, 3, 5)])
def test_weights_and_windows(kind, budget, sink, recent):
    Case([2000, 1500, 501], 2, "bf16", 4, kind).check(budget, sink, recent, True)


@pytest.mark.parametrize("in_place", [True, False])
def test_rows_beyond_shared_memory(in_place):
    """More rows than the selection holds on chip: weights are read again, and moved in order when in place."""
    Case([60000, 45057, 45056, 10], 1, "fp8_e4m3", 5, "ties").check(20000, 4, 100, in_place)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3", "int4"])
def test_one_row_goes(kv):
    """Everything behind one early row moves by one: every chunk's sources lie in the next chunk's destination."""
    c = Case([5000, 4097], 4, kv, 6, "equal")
    c.scores[:, :, 3] = 0.0
    c.check(4999, 0, 0, True)
    c = Case([4097], 2, kv, 7, "equal")
    c.scores[:, :, 0] = -1.0
    c.check(4096, 0, 0, True)


@pytest.mark.parametrize("kv", ["bf16", "int4"])
def test_many_heads_in_flight_repeated(kv):
    """More chunks than the GPU holds at once, several times: the order in which chunks run varies, the result does not."""
    for seed in range(3):
        Case([3000] * 24, 16, kv, 10 + seed, "heavy", extra=1, slots_extra=0).check(1500 + 300 * seed, 4, 64, True)


def test_captured_twice_and_another_stream():
    from glake_b200 import ops
    c = Case([900, 40], 4, "bf16", 8)
    scores, out = c.scores.cuda(), torch.zeros_like(c.scores).cuda()
    k0, v0 = c.k.clone(), c.v.clone()

    def call():
        return ops.evict_rows(scores, c.kt.data_ptr(), c.vt.data_ptr(), 4, c.ids, c.seq, 900, 128, 4, 8, scores_out=out)
    want = call().clone()
    k1, o1 = c.k.clone(), out.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            kept = call()
        for _ in range(3):
            c.k.copy_(k0)
            c.v.copy_(v0)
            out.zero_()
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, want) and torch.equal(c.k, k1) and torch.equal(out, o1)
