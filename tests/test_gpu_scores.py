"""Accumulated attention weights on the GPU (decode steps and prompts), against 64-bit forms."""
import numpy as np
import pytest
import torch

from tests import gpu_util, kv_util as U
from tests.synth import normal_bf16

pytestmark = pytest.mark.gpu


def make(seed, lens, kvh, kv):
    rs = np.random.RandomState(seed)
    k = [normal_bf16(rs, n, kvh, 128) for n in lens]
    v = [normal_bf16(rs, n, kvh, 128) for n in lens]
    if kv == "bf16":
        return U.Ranges(k, v, kv), rs
    scale = lambda rows: torch.cat(rows).float().abs().amax((0, 2)) / 448.0 * 0.97  # noqa: E731
    return U.Ranges(k, v, kv, scale(k), scale(v)), rs


def fresh_scores(r, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(r.k.shape[0], r.kvh, r.cap, generator=g)


def weight_tolerance(r, q, i, scale, want, before):
    """Weights are exp2 of an fp32 logit minus an fp32 maximum over an fp32 sum: the logit's error (twice: the weight's
    own and the sum's), a few units of exp2 and the division, and the rounding of the sum that is stored."""
    e = U.logit_error(q, r.rows64("k", i), scale, r.kv)
    return want * (2 * e + 2.0 ** -19) + (before + want) * 2.0 ** -23 + 1e-30


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3", "int4"])
@pytest.mark.parametrize("h,kvh", [(8, 8), (32, 8), (64, 8), (16, 1), (8, 1), (4, 2), (6, 3), (12, 12), (16, 4), (24, 6)])
def test_decode_accumulates(kv, h, kvh):
    from glake_b200 import ops
    lens = [1, 2, 15, 16, 17, 33, 0, 64, 129, 255, 257, 700, 1500]
    r, rs = make(h * 100 + kvh, lens, kvh, kv)
    scale = 128 ** -0.5
    scores = fresh_scores(r, 3)
    want = scores.double().clone()
    dev = scores.cuda()
    plain_out = None
    for step in range(2):
        q = (normal_bf16(rs, len(lens), h, 128).float() * 1.5).bfloat16()
        args = (q.cuda().unsqueeze(1), r.k_table.data_ptr(), r.v_table.data_ptr(), r.max_len, kvh, len(lens), r.slot_ids, None, None,
                r.seq_lens, None, None, None, None, None, None, scale, True, -1, -1, None, 0)
        before = want.clone()
        out, lse = ops.fwd_kvcache(*args, **r.quant(), scores=dev)
        plain_out, plain_lse = ops.fwd_kvcache(*args, **r.quant())
        torch.cuda.synchronize()
        assert ops.attn_status() == 0
        assert torch.equal(out, plain_out) and torch.equal(lse, plain_lse)      # the accumulating form attends the same
        got = dev.cpu().double()
        for i, n in enumerate(lens):
            s = r.slots[i]
            w = U.attention64(q[i], r.rows64("k", i), r.rows64("v", i), scale)[2]
            want[s, :, :n] += w
            tol = weight_tolerance(r, q[i], i, scale, w, before[s, :, :n])
            assert bool(((got[s, :, :n] - before[s, :, :n] - w).abs() <= tol).all()), (i, n)
            assert torch.equal(got[s, :, n:], scores[s, :, n:].double())        # rows behind the context
        spare = [s for s in range(r.k.shape[0]) if s not in r.slots.tolist()]
        assert torch.equal(got[spare], scores[spare].double())                  # slots that no entry names
        want = got.clone()


@pytest.mark.parametrize("kv,h,kvh", [("bf16", 32, 8), ("fp8_e4m3", 8, 1), ("int4", 32, 8), ("int4", 16, 16)])
def test_long_contexts_sum_to_the_query_heads(kv, h, kvh):
    """Contexts cut over many CTAs: the weights of a kv head sum to its number of q heads, and match the 64-bit ones."""
    from glake_b200 import ops
    lens = [20000, 12345]
    r, rs = make(5, lens, kvh, kv)
    q = normal_bf16(rs, 2, h, 128)
    dev = torch.zeros(r.k.shape[0], kvh, r.cap, device="cuda")
    out = torch.empty(2, h, 128, dtype=torch.bfloat16, device="cuda")
    quant = r.quant()
    ops.paged_attention_v1(out, q.cuda(), r.k_table.data_ptr(), r.v_table.data_ptr(), kvh, 128 ** -0.5, r.seq_lens, 1, r.max_len, None,
                           quant.get("kv_cache_dtype", "auto"), 1.0, r.slot_ids, k_scale=quant.get("k_scale"),
                           v_scale=quant.get("v_scale"), scores=dev)
    torch.cuda.synchronize()
    got = dev.cpu().double()
    for i in range(2):
        w = U.attention64(q[i], r.rows64("k", i), r.rows64("v", i), 128 ** -0.5)[2]
        tol = weight_tolerance(r, q[i], i, 128 ** -0.5, w, torch.zeros_like(w))
        assert bool(((got[r.slots[i], :, :lens[i]] - w).abs() <= tol).all())
        assert bool(((got[r.slots[i]].sum(-1) - h // kvh).abs() < 1e-3 * (h // kvh)).all())


def test_batches_beyond_the_schedules_table():
    from glake_b200 import ops
    rs = np.random.RandomState(0)
    lens = [int(x) for x in rs.randint(0, 60, size=1030)]
    for kv in ("bf16", "int4"):
        r, rs = make(1, lens, 2, kv)
        q = normal_bf16(rs, len(lens), 4, 128)
        dev = torch.zeros(r.k.shape[0], 2, r.cap, device="cuda")
        out, _ = ops.fwd_kvcache(q.cuda().unsqueeze(1), r.k_table.data_ptr(), r.v_table.data_ptr(), r.max_len, 2, len(lens), r.slot_ids,
                                 None, None, r.seq_lens, None, None, None, None, None, None, 0.1, True, -1, -1, None, 0, **r.quant(),
                                 scores=dev)
        got = dev.cpu().double()
        for i, n in enumerate(lens):
            w = U.attention64(q[i], r.rows64("k", i), r.rows64("v", i), 0.1)[2]
            assert bool(((got[r.slots[i], :, :n] - w).abs() <= weight_tolerance(r, q[i], i, 0.1, w, 0 * w)).all())


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3", "int4"])
def test_fused_step_accumulates_the_new_row_too(kv):
    """decode_step with scores: the appended row takes part; a strided, non-contiguous score tensor; one slot twice."""
    from glake_b200 import ops
    h, kvh, lens = 16, 4, [1, 16, 300]
    rs = np.random.RandomState(9)
    k = [normal_bf16(rs, n, kvh, 128) for n in lens]
    v = [normal_bf16(rs, n, kvh, 128) for n in lens]
    ks = vs = torch.full((kvh,), 0.0101) if kv != "bf16" else None
    r = U.Ranges([x[:-1] for x in k], [x[:-1] for x in v], kv, ks, vs)
    r.lens = lens
    r.seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()
    q = normal_bf16(rs, 3, h, 128)
    wide = torch.zeros(r.k.shape[0], 2, kvh, r.cap + 3, device="cuda")
    scores = wide[:, 1, :, :r.cap]
    off = torch.tensor([(n - 1) * r.row for n in lens]).cuda()
    out = torch.empty(3, h, 128, dtype=torch.bfloat16, device="cuda")
    quant = r.quant()
    ops.decode_step(out, q.cuda(), torch.stack([x[-1] for x in k]).cuda(), torch.stack([x[-1] for x in v]).cuda(),
                    r.k_table.data_ptr(), r.v_table.data_ptr(), off, r.slot_ids, r.seq_lens, max(lens), kvh, 0.1, scores=scores, **quant)
    torch.cuda.synchronize()
    got = scores.cpu().double()
    assert float(wide[:, 0].abs().max()) == 0 and float(wide[:, 1, :, r.cap:].abs().max()) == 0
    for i, n in enumerate(lens):
        assert torch.equal(r.k[r.slots[i], n - 1].cpu(), U.encode(k[i][-1:], kv, ks)[0])
        w = U.attention64(q[i], r.rows64("k", i), r.rows64("v", i), 0.1)[2]
        assert bool(((got[r.slots[i], :, :n] - w).abs() <= weight_tolerance(r, q[i], i, 0.1, w, 0 * w)).all())
    # the same slot named by two entries receives both
    two = torch.tensor([int(r.slots[2])] * 2).cuda()
    dev = torch.zeros(r.k.shape[0], kvh, r.cap, device="cuda")
    ops.paged_attention_v1(out[:2], q[:2].cuda(), r.k_table.data_ptr(), r.v_table.data_ptr(), kvh, 0.1, r.seq_lens[[2, 2]], 1, 300, None,
                           quant.get("kv_cache_dtype", "auto"), 1.0, two, k_scale=quant.get("k_scale"), v_scale=quant.get("v_scale"), scores=dev)
    w = sum(U.attention64(q[j], r.rows64("k", 2), r.rows64("v", 2), 0.1)[2] for j in (0, 1))
    assert bool(((dev[two[0]].cpu()[:, :300].double() - w).abs() <= 2 * weight_tolerance(r, q[0], 2, 0.1, w, w)).all())


def prompt64(r, q, i, q_start, q_len, window, scale):
    k = r.rows64("k", i)
    if r.kv != "bf16":
        k = k.bfloat16().double()      # quantised caches are read back into bf16 first
    n, (_, h, _) = r.lens[i], q.shape
    w = min(window, q_len, n)
    total = torch.zeros(r.kvh, n, dtype=torch.float64)
    for j in range(w):
        end = n - w + j + 1
        total[:, :end] += U.attention64(q[q_start + q_len - w + j], k[:end], k[:end], scale)[2]
    return total


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3", "int4"])
@pytest.mark.parametrize("h,kvh,window", [(8, 8, 1), (32, 8, 16), (8, 1, 33), (16, 1, 64), (6, 3, 5), (4, 2, 100)])
def test_prompt_scores(kv, h, kvh, window):
    from glake_b200 import ops
    lens, q_lens = [1, 17, 64, 65, 0, 200, 901], [1, 3, 64, 40, 0, 200, 130]
    r, rs = make(window, lens, kvh, kv)
    q = normal_bf16(rs, sum(q_lens) + 2, h, 128)
    start = [2 + sum(q_lens[:i]) for i in range(len(lens))]
    scale = 0.11
    scores = fresh_scores(r, 4)
    dev = scores.cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    quant = r.quant()
    quant.pop("v_scale", None)
    ops.prompt_scores(dev, q.cuda(), r.k_table.data_ptr(), kvh, scale, r.slot_ids, r.seq_lens, i32(q_lens), i32(start), r.max_len, window,
                      **quant)
    torch.cuda.synchronize()
    got = dev.cpu().double()
    want_all = scores.double().clone()
    for i, n in enumerate(lens):
        s = r.slots[i]
        want = prompt64(r, q, i, start[i], q_lens[i], window, scale)
        e = max((U.logit_error(q[j], r.rows64("k", i), scale, "bf16") for j in range(start[i], start[i] + q_lens[i])), default=0)
        # the sum of at most window x g weights adds its own roundings, half a step each
        tol = want * (2 * e + 2.0 ** -18) + scores[s, :, :n].double() * 2.0 ** -23 + 1e-30
        assert bool(((got[s, :, :n] - scores[s, :, :n].double() - want).abs() <= tol).all()), (i, n)
        want_all[s, :, :n] = got[s, :, :n]
    assert torch.equal(got, want_all)


def test_prompt_scores_runs_and_windows_past_the_prompt():
    """A long prompt in many runs, and rows in more than one round of warps."""
    from glake_b200 import ops
    lens, h, kvh, window = [9000], 16, 1, 64
    r, rs = make(2, lens, kvh, "bf16")
    q = normal_bf16(rs, 9000, h, 128)
    dev = torch.zeros(r.k.shape[0], kvh, r.cap, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    ops.prompt_scores(dev, q.cuda(), r.k_table.data_ptr(), kvh, 0.2, r.slot_ids, r.seq_lens, i32([9000]), i32([0]), 9000, window)
    want = prompt64(r, q, 0, 0, 9000, window, 0.2)
    got = dev[r.slots[0]].cpu().double()
    assert bool(((got[:, :9000] - want).abs() <= want * (2.0 ** -14) + 1e-9).all())   # 2 x 2^-20 x 0.2 x |q||k| (< 150 x 4)
    assert float(got[:, 9000:].abs().max()) == 0


def test_capture_and_two_streams():
    """Captured calls own their scratch; calls on two streams at once do not share any."""
    from glake_b200 import ops
    r, rs = make(3, [3000, 40], 8, "bf16")
    q = normal_bf16(rs, 2, 32, 128).cuda()
    shape = (r.k.shape[0], 8, r.cap)

    def call(dev):
        return ops.fwd_kvcache(q.unsqueeze(1), r.k_table.data_ptr(), r.v_table.data_ptr(), r.max_len, 8, 2, r.slot_ids, None, None,
                               r.seq_lens, None, None, None, None, None, None, 0.1, True, -1, -1, None, 0, scores=dev)[0]
    want = torch.zeros(shape, device="cuda")
    out = call(want).clone()
    a, b = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            call(a)
        with torch.cuda.stream(s2):
            call(b)
    torch.cuda.synchronize()
    five = torch.zeros(shape, device="cuda")
    for _ in range(5):
        five += want
    assert torch.equal(a, five) and torch.equal(b, five)
    g = torch.cuda.CUDAGraph()
    c = torch.zeros(shape, device="cuda")
    with torch.cuda.graph(g):
        o = call(c)
    c.zero_()
    g.replay()
    call(a)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, want + want) and torch.equal(o, out)


@pytest.mark.parametrize("kv", ["auto", "int4"])
def test_decode_runner_accumulates(kv):
    """Graph-replayed steps of two layers equal the same steps through the op, scores and cache rows included."""
    from glake_b200 import ops
    from glake_b200.backend import DecodeRunner, VTensorAttentionImpl, VTensorCacheEngine, VTensorMetadata
    gpu_util.ensure_pool()
    h, kvh, b = 8, 4, 3
    scales = [torch.full((kvh,), 0.01, device="cuda")] * 2 if kv == "int4" else None
    got = []
    for graph in (True, False):
        eng = VTensorCacheEngine(2, kvh, 128, b, 300, cache_dtype=kv)
        try:
            impl = VTensorAttentionImpl(h, 128, 0.1, kvh, kv)
            scores = eng.new_scores(256)
            rs = np.random.RandomState(3)
            runner = DecodeRunner(eng, impl, b, k_scale=scales, v_scale=scales, scores=scores) if graph else None
            outs = []
            for step in range(5):
                for s in eng.vmm_kvcache_segment:
                    s.ensure_mapped((step + 1) * eng.token_size)
                meta = VTensorMetadata(list(range(b)), [step + 1] * b, kvh, 128, num_decode_tokens=b)
                ins = [[normal_bf16(rs, b, x * 128).cuda() for x in (h, kvh, kvh)] for _ in range(2)]
                if graph:
                    for layer, (q, k, v) in enumerate(ins):
                        runner.q[layer].copy_(q), runner.k[layer].copy_(k), runner.v[layer].copy_(v)
                    torch.cuda.synchronize()
                    runner.step(meta)
                    runner.synchronize()
                    assert runner.status() == 0
                    outs.append(runner.out.clone())
                else:
                    from glake_b200.backend import prepare_step
                    prepare_step(meta, eng)
                    outs.append(torch.stack([impl.forward(q, k, v, *eng.gpu_cache[layer], meta, k_scale=scales[layer] if scales else None,
                                                          v_scale=scales[layer] if scales else None, scores=scores[layer])
                                             for layer, (q, k, v) in enumerate(ins)]))
                    torch.cuda.synchronize()
            got.append((torch.stack(outs), torch.stack(scores)))
            if graph:
                with pytest.raises(RuntimeError, match="scores hold 256"):
                    runner.step(VTensorMetadata([0, 1, 2], [257, 1, 1], kvh, 128, num_decode_tokens=3, set_used_size=[1, 1, 1]))
        finally:
            torch.cuda.synchronize()
            eng.close()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert bool(((got[0][1].sum((0, 2, 3)) - 5 * 2 * h).abs() < 1e-3).all())


def test_backend_scores_and_evicts():
    """A prompt scored by its window, decode steps that accumulate, an eviction that gives chunks back, and more steps:
    every layer follows the plain computation on its own list of rows."""
    from glake_b200 import vmmAllocator as A
    from glake_b200.backend import VTensorAttentionImpl, VTensorCacheEngine, VTensorMetadata, prepare_step
    gpu_util.ensure_pool()
    h, kvh, scale, layers, window = 8, 8, 128 ** -0.5, 2, 8
    rs = np.random.RandomState(11)
    rows_per_chunk = A.granularitySize // (kvh * 256)
    n0, budget = rows_per_chunk + 300, 200
    eng = VTensorCacheEngine(layers, kvh, 128, 3, 4 * rows_per_chunk)
    try:
        impl = VTensorAttentionImpl(h, 128, scale, kvh)
        scores = eng.new_scores()
        slot = 2
        mine = [{"k": None, "v": None, "s": None} for _ in range(layers)]
        length = 0

        def step(n):
            nonlocal length
            length += n
            meta = VTensorMetadata([slot], [length], kvh, 128, num_prefills=1 if n > 1 else 0, query_lens=[n] if n > 1 else None)
            prepare_step(meta, eng)
            for layer in range(layers):
                q, key, value = (normal_bf16(rs, n, x * 128) for x in (h, kvh, kvh))
                kc, vc = eng.gpu_cache[layer]
                impl.forward(q.cuda(), key.cuda(), value.cuda(), kc, vc, meta, scores=scores[layer], score_window=window)
                m = mine[layer]
                kd, vd = key.view(n, kvh, 128).double(), value.view(n, kvh, 128).double()
                m["k"] = kd if m["k"] is None else torch.cat([m["k"], kd])
                m["v"] = vd if m["v"] is None else torch.cat([m["v"], vd])
                w = torch.zeros(kvh, length, dtype=torch.float64)
                for j in range(min(window, n)):
                    end = length - min(window, n) + j + 1
                    w[:, :end] += U.attention64(q.view(n, h, 128)[n - min(window, n) + j], m["k"][:end], m["v"][:end], scale)[2]
                m["s"] = w if m["s"] is None else torch.cat([m["s"], torch.zeros(kvh, n, dtype=torch.float64)], -1) + w
                torch.cuda.synchronize()
                got = scores[layer][slot].cpu().double()
                assert bool(((got[:, :length] - m["s"]).abs() <= m["s"] * 1e-4 + 1e-9).all())
                assert float(got[:, length:].abs().max()) == 0
        step(n0)
        for _ in range(3):
            step(1)
        free = A.showFreeBlocks()
        (new_len,), kept = eng.evict(scores, [slot], [length], budget, sink=4, recent=16)
        assert new_len == budget and A.showFreeBlocks() == free + 2 * layers
        assert eng.vmm_kvcache_segment[slot].get_used_slot() == budget * eng.token_size
        for layer in range(layers):
            m, idx = mine[layer], kept[layer][0].cpu().long()
            for name in ("k", "v"):
                m[name] = torch.stack([m[name][idx[j], j] for j in range(kvh)], 1)
            m["s"] = torch.gather(m["s"], 1, idx)
            assert torch.equal(idx[:, :4], torch.arange(4).expand(kvh, 4))
            assert torch.equal(idx[:, -16:], torch.arange(length - 16, length).expand(kvh, 16))
        length = new_len
        for _ in range(3):
            step(1)
        (new_len,), _ = eng.evict(scores, [slot], [length], 1000)        # within the budget: nothing happens
        assert new_len == length == budget + 3
        step(1)
        with pytest.raises(RuntimeError, match="distinct"):
            eng.evict(scores, [slot, slot], [length, length], 10)
    finally:
        eng.close()
