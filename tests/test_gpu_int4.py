"""The 4-bit KV cache on the GPU: append, read-back, decode attention (split and fused), prompt attention, engine."""
import math

import pytest
import torch

from tests import gpu_util, kv_util as U
from tests.synth import normal_bf16

import numpy as np

pytestmark = pytest.mark.gpu


def scales_of(rows, kvh):
    x = torch.cat([r for r in rows if r.shape[0]]).float().abs().amax((0, 2))
    return (x / 448.0 * 0.97).contiguous()


def make(seed, lens, kvh):
    rs = np.random.RandomState(seed)
    k = [normal_bf16(rs, n, kvh, 128) for n in lens]
    v = [normal_bf16(rs, n, kvh, 128) for n in lens]
    return k, v, scales_of(k, kvh), scales_of(v, kvh), rs


def v_step(r, i, h):
    """Largest step of a head's stored V values, per q head [h, 1]."""
    if r.lens[i] == 0:
        return 0.0
    _, s8 = parts(r.v[r.slots[i], :r.lens[i]].cpu(), r.kvh)
    return (s8.amax((0, 2)).double() * r.v_scale.double()).repeat_interleave(h // r.kvh)[:, None]


def check_attention(r, q, out, lse, scale, k_rows=None):
    """out within its roundings of the 64-bit result over the stored values: bf16 output (2^-8 of the value), P in f16
    twice (2 x 2^-11 of the weighted magnitudes), logits in fp32, and the sums of the nibbles as f16 subnormals: u 2^-24
    enters the tensor core's 24-bit sum with the exponent 2^-14 of its format, 10 places above its own, so a product is
    cut at 2^-23 x 2^10 p s = 2^-13 p s at worst, and the weights p sum to 1: 2^-13 of the largest step (also where all
    stored values are 0, since a zero is the nibble 8 and its offset)."""
    for i in range(len(r.lens)):
        k, v = r.rows64("k", i), r.rows64("v", i)
        want, want_lse, _, mag = U.attention64(q[i], k, v, scale)
        e = U.logit_error(q[i], k, scale, r.kv)
        tol = want.abs() * 2.0 ** -8 + mag * (2.0 ** -10 + 2 * e) + v_step(r, i, q.shape[1]) * 2.0 ** -13
        assert bool(((out[i].double() - want).abs() <= tol).all()), (i, r.lens[i], float((out[i].double() - want).abs().max()))
        if lse is not None:
            if r.lens[i] == 0:
                assert bool((lse[i] == -math.inf).all())
            else:
                assert bool(((lse[i].double() - want_lse).abs() <= e + want_lse.abs() * 2.0 ** -22).all())


# every unit width (8, 4, 2, 1), several units, odd head counts; contexts at the 16-token steps and tile edges
@pytest.mark.parametrize("h,kvh", [(8, 8), (32, 8), (64, 8), (16, 1), (8, 1), (4, 2), (16, 4), (32, 32), (6, 3), (12, 12), (32, 2)])
def test_decode_attention(h, kvh):
    from glake_b200 import ops
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 255, 257, 511, 1000]
    k, v, ks, vs, rs = make(h * 100 + kvh, lens, kvh)
    r = U.Ranges(k, v, "int4", ks, vs)
    q = (normal_bf16(rs, len(lens), h, 128).float() * 1.5).bfloat16()
    scale = 128 ** -0.5
    out, lse = ops.fwd_kvcache(q.cuda().unsqueeze(1), r.k_table.data_ptr(), r.v_table.data_ptr(), r.max_len, kvh, len(lens),
                               r.slot_ids, None, None, r.seq_lens, None, None, None, None, None, None, scale, True, -1, -1,
                               None, 0, **r.quant())
    torch.cuda.synchronize()
    assert ops.attn_status() == 0
    check_attention(r, q, out[:, 0].cpu(), lse[..., 0].cpu(), scale)


@pytest.mark.parametrize("h,kvh,batch,hi", [(32, 8, 3, 20000), (8, 1, 2, 30000), (8, 8, 300, 40), (8, 1, 1100, 90)])
def test_decode_attention_long_and_many(h, kvh, batch, hi):
    """Streams cut over many CTAs, and batches beyond the address cache (256) and the schedule's table (1024)."""
    from glake_b200 import ops
    rs = np.random.RandomState(hi)
    lens = [int(x) for x in rs.randint(0 if batch > 10 else hi // 2, hi + 1, size=batch)]
    k, v, ks, vs, rs = make(batch, lens, kvh)
    r = U.Ranges(k, v, "int4", ks, vs)
    q = normal_bf16(rs, batch, h, 128)
    out = torch.empty(batch, h, 128, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention_v1(out, q.cuda(), r.k_table.data_ptr(), r.v_table.data_ptr(), kvh, 128 ** -0.5, r.seq_lens, 1, r.max_len,
                           None, "int4", 1.0, r.slot_ids, k_scale=ks.cuda(), v_scale=vs.cuda())
    torch.cuda.synchronize()
    assert ops.attn_status() == 0
    check_attention(r, q, out.cpu(), None, 128 ** -0.5)


def test_more_pieces_than_a_share_lists_at_once():
    """A thousand contexts of 1 to 5 rows over 128 kv heads: about 54 one-tile streams per CTA."""
    from glake_b200 import ops
    h = kvh = 128
    rs = np.random.RandomState(0)
    lens = [int(x) for x in rs.randint(1, 6, size=1000)]
    k, v, ks, vs, rs = make(1, lens, kvh)
    r = U.Ranges(k, v, "int4", ks, vs)
    q = normal_bf16(rs, len(lens), h, 128)
    out = torch.empty(len(lens), h, 128, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention_v1(out, q.cuda(), r.k_table.data_ptr(), r.v_table.data_ptr(), kvh, 128 ** -0.5, r.seq_lens, 1, r.max_len,
                           None, "int4", 1.0, r.slot_ids, k_scale=ks.cuda(), v_scale=vs.cuda())
    torch.cuda.synchronize()
    assert ops.attn_status() == 0
    for i in range(0, len(lens), 7):
        kk, vv = r.rows64("k", i), r.rows64("v", i)
        want, _, _, mag = U.attention64(q[i], kk, vv, 128 ** -0.5)
        e = U.logit_error(q[i], kk, 128 ** -0.5, "int4")
        tol = want.abs() * 2.0 ** -8 + mag * (2.0 ** -10 + 2 * e) + v_step(r, i, h) * 2.0 ** -13
        assert bool(((out[i].cpu().double() - want).abs() <= tol).all())


def test_small_and_large_magnitudes():
    """Queries far from 1, values whose scales differ by 2^60 between heads, one-sided logits of several hundred."""
    from glake_b200 import ops
    lens, h, kvh = [40, 333], 16, 8
    k, v, _, _, rs = make(7, lens, kvh)
    mag = 2.0 ** torch.linspace(-30, 30, kvh)
    k = [(x.float() / mag[:, None]).bfloat16() for x in k]
    v = [(x.float() * mag[:, None]).bfloat16() for x in v]
    ks, vs = scales_of(k, kvh), scales_of(v, kvh)
    r = U.Ranges(k, v, "int4", ks, vs)
    q = (normal_bf16(rs, 2, h, 128).float().view(2, kvh, 2, 128) * mag[:, None, None] * 20).bfloat16().view(2, h, 128)
    out = torch.empty(2, h, 128, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention_v1(out, q.cuda(), r.k_table.data_ptr(), r.v_table.data_ptr(), kvh, 128 ** -0.5, r.seq_lens, 1, r.max_len,
                           None, "int4", 1.0, r.slot_ids, k_scale=ks.cuda(), v_scale=vs.cuda())
    torch.cuda.synchronize()
    check_attention(r, q, out.cpu(), None, 128 ** -0.5)


@pytest.mark.parametrize("kvh", [8, 16, 4, 2, 1, 3])
@pytest.mark.parametrize("offset", [0, 1])
def test_append_and_read_back(kvh, offset):
    """Cache bytes equal the definition's; rows behind the appended ones and entries with a negative offset stay as they
    were; read-back equals the stored values rounded once.  ``offset`` shifts the inputs off their 8-byte alignment."""
    from glake_b200 import ops
    rows, prefix = [5, 1, 0, 33], [0, 7, 3, 16]
    rs = np.random.RandomState(kvh)
    total = sum(rows)
    key, value = normal_bf16(rs, total, kvh, 128), normal_bf16(rs, total, kvh, 128)
    key[0, 0, 3], key[0, 0, 40], key[1, 0, 70], value[2, 0, 5] = math.nan, math.inf, 0.0, -math.inf
    key[3] = 0
    key[4, 0] *= 0.001
    g = torch.Generator().manual_seed(kvh)
    ks, vs = (torch.rand(kvh, generator=g) * 0.004 + 0.004 for _ in range(2))
    empty = [torch.zeros(n + p, kvh, 128, dtype=torch.bfloat16) for n, p in zip(rows, prefix)]
    r = U.Ranges(empty, empty, "int4", ks, vs, extra=3)
    before = {n: getattr(r, n).cpu().clone() for n in ("k", "v")}

    def dev(x):   # a view whose rows start `offset` elements into a wider buffer
        wide = kvh * 128 + 8
        view = torch.empty(total * wide + 8, dtype=torch.bfloat16, device="cuda").as_strided((total, kvh, 128), (wide, 128, 1), offset)
        view.copy_(x.cuda())
        return view
    slot_m = torch.tensor([p * r.row for p in prefix])
    starts = torch.tensor([sum(rows[:i]) for i in range(4)], dtype=torch.int32)
    ops.reshape_and_cache(dev(key), dev(value), r.k_table, r.v_table, slot_m.cuda(), r.slot_ids, torch.tensor(rows, dtype=torch.int32).cuda(),
                          starts.cuda(), max(rows), kvh, 128, "int4", ks.cuda(), vs.cuda())
    torch.cuda.synchronize()
    pad = torch.ones(r.row, dtype=torch.bool)
    u = U.unit(kvh)
    pad.view(kvh // u, -1)[:, 68 * u:] = False       # padding bytes are not part of the format
    for name, x, scale in (("k", key, ks), ("v", value, vs)):
        now, want = getattr(r, name).cpu(), before[name].clone()
        packed = U.pack4(x, scale)
        for i in range(4):
            want[r.slots[i], prefix[i]:prefix[i] + rows[i]] = packed[int(starts[i]):int(starts[i]) + rows[i]]
        assert torch.equal(now[..., pad], want[..., pad])
        assert torch.equal(now[..., ~pad], before[name][..., ~pad])
    # decode form: one row per entry, a skipped entry among them
    one = normal_bf16(rs, 4, kvh, 128)
    m = torch.tensor([p * r.row for p in prefix])
    m[1] = -1
    before = r.k.cpu().clone()
    ops.reshape_and_cache(one.cuda(), one.cuda(), r.k_table, r.v_table, m.cuda(), r.slot_ids, None, None, 1, kvh, 128, "int4", ks.cuda(), vs.cuda())
    torch.cuda.synchronize()
    for i in (0, 2, 3):
        before[r.slots[i], prefix[i]] = torch.where(pad, U.pack4(one, ks)[i], before[r.slots[i], prefix[i]])
    assert torch.equal(r.k.cpu(), before)
    # read-back, K alone and both
    lens = [n + p for n, p in zip(rows, prefix)]
    at = [sum(lens[:i]) + i for i in range(4)]
    ko = torch.full((sum(lens) + 5, kvh, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    vo = ko.clone()
    args = (r.k_table.data_ptr(), r.v_table.data_ptr(), kvh, r.slot_ids, r.seq_lens, torch.tensor(at, dtype=torch.int32).cuda(), max(lens))
    ops.dequantize_ranges(ko, vo, *args, **r.quant())
    k2 = torch.full_like(ko, 3.0)
    ops.dequantize_ranges(k2, None, *args, **r.quant())
    torch.cuda.synchronize()
    assert torch.equal(k2, ko)
    want = torch.full(ko.shape, 3.0, dtype=torch.bfloat16)
    for i in range(4):   # (nibble * e4m3) is exact, the product with the scale is an fp32 rounding, then one to bf16
        q, s8 = (t.float() for t in parts(r.k[r.slots[i], :lens[i]].cpu(), kvh))
        want[at[i]:at[i] + lens[i]] = (q * s8 * ks[:, None]).bfloat16()
    assert torch.equal(ko.cpu(), want)


def parts(rows, kvh):
    one = torch.ones(kvh)
    at, hi, sc = (t.reshape(-1) for t in U._int4_places(kvh))
    s8 = rows[:, sc].contiguous().view(torch.float8_e4m3fn).float().view(-1, kvh, 128)
    q = torch.where(hi == 1, rows.long()[:, at] // 16, rows.long()[:, at] % 16).view(-1, kvh, 128) - 8
    return q, s8 * one[:, None]


def test_read_back_of_an_fp8_cache():
    from glake_b200 import ops
    kvh, lens = 3, [5, 40]
    k, v, ks, vs, _ = make(3, lens, kvh)
    r = U.Ranges(k, v, "fp8_e4m3", ks, vs)
    ko = torch.empty(45, kvh, 128, dtype=torch.bfloat16, device="cuda")
    vo = torch.empty_like(ko)
    ops.dequantize_ranges(ko, vo, r.k_table.data_ptr(), r.v_table.data_ptr(), kvh, r.slot_ids, r.seq_lens,
                          torch.tensor([0, 5], dtype=torch.int32).cuda(), 40, **r.quant())
    for i, at in enumerate((0, 5)):
        rows = r.v[r.slots[i], :lens[i]].cpu().view(torch.float8_e4m3fn).float().view(-1, kvh, 128)
        assert torch.equal(vo[at:at + lens[i]].cpu(), (rows * vs[:, None]).bfloat16())


@pytest.mark.parametrize("h,kvh", [(32, 8), (8, 1), (16, 2), (16, 16), (6, 3), (16, 4), (16, 1)])
def test_fused_steps(h, kvh):
    """Three fused steps: the rows written equal a separate append's, the attention sees them, padded entries (negative
    offset) attend without appending."""
    from glake_b200 import ops
    lens = [1, 15, 16, 17, 32, 64, 200, 1025]
    k, v, ks, vs, rs = make(h + kvh, lens, kvh)
    r = U.Ranges([x[:-1] for x in k], [x[:-1] for x in v], "int4", ks, vs)
    scale = 128 ** -0.5
    for step in range(3):
        grown = [n + step for n in lens]
        skip = 2 if step == 1 else None
        key, value, q = (normal_bf16(rs, len(lens), n, 128) for n in (kvh, kvh, h))
        off = torch.tensor([(n - 1) * r.row for n in grown])
        if skip is not None:
            off[skip] = -1
        r.lens = grown
        r.seq_lens = torch.tensor(grown, dtype=torch.int32).cuda()
        before = r.k.cpu().clone()
        out = torch.empty(len(lens), h, 128, dtype=torch.bfloat16, device="cuda")
        ops.decode_step(out, q.cuda(), key.cuda(), value.cuda(), r.k_table.data_ptr(), r.v_table.data_ptr(), off.cuda(), r.slot_ids,
                        r.seq_lens, max(grown), kvh, scale, "int4", ks.cuda(), vs.cuda())
        torch.cuda.synchronize()
        packed, u = U.pack4(key, ks), U.unit(kvh)
        pad = torch.ones(r.row, dtype=torch.bool)
        pad.view(kvh // u, -1)[:, 68 * u:] = False
        for i, n in enumerate(grown):
            if i != skip:
                before[r.slots[i], n - 1] = torch.where(pad, packed[i], before[r.slots[i], n - 1])
        assert torch.equal(r.k.cpu(), before)
        if skip is not None:   # its last row is the poison the range was made with: give it a row for the next step
            r.k[r.slots[skip], grown[skip] - 1] = packed[skip].cuda()
            r.v[r.slots[skip], grown[skip] - 1] = U.pack4(value, vs)[skip].cuda()
            keep = [i for i in range(len(lens)) if i != skip]
        else:
            keep = list(range(len(lens)))
        o = out.cpu()
        for i in keep:
            want, _, _, mag = U.attention64(q[i], r.rows64("k", i), r.rows64("v", i), scale)
            e = U.logit_error(q[i], r.rows64("k", i), scale, "int4")
            tol = want.abs() * 2.0 ** -8 + mag * (2.0 ** -10 + 2 * e) + v_step(r, i, h) * 2.0 ** -13
            assert bool(((o[i].double() - want).abs() <= tol).all())


def test_steps_over_one_clean_workspace():
    """One zero-filled workspace for steps of different batch sizes, one of them beyond the schedule's table: every call
    finds its counters clean (same result, bit for bit, as with a buffer that is cleared for the call)."""
    from glake_b200 import ops
    h, kvh = 8, 2
    lens = [2600, 1300] + [1 + 7 * i % 90 for i in range(1028)]
    k, v, ks, vs, rs = make(5, lens, kvh)
    r = U.Ranges([x[:-1] for x in k], [x[:-1] for x in v], "int4", ks, vs)
    ws = ops.new_workspace(torch.device("cuda"), len(lens), h, 128, max(lens))
    key, value, q = (normal_bf16(rs, len(lens), n, 128).cuda() for n in (kvh, kvh, h))
    off = torch.tensor([(n - 1) * r.row for n in lens]).cuda()
    seq_lens = torch.tensor(lens, dtype=torch.int32).cuda()

    def step(n, **how):
        out = torch.zeros(n, h, 128, dtype=torch.bfloat16, device="cuda")
        ops.decode_step(out, q[:n], key[:n], value[:n], r.k_table.data_ptr(), r.v_table.data_ptr(), off[:n], r.slot_ids[:n],
                        seq_lens[:n], max(lens), kvh, 128 ** -0.5, "int4", ks.cuda(), vs.cuda(), **how)
        return out.cpu()

    for n in (1, len(lens), 2, len(lens), len(lens), 40):
        assert torch.equal(step(n, workspace=ws, clean_scratch=True), step(n))


def test_captured_and_replayed_on_another_stream():
    from glake_b200 import ops
    lens, h, kvh = [700, 33], 32, 8
    k, v, ks, vs, rs = make(5, lens, kvh)
    r = U.Ranges(k, v, "int4", ks, vs)
    q = normal_bf16(rs, 2, h, 128).cuda()
    out = torch.zeros(2, h, 128, dtype=torch.bfloat16, device="cuda")
    ws = ops.new_workspace(q.device, 2, h, 128, r.max_len)
    dks, dvs = ks.cuda(), vs.cuda()
    key = torch.zeros(2, kvh, 128, dtype=torch.bfloat16, device="cuda")
    off = torch.full((2,), -1, dtype=torch.int64, device="cuda")

    def call():
        ops.decode_step(out, q, key, key, r.k_table.data_ptr(), r.v_table.data_ptr(), off, r.slot_ids, r.seq_lens, r.max_len, kvh,
                        128 ** -0.5, "int4", dks, dvs, workspace=ws, clean_scratch=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        first = out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
        out.zero_()
        g.replay()
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out)
    check_attention(r, q.cpu(), out.cpu(), None, 128 ** -0.5)


@pytest.mark.parametrize("neox,rot", [(True, 128), (False, 128), (True, 64), (False, 32), (True, 16)])
@pytest.mark.parametrize("h,kvh", [(8, 2), (4, 4), (16, 8), (3, 3)])
@pytest.mark.parametrize("write_key", [False, True])
def test_rope_append(neox, rot, h, kvh, write_key):
    """One launch equals the rotation (bf16 cache, key written back) followed by the 4-bit append of the rotated key."""
    from glake_b200 import ops
    rs = np.random.RandomState(rot + h)
    lens, n = [5, 1, 0, 33], 39
    q, k, v = (normal_bf16(rs, n, x * 128).cuda() for x in (h, kvh, kvh))
    pos = torch.from_numpy(rs.randint(0, 300, size=n)).cuda()
    freq = torch.outer(torch.arange(300.0), 1.0 / 10000.0 ** (torch.arange(0, rot, 2) / rot))
    cs = torch.cat([freq.cos(), freq.sin()], -1).bfloat16().cuda()
    g = torch.Generator().manual_seed(rot + kvh)
    ks, vs = (torch.rand(kvh, generator=g) * 0.004 + 0.006 for _ in range(2))
    empty = [torch.zeros(x, kvh, 128, dtype=torch.bfloat16) for x in lens]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    starts, zero = i32([0, 5, 6, 6]), torch.zeros(4, dtype=torch.int64, device="cuda")
    plain = U.Ranges(empty, empty, "bf16")
    q0, k0 = q.clone(), k.clone()
    ops.rotary_embedding_and_cache(pos, q0, k0, v, 128, cs, neox, plain.k_table, plain.v_table, zero, plain.slot_ids, i32(lens), starts, 33,
                                   kvh, write_key=True)
    r = U.Ranges(empty, empty, "int4", ks, vs)
    before = r.k.clone()
    q1, k1 = q.clone(), k.clone()
    off = zero.clone()
    off[1] = -1            # rotated, not appended
    ops.rotary_embedding_and_cache(pos, q1, k1, v, 128, cs, neox, r.k_table, r.v_table, off, r.slot_ids, i32(lens), starts, 33, kvh, "int4",
                                   ks.cuda(), vs.cuda(), write_key=write_key)
    torch.cuda.synchronize()
    assert torch.equal(q1, q0) and torch.equal(k1, k0 if write_key else k)
    at = 0
    for i, m in enumerate(lens):
        for name, x, scale in (("k", k0, ks), ("v", v, vs)):
            got = U.unpack4(getattr(r, name)[r.slots[i], :m].cpu(), kvh, scale)
            want = U.unpack4(U.pack4(x[at:at + m].cpu().view(m, kvh, 128), scale), kvh, scale)
            if i == 1:
                assert torch.equal(getattr(r, name)[r.slots[i]], before[r.slots[i]])
            else:
                assert torch.equal(got, want)
        assert bool((r.k[r.slots[i], m:] == 0xff).all())
        at += m


def test_backend_prompt_extend_and_decode():
    """Prompt, prefix-extend and decode through the engine's own ranges and VTensorAttentionImpl, two layers."""
    from glake_b200.backend import VTensorAttentionImpl, VTensorCacheEngine, VTensorMetadata, prepare_step
    gpu_util.ensure_pool()
    h, kvh, scale = 8, 2, 128 ** -0.5
    rs = np.random.RandomState(11)
    eng = VTensorCacheEngine(2, kvh, 128, 3, 600, cache_dtype="int4")
    try:
        impl = VTensorAttentionImpl(h, 128, scale, kvh, "int4")
        ks, vs = torch.tensor([0.009, 0.0111]), torch.tensor([0.0105, 0.0093])
        hist = {0: [], 1: []}
        slots, have = [2, 0], [0, 0]
        for rows in ([130, 17], [40, 90], [1, 1], [1, 1]):
            now = [a + b for a, b in zip(have, rows)]
            prompt = rows[0] > 1
            meta = VTensorMetadata(slots, now, kvh, 128, num_prefills=2 if prompt else 0, query_lens=rows if prompt else None,
                                   num_decode_tokens=0 if prompt else 2)
            prepare_step(meta, eng)
            for layer in range(2):
                n = sum(rows)
                q, key, value = normal_bf16(rs, n, h * 128), normal_bf16(rs, n, kvh * 128), normal_bf16(rs, n, kvh * 128)
                hist[layer].append((rows, key.view(n, kvh, 128), value.view(n, kvh, 128)))
                kc, vc = eng.gpu_cache[layer]
                out = impl.forward(q.cuda(), key.cuda(), value.cuda(), kc, vc, meta, k_scale=ks.cuda(), v_scale=vs.cuda())
                torch.cuda.synchronize()
                out = out.cpu().view(n, h, 128)
                at = 0
                for i in range(2):
                    kk, vv = [], []
                    for rr, a, b in hist[layer]:
                        s0 = sum(rr[:i])
                        kk.append(a[s0:s0 + rr[i]])
                        vv.append(b[s0:s0 + rr[i]])
                    kd = U.unpack4(U.pack4(torch.cat(kk), ks), kvh, ks)
                    vd = U.unpack4(U.pack4(torch.cat(vv), vs), kvh, vs)
                    if prompt:   # the prompt kernels run on the rows widened to bf16
                        kd, vd = kd.bfloat16().double(), vd.bfloat16().double()
                    for j in range(rows[i]):
                        qi = q.view(n, h, 128)[at + j]
                        end = have[i] + j + 1
                        want, _, _, mag = U.attention64(qi, kd[:end], vd[:end], scale)
                        # prompt kernels: P to 16 bits; decode: P in f16 twice, sums of nibbles (check_attention; a
                        # step is at most 64 x 0.011 here)
                        tol = want.abs() * 2.0 ** -8 + mag * (2.0 ** -10 + 2.0 ** -13) + 0.75 * 2.0 ** -13
                        assert bool(((out[at + j].double() - want).abs() <= tol).all()), (layer, rows, i, j)
                    at += rows[i]
            have = now
    finally:
        eng.close()
