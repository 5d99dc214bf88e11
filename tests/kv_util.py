"""Plain 64-bit forms of the quantised caches and of attention over them, and ranges in ordinary device memory."""
import math

import torch

D = 128


def unit(kvh):
    return next(u for u in (8, 4, 2, 1) if kvh % u == 0)


def row_bytes(kvh, kv):
    if kv == "int4":
        u = unit(kvh)
        return kvh // u * (64 * u + (4 * u + 15) // 16 * 16)
    return kvh * D * (1 if kv == "fp8_e4m3" else 2)


def _int4_places(kvh):
    """Byte of dim d and of its group's scale for every (head, dim), from the format's definition."""
    u = unit(kvh)
    ub = 64 * u + (4 * u + 15) // 16 * 16
    head, d = torch.arange(kvh)[:, None], torch.arange(D)[None, :]
    grp, r, j = d // 32, d % 32 // 4, d % 4
    base = head // u * ub
    return base + head % u * 64 + 8 * r + 2 * grp + j // 2, (j % 2).expand(kvh, D), base + 64 * u + head % u * 4 + grp


def quantise4(x, scale):
    """x [n, kvh, 128] -> (q in -7..7, s8) as float64, from the definition: its products and quotients are fp32 roundings
    (in 64 bits a quotient within 2^-24 of a tie, about one element in ten million, falls to the other side)."""
    n, kvh, _ = x.shape
    g = x.float().view(n, kvh, 4, 32)
    g = torch.where(torch.isnan(g), 0.0, g)
    t = g.abs().amax(-1) / (7.0 * scale)[:, None]
    s8 = t.clamp(max=448.0).to(torch.float8_e4m3fn).float()
    step = (s8 * scale[:, None])[..., None]
    q = torch.where(step > 0, torch.round(g / step), torch.zeros_like(g)).clamp(-7, 7)
    return q.view(n, kvh, D).double(), s8.double()


def pack4(x, scale):
    n, kvh, _ = x.shape
    q, s8 = quantise4(x, scale)
    at, hi, sc = (t.reshape(-1) for t in _int4_places(kvh))
    rows = torch.zeros(n, row_bytes(kvh, "int4"), dtype=torch.int64)
    rows.scatter_add_(1, at.expand(n, kvh * D), (q.long() + 8).view(n, kvh * D) * torch.where(hi == 1, 16, 1))
    rows[:, sc.view(kvh, 4, 32)[:, :, 0].reshape(-1)] = s8.float().to(torch.float8_e4m3fn).view(torch.uint8).long().view(n, kvh * 4)
    return rows.to(torch.uint8)


def unpack4(rows, kvh, scale):
    at, hi, sc = (t.reshape(-1) for t in _int4_places(kvh))
    b = rows.long()
    q = torch.where(hi == 1, b[:, at] // 16, b[:, at] % 16) - 8
    s8 = rows[:, sc].contiguous().view(torch.float8_e4m3fn).double()
    return (q * s8).view(-1, kvh, D) * scale.double()[:, None]


def encode(x, kv, scale):
    """bf16 rows [n, kvh, 128] on the CPU -> cache bytes [n, row bytes]."""
    n, kvh, _ = x.shape
    if n == 0:
        return torch.zeros(0, row_bytes(kvh, kv), dtype=torch.uint8)
    if kv == "int4":
        return pack4(x, scale)
    if kv == "fp8_e4m3":
        return (x.float() / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).view(n, row_bytes(kvh, kv))
    return x.contiguous().view(torch.uint8).view(n, row_bytes(kvh, kv))


def decode(rows, kv, kvh, scale):
    """Cache bytes [n, row bytes] on the CPU -> float64 [n, kvh, 128]."""
    if rows.shape[0] == 0:
        return torch.zeros(0, kvh, D, dtype=torch.float64)
    if kv == "int4":
        return unpack4(rows, kvh, scale)
    if kv == "fp8_e4m3":
        return rows.contiguous().view(torch.float8_e4m3fn).view(-1, kvh, D).double() * scale.double()[:, None]
    return rows.contiguous().view(torch.bfloat16).view(-1, kvh, D).double()


class Ranges:
    """K and V ranges of every slot in ordinary device memory, filled from per-sequence rows; ``cap`` rows per slot, all
    of them poisoned beyond the context (bytes 0xff: NaN as bf16 and as e4m3)."""

    def __init__(self, k_list, v_list, kv, k_scale=None, v_scale=None, spare_slots=2, extra=9, seed=0):
        self.kv, self.kvh = kv, k_list[0].shape[1]
        self.k_scale, self.v_scale = k_scale, v_scale
        self.lens = [k.shape[0] for k in k_list]
        b = len(self.lens)
        self.cap = max(self.lens) + extra
        self.row = row_bytes(self.kvh, kv)
        g = torch.Generator().manual_seed(seed)
        self.slots = torch.randperm(b + spare_slots, generator=g)[:b]
        host = {}
        for name, rows, scale in (("k", k_list, k_scale), ("v", v_list, v_scale)):
            t = torch.full((b + spare_slots, self.cap, self.row), 0xff, dtype=torch.uint8)
            for i, x in enumerate(rows):
                t[self.slots[i], :x.shape[0]] = encode(x, kv, scale)
            host[name] = t
        self.k, self.v = host["k"].cuda(), host["v"].cuda()
        dev = lambda t: torch.tensor(t, dtype=torch.int64).cuda()  # noqa: E731
        self.k_table = dev([self.k[i].data_ptr() for i in range(self.k.shape[0])])
        self.v_table = dev([self.v[i].data_ptr() for i in range(self.v.shape[0])])
        self.slot_ids = self.slots.to(torch.int64).cuda()
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.max_len = max(max(self.lens), 1)

    def quant(self):
        if self.kv == "bf16":
            return {}
        return {"kv_cache_dtype": self.kv, "k_scale": self.k_scale.cuda(), "v_scale": self.v_scale.cuda()}

    def rows64(self, name, i, n=None):
        n = self.lens[i] if n is None else n
        rows = getattr(self, name)[self.slots[i], :n].cpu()
        return decode(rows, self.kv, self.kvh, self.k_scale if name == "k" else self.v_scale)


def attention64(q, k, v, scale):
    """q [h, 128], k / v float64 [n, kvh, 128] -> out [h, 128], lse [h], weights summed over a group's heads [kvh, n],
    sum p |v| [h, 128]."""
    h, kvh = q.shape[0], k.shape[1]
    if k.shape[0] == 0:
        z = torch.zeros(h, D, dtype=torch.float64)
        return z, torch.full((h,), -math.inf, dtype=torch.float64), torch.zeros(kvh, 0, dtype=torch.float64), z
    x = torch.einsum("kgd,nkd->kgn", q.double().view(kvh, h // kvh, D), k) * scale
    p = torch.softmax(x, -1)
    return (torch.einsum("kgn,nkd->kgd", p, v).reshape(h, D), torch.logsumexp(x, -1).reshape(h), p.sum(1),
            torch.einsum("kgn,nkd->kgd", p, v.abs()).reshape(h, D))


def logit_error(q, k, scale, kv):
    """Bound of an fp32-accumulated logit's error: every product and partial sum is off by at most a few steps of 2^-23
    of the sum of magnitudes (a nibble enters as up to 15 with an offset of 8: at most 2 x 16 / 7 of the value's range)."""
    kvh = k.shape[1]
    if k.shape[0] == 0:
        return 0.0
    mag = torch.einsum("kgd,kd->kg", q.double().abs().view(kvh, -1, D), k.abs().amax(0)).amax().item()
    return 2.0 ** -20 * scale * mag * (5.0 if kv == "int4" else 1.0) + 2.0 ** -20
