"""Cases for the operators beside the tracker's own: attention with a learned relative position bias by buckets, the
largest logits of a row with their places, and the distillation loss against a teacher's largest logits.

`listed()` are the cases that are timed, `draw(rng)` gives more of the same ranges.  `run` computes a case either in
plain torch operations in 32 bits, rounded once at the end, or (`own`) through the framework's entry points; `exact`
computes it in 64 bits.

A key's position is its index; query i of a sequence stands at position offset + i.  Buckets of a sequence: an offset of
n places has bucket n up to half the buckets, then buckets whose borders grow geometrically up to `span`; both directions
have a half each unless the attention is causal.  Buckets of a map of `width` columns: one per (row offset, column offset).
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one frame's template tokens (16 x 16 map, 8 heads of 32 channels): the online tracker's call, all latency
        _att("map16_f32", "attend", "f32", 1, 256, 256, 8, 8, 32, width=16),
        # the search stream of a training step of 40 pairs (32 x 32 map), forward and backward, exact fp32 products
        _att("map32_train_f32", "attend_train", "f32", 40, 1024, 1024, 8, 8, 32, width=32),
        # causal training in bf16 on padded sequences of an odd length, four query heads to a key/value head
        _att("causal_train_bf16", "attend_train", "bf16", 8, 1999, 1999, 16, 4, 64, causal=True, ragged=True),
        # one long sequence without padding, forward only (scoring), heads of 128 channels
        _att("long_f16", "attend", "f16", 1, 8191, 8191, 8, 8, 128),
        # one new token over a short cache: the smallest step of generation
        _att("token_f16", "token", "f16", 1, 1, 257, 8, 8, 64, causal=True),
        # one new token for each of 32 sequences over long caches of different lengths
        _att("token_batch_bf16", "token", "bf16", 32, 1, 16384, 32, 8, 128, causal=True, ragged=True),
        # the teacher's score maps of a batch: the best 16 of 1024 places per clip
        _row("top_map_f32", "top", "f32", 32, 1024, 16),
        # a teacher's answers to 4096 tokens: the best 64 of 32000
        _row("top_bf16", "top", "bf16", 4096, 32000, 64),
        # three rows of an odd, large width: a row has to be cut to fill the card
        _row("top_few_f16", "top", "f16", 3, 100003, 8),
        # the student's score maps against the teacher's best 16 places, loss and gradient
        _row("distill_map_f32", "distill", "f32", 32, 1024, 16),
        # a training step's 4096 tokens at an odd width
        _row("distill_bf16", "distill", "bf16", 4096, 50257, 64),
        # few rows of an odd, large width
        _row("distill_few_f16", "distill", "f16", 5, 131073, 128),
    ]


def _att(name, kind, dtype, B, Lq, Lk, H, Hkv, D, width=0, causal=False, ragged=False):
    return {"name": name, "kind": kind, "type": dtype, "B": B, "Lq": Lq, "Lk": Lk, "H": H, "Hkv": Hkv, "D": D, "width": width,
            "causal": causal, "ragged": ragged}


def _row(name, kind, dtype, N, V, k):
    return {"name": name, "kind": kind, "type": dtype, "N": N, "V": V, "k": k}


def draw(rng):
    log = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))  # noqa: E731
    largest = {k: max((work(c) for c in listed() if c["kind"] == k), key=lambda w: w["bytes"] + w["flops"] / 50) for k in
               ("attend", "attend_train", "token", "top", "distill")}
    while True:
        kind = rng.choice(("attend", "attend", "attend_train", "attend_train", "token", "top", "distill"))
        dtype = rng.choice(("f32", "bf16", "f16"))
        if kind in ("attend", "attend_train"):
            Hkv, D = rng.choice((1, 2, 4, 8)), rng.choice((32, 64, 128))
            width = rng.randint(4, 40) if rng.random() < 0.5 else 0
            L = width * rng.randint(4, 40) if width else log(1, 4096)
            c = _att("", kind, dtype, log(1, 40), L, L, Hkv * rng.choice((1, 2, 4)), Hkv, D, width=width,
                     causal=not width and rng.random() < 0.5, ragged=rng.random() < 0.5)
            if c["B"] * c["H"] * L * L > 1 << 29:
                continue
        elif kind == "token":
            Hkv = rng.choice((1, 2, 4, 8))
            c = _att("", kind, dtype, log(1, 32), rng.choice((1, 1, 1, 2, 4)), log(8, 16384), Hkv * rng.choice((1, 2, 4, 8)), Hkv,
                     rng.choice((32, 64, 128)), causal=True, ragged=rng.random() < 0.5)
        else:
            V = log(128, 131072)
            c = _row("", kind, dtype, log(1, 4096), V, min(V, log(1, 128)))
        del c["name"]
        w, most = work(c), largest[kind]
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def _lengths(c):
    """Valid keys of each sequence: all of them, or lengths between a quarter less and all."""
    B, Lk = c["B"], c["Lk"]
    return [max(min(c["Lq"], Lk), Lk - (b * 37 * Lk // 128) % (Lk // 4 + 1)) for b in range(B)] if c["ragged"] else [Lk] * B


def work(c):
    size = _SIZE[c["type"]]
    if "V" in c:
        N, V, k = c["N"], c["V"], c["k"]
        if c["kind"] == "top":
            return {"bytes": N * V * size + N * k * (size + 4), "flops": N * V}
        return {"bytes": 2 * N * V * size + N * k * (size + 4) + 8 * N, "flops": 8 * N * V}
    B, Lq, Lk, H, Hkv, D = (c[x] for x in ("B", "Lq", "Lk", "H", "Hkv", "D"))
    pairs = keys = 0
    for n in _lengths(c):
        first = n - Lq if c["kind"] == "token" else 0
        pairs += sum(min(n, first + i + 1) for i in range(Lq)) if c["causal"] else Lq * n
        keys += n
    rows, heads = 2 * B * Lq * H * D, 2 * keys * Hkv * D
    if c["kind"] == "attend_train":                   # q, k, v and the gradient of out read; out and four gradients written
        return {"bytes": (2 * rows + 2 * heads) * size + 4 * _num_buckets(c) * H, "flops": 14 * pairs * H * D}
    return {"bytes": (rows + heads) * size + 2 * _num_buckets(c) * H, "flops": 4 * pairs * H * D}


_BUCKETS, _SPAN = 32, 128


def _num_buckets(c):
    return (2 * (c["Lk"] // c["width"]) - 1) * (2 * c["width"] - 1) if c["width"] else _BUCKETS


def _bucket_of_offset(c):
    """The bucket of every offset key - query from -(Lk - 1) to Lk - 1 of a sequence: whole numbers throughout, so that no
    rounding decides at a border."""
    n = torch.arange(c["Lk"])
    buckets = _BUCKETS if c["causal"] else _BUCKETS // 2
    exact_ = buckets // 2
    logs = buckets - exact_
    borders = []
    for j in range(1, logs):
        x = exact_
        while x ** logs * exact_ ** j < _SPAN ** j * exact_ ** logs:
            x += 1
        borders.append(x)
    near = torch.where(n < exact_, n, exact_ + torch.bucketize(n, torch.tensor(borders), right=True))
    ahead = torch.zeros_like(n) if c["causal"] else near + buckets
    return torch.cat([near.flip(0), ahead[1:]])


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[c["type"]]
    rand = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)  # noqa: E731
    s = {"case": dict(c)}
    if "V" in c:
        N, V, k = c["N"], c["V"], c["k"]
        # logits of a trained model: a broad floor and a few outstanding entries
        teacher = torch.randn(N, V, generator=g, device="cuda")
        teacher = teacher * 1.5 + 6.0 * (torch.rand(N, V, generator=g, device="cuda") < 8.0 / V)
        if c["kind"] == "top":
            s["logits"] = teacher.to(dtype)
        else:
            s["student"] = (teacher + torch.randn(N, V, generator=g, device="cuda")).to(dtype).requires_grad_(own)
            values, at = torch.topk(teacher, k, dim=1)
            s["values"], s["indices"] = values.to(dtype), at.to(torch.int32)
            s["grad"] = torch.rand(N, generator=g, device="cuda") / N
            s["temperature"] = 2.0
        return s
    B, Lq, Lk, H, Hkv, D = (c[x] for x in ("B", "Lq", "Lk", "H", "Hkv", "D"))
    s["q"], s["k"], s["v"] = rand(B, Lq, H, D), rand(B, Lk, Hkv, D), rand(B, Lk, Hkv, D)
    s["table"] = rand(_num_buckets(c), H, scale=0.5)
    s["kv_len"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
    if c["kind"] == "attend_train":
        s["grad"] = rand(B, Lq, H, D)
        for x in ("q", "k", "v", "table"):
            s[x].requires_grad_(own)
    if own:
        from spot_amd import ops
        s["buckets"] = (ops.grid_buckets(Lk // c["width"], c["width"], device="cuda") if c["width"] else
                        ops.sequence_buckets(Lk, _BUCKETS, _SPAN, bidirectional=not c["causal"], device="cuda"))
    else:
        s["offsets"] = None if c["width"] else _bucket_of_offset(c).cuda()
    return s


def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        from spot_amd import ops
        if kind == "top":
            return ops.top_logits(s["logits"], c["k"])
        if kind == "distill":
            loss = ops.top_logit_distillation(s["student"], s["values"], s["indices"], s["temperature"])
            return (loss,) + torch.autograd.grad(loss, (s["student"],), s["grad"])
        out = ops.bias_attention(s["q"], s["k"], s["v"], s["table"], s["buckets"], causal=c["causal"],
                                 q_offset="end" if kind == "token" else 0, kv_len=s["kv_len"])
        if kind == "attend_train":
            return (out,) + torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["table"]), s["grad"])
        return out
    if kind == "top":
        values, at = torch.sort(s["logits"], dim=1, descending=True, stable=True)
        return values[:, :c["k"]].contiguous(), at[:, :c["k"]].to(torch.int32)
    return _plain_distill(s) if kind == "distill" else _plain_attend(s)


def _plain_distill(s):
    T, at = s["temperature"], s["indices"].long()
    z = s["student"].float() / T
    z = z - z.amax(1, keepdim=True)
    lse = z.exp().sum(1, keepdim=True).log()
    t = s["values"].float() / T
    t = t - t.amax(1, keepdim=True)
    logp = t - t.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    loss = T * T * (p * (logp - (z.gather(1, at) - lse))).sum(1)
    grad = (z - lse).exp()
    grad.scatter_add_(1, at, -p)
    grad.mul_(s["grad"][:, None] * T)
    return loss, grad.to(s["student"].dtype)


def _bias_index(s):
    """Bucket of each (sequence or 1, query, key), and the positions of the queries."""
    c, dev = s["case"], s["q"].device
    first = torch.zeros(1, dtype=torch.long, device=dev)
    if c["kind"] == "token":
        first = (s["kv_len"].long() if s["kv_len"] is not None else first + c["Lk"]) - c["Lq"]
    p = (first[:, None] + torch.arange(c["Lq"], device=dev))[:, :, None]
    j = torch.arange(c["Lk"], device=dev)[None, None, :]
    if c["width"]:
        w, h = c["width"], c["Lk"] // c["width"]
        return (j // w - p // w + h - 1) * (2 * w - 1) + (j % w - p % w + w - 1), p, j
    return s["offsets"][(j - p).clamp(1 - c["Lk"], c["Lk"] - 1) + c["Lk"] - 1], p, j


def _plain_attend(s):
    c = s["case"]
    B, Lq, Lk, H, Hkv, D = (c[x] for x in ("B", "Lq", "Lk", "H", "Hkv", "D"))
    G, scale = H // Hkv, 1 / math.sqrt(D)
    bucket, p, j = _bias_index(s)
    hidden = (j > p) if c["causal"] else torch.zeros_like(j, dtype=torch.bool)
    if s["kv_len"] is not None:
        hidden = hidden | (j >= s["kv_len"].long()[:, None, None])
    # [B, Hkv, G * Lq, D]: the query heads of a key/value head as rows of one product
    rows = lambda x: x.float().view(B, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Lq, D)  # noqa: E731
    back = lambda x: x.view(B, Hkv, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, H, D)  # noqa: E731
    q, k, v = rows(s["q"]), s["k"].float().transpose(1, 2).contiguous(), s["v"].float().transpose(1, 2).contiguous()
    P = torch.matmul(q, k.transpose(2, 3)).view(B, H, Lq, Lk)
    P.mul_(scale).add_(s["table"].float()[bucket].permute(0, 3, 1, 2)).masked_fill_(hidden[:, None], -math.inf)
    P.sub_(P.amax(3, keepdim=True)).exp_()
    P.div_(P.sum(3, keepdim=True))
    P = P.view(B, Hkv, G * Lq, Lk)
    out = torch.matmul(P, v)
    if c["kind"] != "attend_train":
        return back(out).to(s["q"].dtype)
    g = rows(s["grad"])
    dv = torch.matmul(P.transpose(2, 3), g)
    dS = torch.matmul(g, v.transpose(2, 3)).sub_((g * out).sum(3, keepdim=True)).mul_(P)
    dq = torch.matmul(dS, k).mul_(scale)
    dk = torch.matmul(dS.transpose(2, 3), q).mul_(scale)
    # the sums over sequences and pairs of a bucket are long: 64 bits
    by_pair = dS.view(B, H, Lq, Lk).sum(0, dtype=torch.float64)
    if not c["width"]:
        # a sequence's bucket goes by the offset alone: first the sums along the diagonals, column j + (Lq - 1 - i)
        by_pair = torch.nn.functional.pad(by_pair.flip(1), (0, Lq)).flatten(1)[:, :Lq * (Lk + Lq - 1)].view(H, Lq, Lk + Lq - 1).sum(1)
        bucket = s["offsets"]
    dtable = torch.zeros(s["table"].shape, dtype=torch.float64, device=g.device).index_add_(0, bucket.reshape(-1), by_pair.flatten(1).t())
    t = s["q"].dtype
    return tuple(x.to(t) for x in (back(out), back(dq), dk.transpose(1, 2).contiguous(), dv.transpose(1, 2).contiguous(), dtable))


def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] == "top":
        x, k = s["logits"].double(), c["k"]
        # the k-th value, everything above it, and of what equals it the first places
        kth = torch.topk(x, k, dim=1).values[:, -1:]
        above, equal = x > kth, x == kth
        taken = above | (equal & (equal.cumsum(1) <= k - above.sum(1, keepdim=True)))
        at = taken.nonzero()[:, 1].view(-1, k)
        values = x.gather(1, at)
        order = torch.argsort(values, dim=1, descending=True, stable=True)
        return values.gather(1, order), at.gather(1, order).to(torch.int32)
    if c["kind"] == "distill":
        T, at = s["temperature"], s["indices"].long()
        logq = torch.log_softmax(s["student"].detach().double() / T, 1)
        logp = torch.log_softmax(s["values"].double() / T, 1)
        loss = T * T * (logp.exp() * (logp - logq.gather(1, at))).sum(1)
        return loss, (logq.exp().scatter_add(1, at, -logp.exp())) * (T * s["grad"].double()[:, None])
    B, Lq, Lk, H, Hkv, D = (c[x] for x in ("B", "Lq", "Lk", "H", "Hkv", "D"))
    q, k, v, table = (s[x].detach().double() for x in ("q", "k", "v", "table"))
    train = c["kind"] == "attend_train"
    out = torch.empty_like(q)
    dq, dk, dv, dtable = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(table)
    j = torch.arange(Lk, device=q.device)
    for b, n in enumerate(_lengths(c)):
        p = torch.arange(Lq, device=q.device) + (n - Lq if c["kind"] == "token" else 0)
        off = j[None, :] - p[:, None]
        if c["width"]:
            w = c["width"]
            rows_, cols = torch.div(j, w, rounding_mode="floor")[None] - torch.div(p, w, rounding_mode="floor")[:, None], j[None] % w - p[:, None] % w
            bucket = (rows_ + Lk // w - 1) * (2 * w - 1) + cols + w - 1
        else:
            half = _BUCKETS if c["causal"] else _BUCKETS // 2
            n_off = (-off).clamp(min=0) if c["causal"] else off.abs()
            far = half // 2 + torch.floor(torch.log(n_off.clamp(min=1).double() * 2 / half) / math.log(2 * _SPAN / half) * (half - half // 2) + 1e-9)
            bucket = torch.where(n_off < half // 2, n_off, far.long().clamp(max=half - 1))
            bucket = bucket if c["causal"] else bucket + half * (off > 0)
        seen = (j[None] < n) & ((off <= 0) if c["causal"] else (off == off))
        for h in range(H):
            kh, vh = k[b, :, h * Hkv // H], v[b, :, h * Hkv // H]
            score = (q[b, :, h] @ kh.t()) / math.sqrt(D) + table[:, h][bucket]
            prob = torch.softmax(score.masked_fill(~seen, -math.inf), 1)
            out[b, :, h] = prob @ vh
            if train:
                g = s["grad"][b, :, h].double()
                ds = prob * (g @ vh.t() - (g * out[b, :, h]).sum(1, keepdim=True))
                dq[b, :, h] = ds @ kh / math.sqrt(D)
                dk[b, :, h * Hkv // H] += ds.t() @ q[b, :, h] / math.sqrt(D)
                dv[b, :, h * Hkv // H] += prob.t() @ g
                dtable[:, h] += torch.bincount(bucket.reshape(-1), weights=ds.reshape(-1), minlength=table.shape[0])
    return (out, dq, dk, dv, dtable) if train else out
