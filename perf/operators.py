"""Cases of the batched-serving operators: attention over packed prompts, attention of
new tokens over a paged cache, and the append that fills that cache.

``run`` computes them either in their plain form (elementary torch operations in 32
bits) or, where ``own`` is true, through the package's public calls. ``exact`` is the
same from the definitions in 64 bits."""
import math

import torch

own = False

EPS = 1e-6
THETA = 1.0e6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- the cases -----------------------------------------------------------------------
# A case gives every request's number of new tokens (q_lens) and, for the paged
# operators, the number of its keys once those tokens are in the cache (kv_lens), as
# text. heads / kv_heads / dim are 16 / 8 / 128 (the decode engine's), one rank of its
# tensor-parallel split, or generic.

def _text(lens):
    return ",".join(str(int(n)) for n in lens)


def _lens(text):
    return [int(n) for n in text.split(",")]


def _prompt(name, q_lens, heads=16, kv_heads=8, dim=128, dtype="bf16"):
    return {"name": name, "op": "prompt", "q_lens": _text(q_lens), "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype}


def _paged(name, q_lens, kv_lens, page, heads=16, kv_heads=8, dim=128, dtype="bf16"):
    return {"name": name, "op": "paged", "q_lens": _text(q_lens), "kv_lens": _text(kv_lens), "page": page,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}


def _append(name, q_lens, kv_lens, page, heads=16, kv_heads=8, dim=128, dtype="bf16", source="bf16", norm=True,
            keep_k=False):
    return {"name": name, "op": "append", "q_lens": _text(q_lens), "kv_lens": _text(kv_lens), "page": page,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "source": source, "norm": norm,
            "keep_k": keep_k}


def listed():
    spread = [1 + (i * i * 4095) // (47 * 47) for i in range(48)]            # 48 requests, 1 to 4096 keys
    ragged = [3, 1411, 77, 640, 129, 1, 902, 256, 33, 411, 128, 515]         # 12 prompts, 4506 tokens
    return [
        # one short prompt: a first request on an idle server, all latency
        _prompt("prompt-one-37", [37]),
        # a batch of prompts as they arrive, of uneven lengths
        _prompt("prompt-ragged-12", ragged),
        # other types and heads: FP16, 64-wide heads, three query heads to a KV head
        _prompt("prompt-fp16-d64", [2049, 1000, 4097], heads=24, kv_heads=8, dim=64, dtype="fp16"),
        # one long document
        _prompt("prompt-long", [15999]),
        # one request's next token over a short cache: the latency of a single stream
        _paged("decode-one-33", [1], [33], 16),
        # a decode step of a full batch, every request at another length
        _paged("decode-batch-48", [1] * 48, spread, 16),
        # a few very long contexts, where the work has to be split over the keys
        _paged("decode-long-3", [1] * 3, [60000, 9001, 31234], 64),
        # chunked prefill: 512 new tokens of four prompts over what is cached of them
        _paged("chunk-512", [512] * 4, [3840, 512, 2047, 1500], 32),
        # a mixed step: 28 requests decode while two prompts bring their next chunk
        _paged("mixed-30", [1] * 28 + [700, 256], [90 + 131 * i for i in range(28)] + [2748, 256], 16),
        # the append of a decode step of 48 requests
        _append("append-decode-48", [1] * 48, spread, 16),
        # the append of a batch of prompts, the rotated keys kept packed for the prompt attention
        _append("append-ragged-12", ragged, ragged, 16, keep_k=True),
        # the append of a long prompt's chunk from an FP32 projection, without q/k norms
        _append("append-long-fp32", [16000], [19001], 64, source="fp32", norm=False),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _cost(c):
    w = work(c)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _plain_room(c):
    """Values of the plain form's padded scores and gathered keys."""
    q, kv = _lens(c["q_lens"]), _lens(c.get("kv_lens", c["q_lens"]))
    return max(len(q) * c["heads"] * max(q) * max(kv), 4 * len(q) * c["kv_heads"] * max(kv) * c["dim"])


def draw(rng):
    every = listed()
    top = {op: max(_cost(c) for c in every if c["op"] == op) for op in ("prompt", "paged", "append")}
    room = max(_plain_room(c) for c in every if c["op"] != "append")
    while True:
        heads, kv_heads = rng.choice([(16, 8), (16, 8), (8, 4), (2, 1), (24, 8), (32, 8), (12, 12), (14, 2), (16, 1)])
        more = {"heads": heads, "kv_heads": kv_heads, "dim": rng.choice([128, 128, 64]),
                "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        op = rng.choice(["prompt", "paged", "paged", "append"])
        page = rng.choice([16, 16, 32, 64, 128])
        n = _log(rng, 1, 64)
        if op == "prompt":
            longest = _log(rng, 16, 15999)
            c = _prompt("", [_log(rng, 1, longest) for _ in range(n)] + [longest], **more)
        else:
            kind = rng.choice(["decode", "decode", "chunk", "mixed"])
            longest = _log(rng, 16, 60000)
            past = [_log(rng, 1, longest) - 1 for _ in range(n)]
            long = _log(rng, 2, 2048)
            q = [1 if kind == "decode" or kind == "mixed" and rng.random() < 0.8 else _log(rng, 1, long) for _ in past]
            kv = [a + b for a, b in zip(past, q)]
            if op == "paged":
                c = _paged("", q, kv, page, **more)
            else:
                c = _append("", q, kv, page, source=rng.choice(["bf16", "fp16", "fp32"]), norm=rng.random() < 0.7,
                            keep_k=rng.random() < 0.5, **more)
        del c["name"]
        if _cost(c) <= top[op] and (op == "append" or _plain_room(c) <= room):
            return c


# ---- inputs --------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    dtype = TYPES[case["dtype"]]
    q_lens = _lens(case["q_lens"])
    total, n = sum(q_lens), len(q_lens)

    def normal(*shape, dtype=dtype, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dtype)

    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).to(dev)
    s = {"op": case["op"], "cu": cu, "max_q": max(q_lens), "ragged": max(q_lens) > 1 or total != n}
    if case["op"] == "prompt":
        return {**s, "q": normal(total, hq, d, scale=2.0), "k": normal(total, hk, d), "v": normal(total, hk, d)}

    kv_lens, page = _lens(case["kv_lens"]), case["page"]
    pages = [-(-m // page) for m in kv_lens]
    pool = sum(pages) + 5
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table, at = torch.full((n, max(pages)), -1, dtype=torch.int32), 0  # -1: no page
    for b, m in enumerate(pages):
        table[b, :m] = order[at:at + m]
        at += m
    s.update(kv_lens=torch.tensor(kv_lens, dtype=torch.int32, device=dev), table=table.to(dev), page=page,
             k_cache=normal(pool, hk, page, d), v_cache=normal(pool, hk, page, d))
    if case["op"] == "paged":
        return {**s, "q": normal(total, hq, d, scale=2.0)}

    longest = max(kv_lens)
    freq = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = torch.outer(torch.arange(longest, dtype=torch.float64), freq)
    angle = torch.cat((angle, angle), 1)
    s.update(cos=angle.cos().float().to(dev), sin=angle.sin().float().to(dev), keep_k=case["keep_k"],
             qkv=normal(total, hq + 2 * hk, d, dtype=TYPES[case["source"]], scale=1.5), q_norm=None, k_norm=None)
    if case["norm"]:
        s.update(q_norm=1 + normal(d, scale=0.1), k_norm=1 + normal(d, scale=0.1))
    return s


# ---- one pass ------------------------------------------------------------------------

def run(state):
    s = state
    if own:
        import megakernel_b200 as mk
        if s["op"] == "prompt":
            return mk.prompt_attention(s["q"], s["k"], s["v"], s["cu"])
        cu = s["cu"] if s["ragged"] else None
        if s["op"] == "paged":
            return mk.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], cu)
        got = mk.paged_append(s["qkv"], s["k_cache"], s["v_cache"], s["table"], s["kv_lens"], s["cos"], s["sin"], cu,
                              q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, return_k=s["keep_k"])
        q, k = got if s["keep_k"] else (got, None)
        return {"q": q, "k": k, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if s["op"] == "prompt":
        return _plain_prompt(s)
    return _plain_paged(s) if s["op"] == "paged" else _plain_append(s)


def _requests(cu, total):
    """Of every packed token: its request and its place among that request's tokens."""
    token = torch.arange(total, dtype=cu.dtype, device=cu.device)
    request = torch.searchsorted(cu, token, right=True) - 1
    return request, token - cu[request]


def _padded(x, cu, longest):
    """Packed [T, H, D] to FP32 [B, H, longest, D]; what lies past a request's end is its last row."""
    at = (cu[:-1, None] + torch.arange(longest, device=cu.device)).minimum(cu[1:, None] - 1)
    return x[at].float().transpose(1, 2)


def _attend(q, k, v, sees):
    """softmax(q k^T / sqrt(D)) v where `sees` [B, 1, Lq, Lk]; q [B, Hq, Lq, D], k and v [B, Hk, Lk, D]."""
    n, hq, lq, d = q.shape
    hk = k.shape[1]
    score = torch.matmul((q * d ** -0.5).reshape(n, hk, -1, d), k.transpose(-1, -2)).view(n, hq, lq, -1)
    score.masked_fill_(~sees, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, hk, -1, p.shape[-1]), v).view(n, hq, lq, d)
    return out / total.masked_fill(total == 0, 1.0)


def _plain_prompt(s):
    q, cu = s["q"], s["cu"]
    place = torch.arange(s["max_q"], device=cu.device)
    sees = (place[None, :] <= place[:, None])[None, None]
    out = _attend(*(_padded(x, cu, s["max_q"]) for x in (q, s["k"], s["v"])), sees)
    request, at = _requests(cu, q.shape[0])
    return out[request, :, at].to(q.dtype)


def _plain_paged(s):
    q, cu, lens, table = s["q"], s["cu"], s["kv_lens"], s["table"].clamp(min=0).long()
    k, v = (c[table].transpose(1, 2).flatten(2, 3).float() for c in (s["k_cache"], s["v_cache"]))
    key = torch.arange(k.shape[2], device=cu.device)
    v = v.masked_fill((key >= lens[:, None])[:, None, :, None], 0.0)  # past the last key a page holds anything
    first = lens - (cu[1:] - cu[:-1])
    sees = key <= (first[:, None] + torch.arange(s["max_q"], device=cu.device))[:, :, None]
    sees &= key < lens[:, None, None]
    out = _attend(_padded(q, cu, s["max_q"]), k, v, sees[:, None])
    request, at = _requests(cu, q.shape[0])
    return out[request, :, at].to(q.dtype)


def _plain_append(s):
    cu, lens, kc, vc = s["cu"], s["kv_lens"], s["k_cache"], s["v_cache"]
    x = s["qkv"].float()
    hk, d = kc.shape[1], x.shape[-1]
    q, k, v = x.split([x.shape[1] - 2 * hk, hk, hk], 1)
    request, at = _requests(cu, x.shape[0])
    position = (lens - cu[1:] + cu[:-1])[request] + at
    cos, sin = s["cos"][position, None], s["sin"][position, None]

    def turned(y, weight):
        if weight is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()
        return y * cos + torch.cat((-y[..., d // 2:], y[..., :d // 2]), -1) * sin

    q, k = turned(q, s["q_norm"]).to(kc.dtype), turned(k, s["k_norm"]).to(kc.dtype)
    page, slot = s["table"][request, position // s["page"]].long(), position % s["page"]
    kc[page, :, slot] = k
    vc[page, :, slot] = v.to(vc.dtype)
    return {"q": q, "k": k if s["keep_k"] else None, "k_cache": kc, "v_cache": vc}


# ---- the definitions in 64 bits --------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    ends = s["cu"].tolist()
    if case["op"] == "append":
        return _exact_append(case, s, ends)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, (a, e) in enumerate(zip(ends, ends[1:])):
        if case["op"] == "prompt":
            k, v, keys = s["k"][a:e], s["v"][a:e], e - a
        else:
            keys, ids = _lens(case["kv_lens"])[b], s["table"][b]
            ids = ids[: -(-keys // case["page"])].long()
            k, v = (c[ids].permute(0, 2, 1, 3).reshape(-1, hk, d)[:keys] for c in (s["k_cache"], s["v_cache"]))
        for h in range(hk):
            kh, vh = k[:, h].double(), v[:, h].double()
            for g in range(h * hq // hk, (h + 1) * hq // hk):
                for i in range(a, e, 4096):
                    j = min(e, i + 4096)
                    seen = keys - (e - j)  # the last of these rows sees so many keys
                    z = s["q"][i:j, g].double() @ kh[:seen].T / math.sqrt(d)
                    z += torch.full_like(z, -math.inf).triu(seen - (j - i) + 1)
                    out[i:j, g] = torch.softmax(z, -1) @ vh[:seen]
    return out


def _exact_append(case, s, ends):
    hq, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    kc, vc, x = s["k_cache"].double(), s["v_cache"].double(), s["qkv"].double()
    first = x[:, :hq + hk]
    if case["norm"]:
        first = first / torch.sqrt((first ** 2).sum(-1, keepdim=True) / d + EPS)
        first = torch.cat((first[:, :hq] * s["q_norm"].double(), first[:, hq:] * s["k_norm"].double()), 1)
    lens = _lens(case["kv_lens"])
    place = torch.cat([torch.arange(n - (e - a), n) for a, e, n in zip(ends, ends[1:], lens)]).to(x.device)
    cos, sin = s["cos"].double()[place][:, None], s["sin"].double()[place][:, None]
    low, high = first[..., : d // 2], first[..., d // 2:]
    first = torch.cat((low * cos[..., : d // 2] - high * sin[..., : d // 2],
                       high * cos[..., d // 2:] + low * sin[..., d // 2:]), -1)
    rows = torch.cat([s["table"][b, place[a:e] // page] for b, (a, e) in enumerate(zip(ends, ends[1:]))]).long()
    for h in range(hk):
        kc[rows, h, place % page] = first[:, hq + h]
        vc[rows, h, place % page] = x[:, hq + hk + h]
    return {"q": first[:, :hq], "k": first[:, hq:] if case["keep_k"] else None, "k_cache": kc, "v_cache": vc}


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    q_lens, kv_lens = _lens(case["q_lens"]), _lens(case.get("kv_lens", case["q_lens"]))
    total = sum(q_lens)
    if case["op"] == "append":
        size = 4 if case["source"] == "fp32" else 2
        places = set()
        for n, m in zip(q_lens, kv_lens):
            places.update(range(m - n, m))
        bytes_ = total * (hq + 2 * hk) * d * (size + 2) + len(places) * d * 8 + (total * hk * d * 2 if case["keep_k"] else 0)
        return {"bytes": bytes_, "flops": total * (hq + hk) * d * 7}
    seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q_lens, kv_lens))
    return {"bytes": 2 * d * (2 * total * hq + 2 * sum(kv_lens) * hk), "flops": 4 * hq * d * seen}
