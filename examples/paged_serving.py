"""Many requests at once over a paged cache: a greedy Qwen3-0.6B server in small.

Requests come and go while others decode. A step of the server is one of

* prompts:  whole new prompts, packed    paged_append(return_k=True), prompt_attention
* mixed:    a chunk of one long prompt next to everybody's next token
                                          paged_append, paged_attention(cu_q)
* decode:   everybody's next token        paged_append, paged_attention

over pools of 16-key pages that requests take from a list and give back at their end. The
projections are library GEMMs; residuals are kept in FP32. Weights are random, or a
checkpoint's (``--checkpoint DIR``).

    python examples/paged_serving.py [--layers N] [--requests N] [--tokens N] [--check]

``--check`` decodes every request again by itself on the resident batch-one engine and
compares the tokens up to the first whose two best logits lie within rounding of each other.
"""
from __future__ import annotations

import argparse
import os
import sys
import time
from dataclasses import dataclass, field

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import megakernel_b200 as mk  # noqa: E402
from megakernel_b200.engine import HEAD_DIM, LAYER_SHAPES, N_KV, VOCAB  # noqa: E402

EPS, PAGE = 1e-6, 16


def random_weights(layers: int, device="cuda", seed=0):
    """embed, final norm, and the 11 tensors a layer in LayerWeights order."""
    g = torch.Generator(device=device).manual_seed(seed)

    def draw(shape):
        if len(shape) == 1:
            return torch.ones(shape, dtype=torch.bfloat16, device=device)
        return (torch.randn(shape, generator=g, device=device) * 0.02).to(torch.bfloat16)

    return draw((VOCAB, LAYER_SHAPES[0][0])), draw(LAYER_SHAPES[0]), [draw(s) for _ in range(layers) for s in LAYER_SHAPES]


@dataclass
class Request:
    prompt: list
    budget: int                     # tokens to generate
    seen: int = 0                   # prompt and generated tokens whose keys are in the cache
    out: list = field(default_factory=list)
    margins: list = field(default_factory=list)  # best logit minus the second, of each of them
    pages: list = field(default_factory=list)


class Server:
    def __init__(self, embed, final_norm, layer_weights, *, pages: int, max_len: int, chunk=512, lm_head=None):
        self.embed, self.final_norm, self.head = embed, final_norm, embed if lm_head is None else lm_head
        self.layers = []
        for i in range(0, len(layer_weights), 11):
            n1, q, k, v, qn, kn, o, n2, gate, up, down = layer_weights[i:i + 11]
            self.layers.append((n1, torch.cat((q, k, v)), qn, kn, o, n2, torch.cat((gate, up)), down))
        dev = embed.device
        self.k, self.v = (torch.empty((len(self.layers), pages, N_KV, PAGE, HEAD_DIM), dtype=torch.bfloat16, device=dev)
                          for _ in range(2))
        self.cos, self.sin = mk.rope_tables(max_len, dev)
        self.free, self.width, self.chunk = list(range(pages)), -(-max_len // PAGE), chunk
        self.waiting, self.running = [], []
        self.partial = None          # a long prompt that comes in chunk by chunk

    def add(self, prompt, budget):
        r = Request(list(prompt), budget)
        self.waiting.append(r)
        return r

    # ---- the model over a packed batch ------------------------------------------------
    @torch.no_grad()
    def forward(self, ids, table, kv_lens, cu_q, whole: bool):
        """Logits of each request's last new token. ``cu_q`` None: one token each;
        ``whole``: the new tokens are all of each request's keys."""
        last = torch.arange(ids.shape[0], device=ids.device) if cu_q is None else cu_q[1:].long() - 1
        x = F.embedding(ids, self.embed).float()
        hidden = x.shape[1]
        for layer, (n1, wqkv, qn, kn, wo, n2, wgu, wd) in enumerate(self.layers):
            h = F.rms_norm(x, (hidden,), n1.float(), EPS).to(torch.bfloat16)
            qkv = F.linear(h, wqkv).view(ids.shape[0], -1, HEAD_DIM)
            got = mk.paged_append(qkv, self.k[layer], self.v[layer], table, kv_lens, self.cos, self.sin, cu_q,
                                  q_norm=qn, k_norm=kn, eps=EPS, return_k=whole)
            if whole:
                q, k = got
                o = mk.prompt_attention(q, k, qkv[:, -N_KV:], cu_q)
            else:
                o = mk.paged_attention(got, self.k[layer], self.v[layer], table, kv_lens, cu_q)
            x += F.linear(o.flatten(1), wo)
            h = F.rms_norm(x, (hidden,), n2.float(), EPS).to(torch.bfloat16)
            gate, up = F.linear(h, wgu).chunk(2, -1)
            x += F.linear(F.silu(gate) * up, wd)
        x = F.rms_norm(x[last], (hidden,), self.final_norm.float(), EPS).to(torch.bfloat16)
        return F.linear(x, self.head).float()

    # ---- steps --------------------------------------------------------------------------
    def _run(self, work, whole=False):
        """One step of the model over ``work``: (request, its new tokens)."""
        dev = self.embed.device
        for r, new in work:
            need = -(-(r.seen + len(new)) // PAGE) - len(r.pages)
            if need > len(self.free):
                raise RuntimeError("the pool has no free pages")
            r.pages += [self.free.pop() for _ in range(need)]
        counts = [len(new) for _, new in work]
        table = torch.full((len(work), self.width), -1, dtype=torch.int32)
        for b, (r, _) in enumerate(work):
            table[b, :len(r.pages)] = torch.tensor(r.pages, dtype=torch.int32)
        lens = torch.tensor([r.seen + n for (r, _), n in zip(work, counts)], dtype=torch.int32)
        cu = None
        if whole or max(counts) > 1:
            cu = F.pad(torch.tensor(counts).cumsum(0), (1, 0)).to(torch.int32).to(dev)
        ids = torch.tensor([t for _, new in work for t in new], dtype=torch.int64)
        logits = self.forward(ids.to(dev), table.to(dev), lens.to(dev), cu, whole)
        best = logits.topk(2, -1)
        tokens, margins = best.indices[:, 0].tolist(), (best.values[:, 0] - best.values[:, 1]).tolist()
        code, why = mk.serving_status(dev)
        if code:
            raise RuntimeError(why)
        for (r, new), token, margin in zip(work, tokens, margins):
            r.seen += len(new)
            if r.seen >= len(r.prompt):  # (a chunk of a prompt yields no token before the last)
                r.out.append(token)
                r.margins.append(margin)
        self.last_logits = logits

    def step(self):
        """One step; False once there is nothing left to do."""
        if self.partial is None and self.waiting:
            short = [r for r in self.waiting if len(r.prompt) <= self.chunk]
            if short and (not self.running or len(short) == len(self.waiting)):
                self._run([(r, r.prompt) for r in short], whole=True)
                self.waiting = [r for r in self.waiting if r not in short]
                self.running += short
                return self._retire()
            self.partial = next(r for r in self.waiting if len(r.prompt) > self.chunk)
            self.waiting.remove(self.partial)
        work = [(r, [r.out[-1]]) for r in self.running]
        p = self.partial
        if p is not None:
            work.append((p, p.prompt[p.seen:p.seen + self.chunk]))
        if not work:
            return False
        self._run(work)
        if p is not None and p.seen >= len(p.prompt):
            self.running.append(p)
            self.partial = None
        return self._retire()

    def _retire(self):
        for r in [r for r in self.running if len(r.out) >= r.budget]:
            self.running.remove(r)
            self.free += r.pages
            r.pages = []
        return True


def compare(weights, requests, max_len, rounding, lm_head=None):
    """Each request alone on the batch-one engine; tokens compared while the choice is clear."""
    embed, final_norm, layers = weights
    k = torch.zeros((len(layers) // 11, N_KV, max_len, HEAD_DIM), dtype=torch.bfloat16, device=embed.device)
    eng = mk.DecodeEngine(embed, final_norm, layers, k, torch.zeros_like(k), lm_head=lm_head)
    same = 0
    for r in requests:
        first = eng.prefill(torch.tensor(r.prompt, dtype=torch.int32, device=embed.device), batched=len(r.prompt) > 1)
        alone = [first] + eng.generate(first, len(r.prompt), r.budget - 1).tolist() if r.budget > 1 else [first]
        for mine, theirs, margin in zip(r.out, alone, r.margins):
            if mine != theirs:
                if margin > rounding:
                    raise RuntimeError(f"token {same}: {mine} here, {theirs} alone, by {margin:.3f}")
                break  # a choice within rounding: what follows is another text
            same += 1
    eng.close()
    return same


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=28)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--max-len", type=int, default=2048)
    ap.add_argument("--checkpoint")
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args(argv)
    if a.checkpoint:
        from megakernel_b200.checkpoint import load_qwen3
        w = load_qwen3(a.checkpoint, device="cuda")
        weights, head = (w.embed, w.final_norm, w.layer_weights), w.lm_head
    else:
        weights, head = random_weights(a.layers), None
    g = torch.Generator().manual_seed(1)
    server = Server(*weights, pages=a.requests * -(-a.max_len // PAGE), max_len=a.max_len, lm_head=head)
    lengths = [1 + int(torch.randint(0, 300, (), generator=g)) for _ in range(a.requests)]
    lengths[-1] = max(1, a.max_len - a.tokens)  # one long prompt, in chunks
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in lengths]
    requests = [server.add(p, a.tokens) for p in prompts[:-2]]
    steps, start = 0, time.perf_counter()
    while server.step():
        steps += 1
        if steps == 4:  # the last two come while the others decode
            requests += [server.add(p, a.tokens) for p in prompts[-2:]]
    torch.cuda.synchronize()
    seconds = time.perf_counter() - start
    made = sum(len(r.out) for r in requests)
    print(f"{len(requests)} requests, {sum(lengths)} prompt and {made} generated tokens in {steps} steps, {seconds:.2f} s")
    if a.check:
        print(f"{compare(weights, requests, a.max_len, 0.05, head)} tokens equal to the batch-one engine's")


if __name__ == "__main__":
    main()
