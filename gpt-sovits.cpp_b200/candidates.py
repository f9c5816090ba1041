"""Several candidates of one prompt: the shared cache, attention over it and the tokens' scores, together.

A decoder of the T2S shape (post-LayerNorm blocks of 16 heads x 32, ReLU FFN) that continues semantic tokens.  A
prompt's positions are computed once; its candidates fork its pages, each step's attention reads the shared pages once for all
of them, and every drawn token is scored as it is drawn.  Halfway the worse half of each prompt's candidates
is dropped and the pool compacted, so that the pages in use are the lowest ones again.

    python candidates.py            # two prompts, eight candidates each, random weights
"""
from __future__ import annotations

import math

import numpy as np
import torch

import t2sx

HEADS, DIM, EOS = 16, 32, 1024


class Decoder:
    """tensors: (name, f32 array) pairs named as in the converter's files; projections are kept in f16."""

    def __init__(self, tensors, device: int = 0):
        self.device, self.vec, self.w = device, {}, {}
        for name, a in tensors:
            if name.startswith(("attention.", "sampler.")) and a.ndim == 2:
                self.w[name] = t2sx.Weight(t2sx.F16, np.ascontiguousarray(a, np.float16).view(np.uint8).reshape(-1), *a.shape, device)
            elif name.startswith(("attention.", "encoder.audio")):
                self.vec[name] = torch.tensor(a, device=f"cuda:{device}")
        self.layers = 1 + max(int(n.split(".")[1]) for n in self.w if n.startswith("attention."))
        self.vocab, self.d = self.vec["encoder.audio_embedding"].shape

    def _linear(self, name, x, bias=None):
        w, stream = self.w[name], torch.cuda.current_stream().cuda_stream
        y = torch.empty((x.shape[0], w.N), device=x.device)
        w.matmul(x.data_ptr(), x.shape[0], y.data_ptr(), None if bias is None else bias.data_ptr(), stream)
        return y

    def embed(self, tokens, positions):
        freq = torch.exp(torch.arange(0, self.d, 2, device=tokens.device) * (-math.log(10000.0) / self.d))
        angle = positions[:, None] * freq
        pe = torch.stack([angle.sin(), angle.cos()], 2).flatten(1)
        return self.vec["encoder.audio_embedding"][tokens] + self.vec["encoder.audio_pos_alpha"] * pe

    def forward(self, plan, x):
        """Hidden rows of the plan's step; their keys and values go into the pool."""
        stream = torch.cuda.current_stream().cuda_stream
        for i in range(self.layers):
            p = f"attention.{i}."
            norm = lambda y, n: torch.nn.functional.layer_norm(y, (self.d,), self.vec[p + n + "_w"], self.vec[p + n + "_b"])
            q, k, v = (t.half() for t in self._linear(p + "qkv_w", x, self.vec[p + "qkv_b"]).chunk(3, 1))
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
            out = torch.empty_like(q)
            plan.attend(i, q.data_ptr(), out.data_ptr(), DIM ** -0.5, k.data_ptr(), v.data_ptr(), stream=stream)
            x = norm(x + self._linear(p + "out_proj_w", out.float(), self.vec[p + "out_proj_b"]), "ln1")
            up = self._linear(p + "ffn_up_w", x, self.vec[p + "ffn_up_b"]).relu_()
            x = norm(x + self._linear(p + "ffn_down_w", up, self.vec[p + "ffn_down_b"]), "ln2")
        return x

    def logits(self, x):
        return self._linear("sampler.lm_head_w", x)


def draw(dec: Decoder, prompts, each: int, steps: int, top_k: int = 15, seed: int = 0):
    """Draws `each` continuations of every prompt (lists of one token id or more), `steps` tokens at most.  Returns, for
    each prompt, those kept as (mean log probability, tokens), the best first."""
    if any(len(p) == 0 for p in prompts):
        raise ValueError("a prompt needs a token to continue")
    dev, PAGE = torch.device("cuda", dec.device), t2sx.PagePool.PAGE
    stream = torch.cuda.current_stream().cuda_stream
    gen = torch.Generator(device=dev).manual_seed(seed)
    lens = [len(p) for p in prompts]
    n = len(prompts) * each
    pages = sum(-(-m // PAGE) for m in lens) + sum(each * (-(-(m + steps) // PAGE) - m // PAGE) for m in lens)
    k, v = (torch.empty((dec.layers, pages, HEADS, PAGE, DIM), dtype=torch.float16, device=dev) for _ in range(2))
    pool = t2sx.PagePool(t2sx.F16, dec.layers, pages, HEADS, DIM, n + len(prompts), k.data_ptr(), v.data_ptr(), dec.device)
    plan = pool.plan(HEADS)

    # the prompts, all positions in one step; then their candidates
    parents = list(range(n, n + len(prompts)))
    pool.extend(parents, lens)
    plan.update(parents, lens, stream)
    tokens = torch.tensor([t for p in prompts for t in p], device=dev)
    positions = torch.cat([torch.arange(m, device=dev) for m in lens])
    last = torch.tensor(np.cumsum(lens) - 1, device=dev)
    logits = dec.logits(dec.forward(plan, dec.embed(tokens, positions))[last]).repeat_interleave(each, 0)
    pool.fork([p for p in parents for _ in range(each)], range(n), stream)
    pool.release(parents)

    live, drawn, total = list(range(n)), [[] for _ in range(n)], [0.0] * n
    dropped = set()
    for step in range(steps):
        best = logits.topk(top_k, 1)
        picked = best.indices.gather(1, torch.multinomial(best.values.softmax(1), 1, generator=gen))[:, 0].int()
        score = torch.empty(len(live), device=dev)
        t2sx.token_logprobs(t2sx.F32, len(live), dec.vocab, logits.data_ptr(), picked.data_ptr(), score.data_ptr(),
                            device=dec.device, stream=stream)
        for seq, token, s in zip(live, picked.tolist(), score.tolist()):
            drawn[seq].append(token)
            total[seq] += s
        mean = [t / max(1, len(d)) for t, d in zip(total, drawn)]
        going = [s for s in live if drawn[s][-1] != EOS]
        if step == steps // 2:   # the worse half of each prompt's candidates
            for p in range(len(prompts)):
                dropped |= set(sorted(range(p * each, p * each + each), key=lambda s: -mean[s])[(each + 1) // 2:])
            going = [s for s in going if s not in dropped]
        if gone := [s for s in live if s not in going]:
            pool.release(gone)
            pool.compact(stream)
        live = going
        if not live or step == steps - 1:
            break
        pool.extend(live, [1] * len(live))
        plan.update(live, [1] * len(live), stream)
        at = torch.tensor([pool.length(s) - 1 for s in live], device=dev)
        logits = dec.logits(dec.forward(plan, dec.embed(torch.tensor([drawn[s][-1] for s in live], device=dev), at)))
    plan.sync()   # also reports a tensor-core attention that gave up
    plan.close()
    pool.close()
    mean = [t / max(1, len(d)) for t, d in zip(total, drawn)]
    return [sorted(((mean[s], drawn[s]) for s in range(p * each, p * each + each) if s not in dropped), key=lambda c: -c[0])
            for p in range(len(prompts))]


def main():
    import synth
    dec = Decoder(synth.tensor_values(0, n_layer=4))
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, EOS, m).tolist() for m in (350, 90)]
    for p, found in enumerate(draw(dec, prompts, each=8, steps=40)):
        for score, tokens in found:
            print(f"prompt {p}: {score:8.4f}  {len(tokens)} tokens  {' '.join(map(str, tokens[:8]))} ...")


if __name__ == "__main__":
    main()
