"""A decoder that keeps its own batch: pages, positions and tokens stay on the GPU.

    python examples/decode_loop.py [--batch 16] [--prompt 300] [--steps 64]

Every step is planned from the requests' lengths (luisaml_b200.kv_plan), runs the
layers (norm -> QKV GEMM -> norm and rotation of queries and keys -> cache write ->
attention with a window and sinks -> output GEMM -> FFN) and draws the next tokens
(luisaml_b200.sample), which are the next step's input. Prompts run as they come;
the steps are one CUDA graph, replayed: a request that has its tokens ends there,
its pages go back and its row takes the next one. Random weights; the replayed
steps' tokens are compared with the same steps run one by one.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import luisaml_b200 as lb  # noqa: E402
from decoder_layer import quantized_weight  # noqa: E402


class Decoder:
    """Weights, the layers' paged caches and the state of ``batch`` rows of up to ``max_len`` tokens."""

    def __init__(self, device, batch, max_len, vocab=32000, layers=2, q_heads=16, kv_heads=4, head_dim=128, ffn=2048, page=64, window=256, sinks=4):
        self.hq, self.hk, self.d, self.page, self.window, self.sinks = q_heads, kv_heads, head_dim, page, window, sinks
        width = q_heads * head_dim
        g = torch.Generator(device=device).manual_seed(0)
        torch.manual_seed(2)  # not the embedding's numbers: each token would be followed by itself
        self.embedding = torch.randn(vocab, width, generator=g, device=device).bfloat16()
        self.head = quantized_weight(vocab, width, device)
        self.norms = torch.rand(2 * layers + 1, width, generator=g, device=device) + 0.5
        self.qk_norms = torch.rand(layers, 2, head_dim, generator=g, device=device) + 0.5
        self.weights = [[quantized_weight(rows, cols, device) for rows, cols in
                         (((q_heads + 2 * kv_heads) * head_dim, width), (width, width), (2 * ffn, width), (width, ffn))] for _ in range(layers)]
        self.inv_freq = torch.tensor([10000.0 ** (-2.0 * i / head_dim) for i in range(head_dim // 2)], dtype=torch.float64, device=device)
        cols = -(-max_len // page)
        self.pages = batch * cols
        self.caches = []
        for _ in range(layers):
            codes = torch.zeros(2, self.pages, kv_heads, page, head_dim, dtype=torch.uint8, device=device)
            scales = torch.zeros(2, self.pages, kv_heads, 1, device=device)
            self.caches.append((codes[0], codes[1], scales[0], scales[1]))
        self.table = torch.full((batch, cols), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(self.pages, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), self.pages, dtype=torch.int32, device=device)
        self.held = torch.zeros(batch, dtype=torch.int32, device=device)

    def step(self, tokens, new, ended, max_tokens, draw):
        """Packed ``tokens`` of all rows, ``new`` of each, -> the next token of each row. ``draw``: sample()'s numbers and settings."""
        plan = lb.kv_plan(new, self.held, self.table, self.free, self.free_count, page_size=self.page, total=tokens.shape[0], ended=ended,
                          kv_len=self.held, free_count_out=self.free_count)
        n, x, h = tokens.shape[0], self.embedding[tokens.long()], None
        for i, (w, cache) in enumerate(zip(self.weights, self.caches)):
            qkv_w, out_w, up_w, down_w = w
            a, s, h = lb.rmsnorm_quantize(x, self.norms[2 * i], h, h_out=torch.empty_like(x))
            q, k, v = lb.gemm(a, qkv_w[0], s, qkv_w[1]).view(n, self.hq + 2 * self.hk, self.d).split((self.hq, self.hk, self.hk), 1)
            lb.qk_norm_rope(q, k, plan.positions, self.inv_freq, self.qk_norms[i, 0], self.qk_norms[i, 1], q_out=q, k_out=k)
            lb.kv_cache_write(*cache, k, v, self.table, plan.cu_tokens, plan.start)
            o = lb.kv_attention(q, *cache, self.table, plan.cu_tokens, plan.kv_len, max_tokens=max_tokens, window=self.window, sinks=self.sinks)
            a, s = lb.quantize_rows_dynamic(o.view(n, -1).float())
            a, s, h = lb.rmsnorm_quantize(lb.gemm(a, out_w[0], s, out_w[1]), self.norms[2 * i + 1], h, h_out=h)
            a, s = lb.quantize_rows_dynamic(lb.gemm(a, up_w[0], s, up_w[1], epilogue=lb.EPI_SILU_MUL, out_dtype=torch.float32))
            x = lb.gemm(a, down_w[0], s, down_w[1])
        last = (plan.cu_tokens[1:] - 1).long()
        a, s, _ = lb.rmsnorm_quantize(x[last], self.norms[-1], h[last])
        return lb.sample(lb.gemm(a, self.head[0], s, self.head[1], out_dtype=torch.float32), **draw)


def run(batch=16, prompt=300, steps=64, request=40, device="cuda:0", **sizes):
    """Returns (whether the replayed steps drew what single steps draw, ms of the prompts, ms per step, pages in use)."""
    lens = [max(1, prompt - 11 * b) for b in range(batch)]
    g = torch.Generator(device=device).manual_seed(1)
    prompts = torch.randint(0, sizes.get("vocab", 32000), (sum(lens),), generator=g, device=device).to(torch.int32)
    uniforms = torch.rand(steps + 1, batch, generator=g, device=device)
    fill = lambda v, t: torch.full((batch,), v, dtype=t, device=device)  # noqa: E731
    settings = {"temperature": fill(0.8, torch.float32), "top_k": fill(200, torch.int32), "top_p": fill(0.95, torch.float32)}
    one = fill(1, torch.int32)
    # a row's request ends after `request` steps, the rows' one after the other; its token then begins the next one
    ended = torch.tensor([[(i + 5 * b) % request == request - 1 for b in range(batch)] for i in range(steps)], device=device)
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)

    def begin():
        d = Decoder(device, batch, prompt + steps + 2, **sizes)
        return d, d.step(prompts, torch.tensor(lens, dtype=torch.int32, device=device), None, max(lens), {"uniform": uniforms[0], **settings})

    decoder, token = begin()
    single = []
    for i in range(steps):
        token = decoder.step(token, one, ended[i], 1, {"uniform": uniforms[i + 1], **settings})
        single.append(token)
    del decoder

    start.record()
    decoder, token = begin()
    stop.record()
    u, over, graph = uniforms[0].clone(), ended[0].clone(), torch.cuda.CUDAGraph()
    draw = {"uniform": u, **settings, "out": token}
    torch.cuda.synchronize()
    prompt_ms = start.elapsed_time(stop)
    with torch.cuda.graph(graph):
        decoder.step(token, one, over, 1, draw)
    replayed = torch.empty(steps, batch, dtype=torch.int32, device=device)
    start.record()
    for i in range(steps):
        u.copy_(uniforms[i + 1])
        over.copy_(ended[i])
        graph.replay()
        replayed[i].copy_(token)
    stop.record()
    torch.cuda.synchronize()
    same = all(torch.equal(a, b) for a, b in zip(replayed, single))
    if lb.device_error():
        raise RuntimeError(f"device error {lb.device_error()}")
    return same, prompt_ms, start.elapsed_time(stop) / steps, decoder.pages - int(decoder.free_count)


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--batch", type=int, default=16)
    p.add_argument("--prompt", type=int, default=300)
    p.add_argument("--steps", type=int, default=64)
    a = p.parse_args()
    same, prompt_ms, step_ms, pages = run(a.batch, a.prompt, a.steps)
    print(f"prompts (with the set-up): {prompt_ms:.3f} ms; a token of {a.batch} sequences: {step_ms:.3f} ms; {pages} pages in use; "
          f"replayed tokens {'equal' if same else 'DIFFER FROM'} those of single steps")


if __name__ == "__main__":
    main()
