"""A decoder layer on FP8 GEMMs with a paged e4m3 key/value cache: prompts of
different lengths, then token by token from a CUDA graph.

    python examples/decoder_layer.py [--batch 16] [--prompt 500] [--steps 64]

One step is ten calls of luisaml_b200: norm (with the residual's addition) ->
QKV GEMM -> cache write -> attention -> row quantization -> output GEMM -> norm
-> FFN up (SiLU(gate) * up in the GEMM) -> row quantization -> FFN down. The
prompt's and the steps' outputs are checked against the same layer in plain
torch with fp32 arithmetic, weights decoded and no cache.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import luisaml_b200 as lb  # noqa: E402


def quantized_weight(rows, cols, device):
    """[rows, cols] e4m3 codes and a scale per row (an output column of the GEMM)."""
    return lb.quantize_rows_dynamic(torch.randn(rows, cols, device=device) / cols**0.5)


class DecoderLayer:
    """Weights of a layer and the paged cache of up to ``batch`` sequences of ``max_len`` tokens."""

    def __init__(self, device, batch, max_len, q_heads=32, kv_heads=8, head_dim=128, ffn=11008, page=64):
        self.hq, self.hk, self.d = q_heads, kv_heads, head_dim
        width = q_heads * head_dim
        self.norm1 = torch.rand(width, device=device) + 0.5
        self.norm2 = torch.rand(width, device=device) + 0.5
        self.qkv = quantized_weight((q_heads + 2 * kv_heads) * head_dim, width, device)
        self.proj = quantized_weight(width, width, device)
        self.up = quantized_weight(2 * ffn, width, device)  # 128 gate rows, 128 up rows, and so on
        self.down = quantized_weight(width, ffn, device)
        per_seq = -(-max_len // page)
        pages = batch * per_seq
        self.k = torch.zeros(pages, kv_heads, page, head_dim, dtype=torch.uint8, device=device)
        self.v = torch.zeros_like(self.k)
        self.ks = torch.zeros(pages, kv_heads, 1, device=device)
        self.vs = torch.zeros_like(self.ks)
        self.table = torch.randperm(pages, device=device).to(torch.int32).view(batch, per_seq)  # any order of pages
        self.held = torch.zeros(batch, dtype=torch.int32, device=device)  # tokens in the cache

    def forward(self, x, residual, cu_tokens, max_tokens):
        """x (+ residual) [tokens, width] bf16 of a ragged batch -> (output, its residual stream)."""
        tokens = x.shape[0]
        cache = (self.k, self.v, self.ks, self.vs)
        a, s, h = lb.rmsnorm_quantize(x, self.norm1, residual, h_out=torch.empty_like(x))
        qkv = lb.gemm(a, self.qkv[0], s, self.qkv[1]).view(tokens, self.hq + 2 * self.hk, self.d)
        q, k, v = qkv.split((self.hq, self.hk, self.hk), dim=1)
        lb.kv_cache_write(*cache, k, v, self.table, cu_tokens, self.held)
        self.held += cu_tokens[1:] - cu_tokens[:-1]
        o = lb.kv_attention(q, *cache, self.table, cu_tokens, self.held, max_tokens=max_tokens)
        a, s = lb.quantize_rows_dynamic(o.view(tokens, -1).float())
        y = lb.gemm(a, self.proj[0], s, self.proj[1])
        a, s, h = lb.rmsnorm_quantize(y, self.norm2, h, h_out=h)
        f = lb.gemm(a, self.up[0], s, self.up[1], epilogue=lb.EPI_SILU_MUL, out_dtype=torch.float32)
        a, s = lb.quantize_rows_dynamic(f)
        return lb.gemm(a, self.down[0], s, self.down[1]), h

    def plain(self, x):
        """The layer over one whole sequence [tokens, width] in fp32, without a cache."""
        def decoded(w):
            return w[0].view(torch.float8_e4m3fn).float() * w[1][:, None]

        def norm(h, w):
            return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w

        n, group = x.shape[0], self.hq // self.hk
        h = x.float()
        qkv = (norm(h, self.norm1) @ decoded(self.qkv).T).view(n, -1, self.d).transpose(0, 1)
        q, k, v = qkv.split((self.hq, self.hk, self.hk))
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        seen = torch.ones(n, n, dtype=torch.bool, device=x.device).tril()
        p = (q @ k.transpose(1, 2) / self.d**0.5).masked_fill(~seen, float("-inf")).softmax(-1)
        h = h + (p @ v).transpose(0, 1).reshape(n, -1) @ decoded(self.proj).T
        f = (norm(h, self.norm2) @ decoded(self.up).T).view(n, -1, 2, 128)
        return (torch.nn.functional.silu(f[:, :, 0]) * f[:, :, 1]).reshape(n, -1) @ decoded(self.down).T + h


def relative_error(got, want):
    return ((got.float() - want).norm() / want.norm()).item()


def run(batch=16, prompt=500, steps=64, device="cuda:0", check=2, **sizes):
    """Returns (relative error of the prompts, of the steps, ms of the prompts, ms per step)."""
    torch.manual_seed(0)
    lens = [max(1, prompt - 13 * b) for b in range(batch)]
    layer = DecoderLayer(device, batch, prompt + steps + 4, **sizes)
    width = layer.hq * layer.d
    seqs = [torch.randn(n + steps + 4, width, device=device).bfloat16() for n in lens]
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)

    cu = torch.tensor([0] + lens, device=device).cumsum(0).to(torch.int32)
    x = torch.cat([s[:n] for s, n in zip(seqs, lens)])
    layer.forward(x, None, cu, max(lens))  # warm up, then forget it
    layer.held.zero_()
    start.record()
    out, h = layer.forward(x, None, cu, max(lens))
    stop.record()
    full = (out.float() + h.float()).split(lens)
    torch.cuda.synchronize()
    prompt_ms = start.elapsed_time(stop)

    # one token of every sequence, captured once
    cu1 = torch.arange(batch + 1, dtype=torch.int32, device=device)
    x1 = torch.stack([s[n] for s, n in zip(seqs, lens)])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.forward(x1, None, cu1, 1)  # warm up: the same tokens are written again below
        layer.held -= 1
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y1, h1 = layer.forward(x1, None, cu1, 1)
    got = []
    for i in range(steps):
        x1.copy_(torch.stack([s[n + i] for s, n in zip(seqs, lens)]))
        graph.replay()
        got.append(y1.float() + h1.float())
    start.record()
    for _ in range(4):
        graph.replay()
    stop.record()
    torch.cuda.synchronize()

    prompt_error = step_error = 0.0
    for b in range(min(check, batch)):
        want = layer.plain(seqs[b][:lens[b] + steps])
        prompt_error = max(prompt_error, relative_error(full[b], want[:lens[b]]))
        step_error = max(step_error, relative_error(torch.stack([g[b] for g in got]), want[lens[b]:]))
    if lb.device_error():
        raise RuntimeError(f"device error {lb.device_error()}")
    return prompt_error, step_error, prompt_ms, start.elapsed_time(stop) / 4


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--batch", type=int, default=16)
    p.add_argument("--prompt", type=int, default=500)
    p.add_argument("--steps", type=int, default=64)
    a = p.parse_args()
    prompt_error, step_error, prompt_ms, step_ms = run(a.batch, a.prompt, a.steps)
    print(f"prompts: {prompt_ms:.3f} ms, relative error {prompt_error:.4f}; "
          f"a token of {a.batch} sequences: {step_ms:.3f} ms, relative error {step_error:.4f}")


if __name__ == "__main__":
    main()
