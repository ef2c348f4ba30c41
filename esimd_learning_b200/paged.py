"""Serving with the paged 4-bit key/value cache: the decode chain's kernels
(chain.py) with the attention between them.

`PagedKV4Cache` owns the pages of all layers, the block tables and the free
list, all on the device; `PagedDecoder` runs a stack of layers over it, prompts
and single tokens alike:

    cache = PagedKV4Cache(layers=2, shape=SMALL, num_pages=64, max_requests=4, max_seq_len=512, device=dev)
    model = PagedDecoder([layer_weights(SMALL, seed=i, device=dev) for i in range(2)], SMALL, cache)
    out = model.forward(prompt_hidden, query_lens=[70, 33])      # prompts, ragged
    step = model.capture(2)                                       # one token a request, one CUDA graph
    step.hidden.copy_(next_hidden); step.replay()

One layer of a step:
  fused add+RMSNorm -> QKV projection (W8A16 up to 16 tokens, per-token FP8
  above), q/k-norm + RoPE, ``esimd_kv4_append`` of the new keys and values,
  ``esimd_kv4_attention``, the output projection, then the MLP as in chain.py.
``esimd_kv_plan`` opens the step: it hands out pages and computes slots and
positions from the request lengths on the device and advances them in place, so
a captured decode step needs no host work between replays.

`python -m esimd_learning_b200.paged` runs a small model and prints its rate.
"""
from __future__ import annotations

import dataclasses

import torch

from esimd_learning_b200.chain import ChainShape, SMALL, _quantize_rows, full_weights, rope_cache


def layer_weights(shape: ChainShape, seed: int = 0, device="cpu") -> dict:
    """chain.full_weights plus the output projection "o" [hidden, q_heads * head_dim]."""
    w = full_weights(shape, seed, device)
    gen = torch.Generator(device=device).manual_seed(seed + 10_000)
    w["o"] = _quantize_rows(torch.randn(shape.hidden, shape.num_q_heads * shape.head_dim, generator=gen, device=device) * 0.02)
    return w


class PagedKV4Cache:
    """Pages of 4-bit keys and values for `layers` layers and `max_requests` requests.

    pages: uint8 [layers, num_pages, kv_heads, page bytes]; one page number
    serves all layers.  scales: fp32 [layers, 2, kv_heads] (keys, values), to be
    calibrated; 1.0 keeps values between 2^-10 and 2688.  block_table,
    context_lens, free_pages and free_count are the planner's state.  Requests
    end at whole pages: max_seq_len is rounded up to one."""

    def __init__(self, layers: int, shape: ChainShape, num_pages: int, max_requests: int, max_seq_len: int, device,
                 page_size: int = 64):
        from esimd_learning_b200 import cabi

        self.page_size, self.max_requests, self.device = page_size, max_requests, device
        nbytes = cabi.lib().cek_kv4_page_bytes(page_size, shape.head_dim)
        if nbytes == 0:
            raise ValueError(f"page_size {page_size} or head_dim {shape.head_dim} is not supported")
        if max_seq_len > shape.max_position:  # RoPE would take the last position for all behind it
            raise ValueError(f"max_seq_len {max_seq_len} is beyond the {shape.max_position} positions of the shape")
        width = -(-max_seq_len // page_size)
        self.max_seq_len = width * page_size  # what the planner grants a row, and attention's bound
        i32 = dict(dtype=torch.int32, device=device)
        self.pages = torch.empty(layers, num_pages, shape.num_kv_heads, nbytes, dtype=torch.uint8, device=device)
        self.scales = torch.ones(layers, 2, shape.num_kv_heads, dtype=torch.float32, device=device)
        self.block_table = torch.zeros(max_requests, width, **i32)
        self.context_lens = torch.zeros(max_requests, **i32)
        self.free_pages = torch.arange(num_pages, **i32)
        self.free_count = torch.tensor([num_pages], **i32)

    def release(self, request: int) -> None:
        """Returns a request's pages to the stack and empties its row (host bookkeeping between steps: synchronises)."""
        n = int(self.context_lens[request])
        n = ~n if n < 0 else n  # refused
        used = -(-n // self.page_size)
        count = int(self.free_count)
        self.free_pages[count:count + used] = self.block_table[request, :used]
        self.free_count += used
        self.context_lens[request] = 0

    def refused(self) -> list:
        """Requests that the last plan could not serve (no pages left, or longer than max_seq_len)."""
        return (self.context_lens < 0).nonzero().flatten().tolist()


class _Step:
    """A captured decode step: write `hidden`, replay, read `output`.  Holds what the graph reads besides: the
    lengths, and the model with its weights and cache."""

    def __init__(self, hidden, query_lens, output, graph, model):
        self.hidden, self.query_lens, self.output, self.graph, self.model = hidden, query_lens, output, graph, model

    def replay(self):
        self.graph.replay()
        return self.output


class PagedDecoder:
    """A stack of layers (layer_weights dicts) over a PagedKV4Cache.  Rows of every request lie side by side, in the
    order of the cache's rows; fp16."""

    def __init__(self, layers: list, shape: ChainShape, cache: PagedKV4Cache, window: int = 0):
        import esimd_learning_b200 as ops

        self.ops, self.shape, self.cache, self.window = ops, shape, cache, window
        dev = cache.device
        self.layers = [{k: tuple(t.to(dev) for t in v) if isinstance(v, tuple) else v.to(dev) for k, v in w.items()} for w in layers]
        # the cache's last page may reach past the shape's positions
        self.cos_sin = rope_cache(dataclasses.replace(shape, max_position=max(shape.max_position, cache.max_seq_len)), dev)

    def _project(self, x, weight, scale):
        """x [T, K] @ weight^T: the GEMV family up to 16 tokens, per-token FP8 on the tensor cores above."""
        o, T = self.ops, x.shape[0]
        y = torch.empty(T, weight.shape[0], dtype=x.dtype, device=x.device)
        if T <= 16:
            return o.esimd_gemv_fp8_pern(x, weight, scale, y, weight.shape[0], weight.shape[1])
        q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
        s = torch.empty(T, dtype=torch.float32, device=x.device)
        o.esimd_quant_fp8_per_token(x, q, s)
        return o.esimd_gemm_fp8_pertoken_pern(q, s, weight, scale, y)

    def _norm_project(self, hidden, residual, gamma, weight, scale):
        """residual += hidden; RMSNorm(residual) * gamma @ weight^T."""
        o, T = self.ops, hidden.shape[0]
        if T <= 16:
            y = torch.empty(T, weight.shape[0], dtype=hidden.dtype, device=hidden.device)
            return o.esimd_fused_add_rms_norm_batched_fp8(hidden, residual, gamma, self.shape.eps, weight, scale, y)
        return self._project(o.esimd_fused_add_rms_norm_batched(hidden, residual, gamma, self.shape.eps), weight, scale)

    def _mlp(self, hidden, residual, w):
        o, T, f = self.ops, hidden.shape[0], self.shape.intermediate
        act = torch.empty(T, f, dtype=hidden.dtype, device=hidden.device)
        if T <= 16:
            o.esimd_fused_add_rms_norm_gelu_mul_fp8(hidden, residual, w["gamma_mlp"], self.shape.eps, *w["gate_up"], act)
        else:
            o.esimd_gelu_and_mul(self._norm_project(hidden, residual, w["gamma_mlp"], *w["gate_up"]), act)
        return self._project(act, *w["down"])

    def _run(self, hidden, query_lens, tokens, max_query_len):
        """hidden [tokens, hidden]; query_lens int32 [max_requests] on the device."""
        o, s, c, dev = self.ops, self.shape, self.cache, self.cache.device
        hq, hkv, d = s.num_q_heads, s.num_kv_heads, s.head_dim
        positions = torch.empty(tokens, dtype=torch.int64, device=dev)
        slots = torch.empty_like(positions)
        start = torch.empty(c.max_requests + 1, dtype=torch.int32, device=dev)
        # context_lens becomes this step's sequence lengths, free_count what is left
        o.esimd_kv_plan(query_lens, c.context_lens, c.block_table, c.free_pages, c.free_count, c.page_size, start,
                        c.context_lens, c.free_count, positions, slots)
        residual = torch.zeros_like(hidden)
        for i, w in enumerate(self.layers):
            qkv = self._norm_project(hidden, residual, w["gamma_attn"], *w["qkv"])
            o.esimd_qkv_norm_rope(qkv, positions, w["q_norm"], w["k_norm"], self.cos_sin, hq, hkv, d, s.eps, True)
            heads = qkv.view(tokens, hq + 2 * hkv, d)
            o.esimd_kv4_append(heads[:, hq:hq + hkv], heads[:, hq + hkv:], c.scales[i], slots, c.pages[i], c.page_size)
            attn = torch.zeros(tokens, hq, d, dtype=hidden.dtype, device=dev)
            o.esimd_kv4_attention(heads[:, :hq], c.pages[i], c.scales[i], c.block_table, start, c.context_lens, attn,
                                  c.page_size, d ** -0.5, max_query_len, c.max_seq_len, self.window)
            self.last = dict(qkv=heads, attention=attn, start=start)
            hidden = self._mlp(self._project(attn.view(tokens, hq * d), *w["o"]), residual, w)
        return hidden + residual

    def forward(self, hidden, query_lens: list):
        """New tokens of every request (query_lens[i] of them, 0 for none), rows side by side in `hidden`
        [sum, hidden] fp16; returns the stack's output for each."""
        c = self.cache
        lens = list(query_lens) + [0] * (c.max_requests - len(query_lens))
        if hidden.shape[0] != sum(lens):
            raise ValueError(f"hidden has {hidden.shape[0]} rows for {sum(lens)} tokens")
        n = torch.tensor(lens, dtype=torch.int32, device=c.device)
        return self._run(hidden.clone(), n, hidden.shape[0], max(lens, default=0))

    def capture(self, requests: int) -> _Step:
        """One token for each of the first `requests` rows as a CUDA graph (at most 16: the decode kernels)."""
        if not 1 <= requests <= min(16, self.cache.max_requests):
            raise ValueError("1 to 16 requests, within the cache's rows")
        dev = self.cache.device
        hidden = torch.zeros(requests, self.shape.hidden, dtype=torch.float16, device=dev)
        n = torch.zeros(self.cache.max_requests, dtype=torch.int32, device=dev)
        n[:requests] = 1
        st = torch.cuda.Stream(dev)
        st.wait_stream(torch.cuda.current_stream(dev))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st), torch.cuda.graph(graph, stream=st):
            output = self._run(hidden, n, requests, 1)
        torch.cuda.current_stream(dev).wait_stream(st)
        return _Step(hidden, n, output, graph, self)


def main() -> None:
    dev = torch.device("cuda")
    layers, requests, steps, warm = 4, 8, 64, 8
    cache = PagedKV4Cache(layers, SMALL, num_pages=requests * 8, max_requests=requests, max_seq_len=512, device=dev)
    model = PagedDecoder([layer_weights(SMALL, seed=i, device=dev) for i in range(layers)], SMALL, cache)
    gen = torch.Generator(device=dev).manual_seed(0)
    prompts = [37 + 41 * i for i in range(requests)]
    hidden = torch.randn(sum(prompts), SMALL.hidden, generator=gen, device=dev).half()
    out = model.forward(hidden, prompts)
    last = out[torch.tensor(prompts, device=dev).cumsum(0) - 1]
    step = model.capture(requests)
    step.hidden.copy_(last)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for i in range(warm + steps):
        if i == warm:
            torch.cuda.synchronize()
            begin.record()
        step.hidden.copy_(torch.nn.functional.normalize(step.replay().float(), dim=-1).mul_(SMALL.hidden ** 0.5))
    end.record()
    torch.cuda.synchronize()
    ms = begin.elapsed_time(end) / steps
    print(f"{layers} layers, {requests} requests after prompts of {min(prompts)}..{max(prompts)} tokens: "
          f"{ms * 1e3:.1f} us a step, {requests / ms * 1e3:.0f} tokens/s, lengths {cache.context_lens.tolist()}, "
          f"{int(cache.free_count)} pages left")


if __name__ == "__main__":
    main()
