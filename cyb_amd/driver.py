"""A soma-style driver over the linear stack: the caller loop of the op, reporting in
the reference's own units.

The reference's mind streams events to its UI while it answers -
`Prefill { done, total }` while it reads the question, one `Delta` per generated
piece, then `Answer { tokens, tok_per_s, tok_in_s, tok_out_s, .. }`
(/root/reference/shell/src/worlds/soma_bridge.rs:252-277); the UI keeps running
means of `tok_in_s` / `tok_out_s` (/root/reference/shell/src/worlds/models/mod.rs:44-52)
and compares them with `SPEED_ANCHORS` (same file, :116).  This module walks the
same two phases over the quantised linears only (with --experts, over the router and the experts of every layer too; with
--cache, over whole layers: norms, RoPE, the paged cache and its attention among them):

  prefill  the prompt in chunks of `chunk` tokens, every chunk one pass of
           `cybq_matmul_many` over the stack with bf16 activations (M = chunk),
  decode   one pass per new token with f16 activations (M = batch).

With a cache each of the `batch` conversations reads the prompt and keeps it.  Without one, attention, norms
and RoPE are not part of the path, so the rates are those of the weight-bound part of a step; they are upper
bounds for a whole model.  Sampling and the tokenizer never are.  Nothing is computed on the host.
"""
from __future__ import annotations

import time
from dataclasses import dataclass
from typing import Dict, Iterator, Optional

from . import stack as stk
from .backend import Backend


@dataclass
class Answer:
    tokens: int            # generated tokens
    tok_per_s: float       # (prompt + generated) / wall time of the whole ask
    tok_in_s: float        # prompt tokens / prefill time
    tok_out_s: float       # generated tokens / decode time


def ask(backend: Backend, st, prompt_tokens: int, new_tokens: int, chunk: int = 512,
        batch: int = 1, shapes: Optional[Dict[str, tuple]] = None, stream: int = 0) -> Iterator[dict]:
    """Walks a LinearStack, an ExpertStack or a CachedStack.  Yields {"Prefill": {"done", "total"}} per chunk, {"Delta": i} per decode step and finally
    {"Answer": Answer}.  Device work is timed with events on the launch stream."""
    import torch
    if prompt_tokens < 0 or new_tokens < 0 or chunk < 1 or batch < 1 or batch > 16:
        raise ValueError("prompt_tokens, new_tokens >= 0; chunk >= 1; 1 <= batch <= 16")
    cached = isinstance(st, stk.CachedStack)
    if cached and (batch > st.conversations or prompt_tokens + new_tokens + 1 > st.context):
        raise ValueError("the cache has fewer conversations, or pages for fewer tokens")
    launch = torch.cuda.ExternalStream(stream, device=backend.device) if stream else torch.cuda.default_stream(backend.device)

    def on_launch(f, *args, **kw):                             # torch's own work among the steps': buffers, lengths
        with torch.cuda.stream(launch):
            return f(*args, **kw)

    torch.cuda.synchronize(backend.device)                     # the stack was made on whatever stream was current
    if cached:
        on_launch(st.set_lengths, 0)
    read = prompt_tokens * batch if cached else prompt_tokens
    t_wall = time.time()
    yield {"Prefill": {"done": 0, "total": read}}
    ms_in = 0.0
    steps = {}

    def step_for(M: int, xdtype):
        if M not in steps:
            steps[M] = on_launch(stk.stepper, st, M, shapes=shapes, xdtype=xdtype)
        return steps[M]

    done = 0
    while done < read:
        M = min(chunk, prompt_tokens - done % prompt_tokens)
        step = step_for(M, torch.bfloat16 if M > 16 else torch.float16)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record(launch)
        step(stream, done // prompt_tokens) if cached else step(stream)
        b.record(launch)
        b.synchronize()
        ms_in += a.elapsed_time(b)
        done += M
        yield {"Prefill": {"done": done, "total": read}}

    ms_out = 0.0
    if new_tokens:
        step = on_launch(st.stepper, batch, torch.float16, count=batch) if cached else step_for(batch, torch.float16)
        step(stream)                                           # first touch of this plan's buffers, untimed
        torch.cuda.synchronize()
        if cached:
            on_launch(st.set_lengths, prompt_tokens, batch)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record(launch)
        for i in range(new_tokens):
            step(stream)
        b.record(launch)
        b.synchronize()
        ms_out = a.elapsed_time(b)
        for i in range(new_tokens):
            yield {"Delta": i}
    wall = max(time.time() - t_wall, 1e-9)
    yield {"Answer": Answer(tokens=new_tokens * batch,
                            tok_per_s=(read + new_tokens * batch) / wall,
                            tok_in_s=read / (ms_in * 1e-3) if ms_in else 0.0,
                            tok_out_s=new_tokens * batch / (ms_out * 1e-3) if ms_out else 0.0)}


def main(argv=None) -> int:
    import argparse
    ap = argparse.ArgumentParser(description="prefill / decode rates of the quantised linear stack (Llama-3-8B shapes, random init)")
    ap.add_argument("--prompt", type=int, default=2048)
    ap.add_argument("--new", type=int, default=128)
    ap.add_argument("--chunk", type=int, default=512)
    ap.add_argument("--batch", type=int, default=1)
    ap.add_argument("--layers", type=int, default=32)
    ap.add_argument("--separate", action="store_true", help="q/k/v and gate/up as separate launches (224 per step)")
    ap.add_argument("--epilogues", action="store_true", help="SwiGLU and residual adds fused into the linears")
    ap.add_argument("--experts", type=int, default=0, help="FFNs of this many experts (hidden 2048, width 768) instead of the Llama-3-8B shapes")
    ap.add_argument("--top-k", type=int, default=8, help="experts per token")
    ap.add_argument("--cache", choices=["f16", "bf16", "q8", "q4"], help="whole layers, with a cache of this kind")
    ap.add_argument("--window", type=int, default=0, help="tokens that attention looks back at (with --cache; 0: all)")
    args = ap.parse_args(argv)
    if args.cache and (args.experts or args.separate):
        ap.error("--cache walks whole layers of the Llama-3-8B shapes")
    import torch
    torch.cuda.init()          # torch brings its own HIP runtime: let it find the device before libcybq does
    be = Backend(0)
    shapes = None if args.separate else stk.fused_shapes()
    if args.experts:
        st = stk.build_experts(be, layers=args.layers, experts=args.experts, top_k=args.top_k)
    elif args.cache:
        st = stk.build_cached(be, layers=args.layers, kind=args.cache, conversations=args.batch, context=args.prompt + args.new + 1,
                              window=args.window)
    else:
        st = stk.build(be, layers=args.layers, shapes=shapes, order=list(shapes) if shapes else None,
                       epilogues=args.epilogues and shapes is not None)
    for ev in ask(be, st, args.prompt, args.new, args.chunk, args.batch, shapes=shapes):
        if "Prefill" in ev:
            p = ev["Prefill"]
            print(f"reading {p['done']} / {p['total']}", flush=True)
        elif "Answer" in ev:
            a = ev["Answer"]
            print(f"tokens {a.tokens}  tok_in_s {a.tok_in_s:.1f}  tok_out_s {a.tok_out_s:.1f}  tok_per_s {a.tok_per_s:.1f}  "
                  f"({st.weight_bytes / 1e9:.2f} GB of Q{st.bits} weights, {len(st.nodes)} launches per step)", flush=True)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
