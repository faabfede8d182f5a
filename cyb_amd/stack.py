"""The decode-step linear stack: the caller loop around the op.

One decode step of a LlamaStyle model issues, per layer, the quantised matmuls
q, k, v, o, gate, up, down ("norm -> QKV -> RoPE -> KV cache -> attention -> O
proj -> residual -> norm -> FFN -> residual" x layers -
/root/reference/decide/pipeline.md:51).  This module builds that list of graph
nodes for a random-init Llama-3-8B-shaped model and runs it through
`cybq_matmul_many`.  The glue between the linears (norm, RoPE, attention,
SwiGLU) is not part of LinearStack's path: every linear reads a fresh seeded N(0,1) f16
input of its width, so each output can be checked on its own.  CachedStack runs whole
layers, the cache and its attention among them.

Weights are generated and quantised on the device (torch.randn ->
cybq_quantize -> cybq_weight_from_device): 7 B weights never exist on the host.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Optional

from . import formats, synth
from .backend import Backend, CybqError, KVCache, QMatMul, QWeight

LINEAR_ORDER = ["q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"]
_PREFIX = {"q_proj": "self_attn", "k_proj": "self_attn", "v_proj": "self_attn", "o_proj": "self_attn",
           "gate_proj": "mlp", "up_proj": "mlp", "down_proj": "mlp"}


def tensor_name(layer: int, lin: str) -> str:
    return f"model.layers.{layer}.{_PREFIX.get(lin, 'fused')}.{lin}.weight"


@dataclass
class LinearStack:
    backend: Backend
    layers: int
    bits: int
    nodes: List[QMatMul] = field(default_factory=list)
    weights: List[QWeight] = field(default_factory=list)
    planar: Dict[str, tuple] = field(default_factory=dict)     # name -> (q bytes, scales) kept for checks
    epilogues: List[str] = field(default_factory=list)         # per node: "none" | "add" | "swiglu" (empty = none anywhere)
    gammas: List[object] = field(default_factory=list)         # per node: RMSNorm weight folded in front of it, or None (empty = no norms)
    eps: float = 1e-5

    @property
    def weight_bytes(self) -> int:
        return sum(w.algorithmic_bytes for w in self.weights)

    def step_bytes(self, M: int) -> int:
        """Algorithmic HBM bytes of one step: every weight once, f16 inputs, f32 outputs."""
        return sum(formats.matmul_bytes(self.bits, w.N, w.K, M, 2, 4) for w in self.weights)


def fused_shapes(shapes: Dict[str, tuple] = None) -> Dict[str, tuple]:
    """q/k/v and gate/up read the same input: concatenating their rows at load time
    turns five launches into two (the outputs are column slices of one y)."""
    shapes = shapes or synth.LLAMA3_8B_LINEARS
    K = shapes["q_proj"][0]
    return {"qkv_proj": (K, shapes["q_proj"][1] + shapes["k_proj"][1] + shapes["v_proj"][1]),
            "o_proj": shapes["o_proj"],
            "gate_up_proj": (K, shapes["gate_proj"][1] + shapes["up_proj"][1]),
            "down_proj": shapes["down_proj"]}


NORMED = ("q_proj", "k_proj", "v_proj", "qkv_proj", "gate_proj", "up_proj", "gate_up_proj")      # linears that follow an RMSNorm


def build(backend: Backend, layers: int = 32, bits: int = formats.Q4, seed: int = 5, keep_planar=0,
          shapes: Dict[str, tuple] = None, order: List[str] = None, epilogues: bool = False, norms: bool = False) -> LinearStack:
    """Random-init stack with N(0, 0.02) weights quantised on the device.

    keep_planar: for the first that many layers (or for the layers listed), the PLANAR device
    buffers are kept in `stack.planar` so that a checker can pull them back and recompute outputs.
    epilogues: with the fused shapes, `gate_up_proj` becomes a strip-interleaved pair run with the
    SwiGLU epilogue (its output has half the columns) and `o_proj` / `down_proj` add a residual.
    norms: the linears that follow an RMSNorm in the decode loop (q / k / v, gate / up) get a seeded
    gamma (f16, 1 +- 0.1) per layer and norm, folded into their activation load."""
    import torch
    shapes = shapes or synth.LLAMA3_8B_LINEARS
    st = LinearStack(backend, layers, bits)
    gen = torch.Generator(device="cuda")
    gen.manual_seed((synth.BASE_SEED ^ seed) & 0x7FFFFFFF)
    order = order or [l for l in LINEAR_ORDER if l in shapes] or list(shapes)
    kept = set(range(keep_planar)) if isinstance(keep_planar, int) else set(keep_planar)
    for layer in range(layers):
        layer_gamma = {}
        for lin in order:
            K, N = shapes[lin]
            w = torch.empty((N, K), dtype=torch.float32, device="cuda").normal_(0.0, 0.02, generator=gen)
            qd = torch.empty(N * K * bits // 8, dtype=torch.uint8, device="cuda")
            sd = torch.empty(N * (K // 32), dtype=torch.int16, device="cuda")
            backend.quantize(bits, w, N, K, qd, sd)
            name = tensor_name(layer, lin)
            epi = "none"
            if epilogues and lin == "gate_up_proj":
                # rows [0, N/2) are the gate projection, [N/2, N) the up projection
                h = N // 2
                hq, hs = h * K * bits // 8, h * (K // 32)
                g = backend.weight_from_device(bits, h, K, qd[:hq], sd[:hs])
                u = backend.weight_from_device(bits, h, K, qd[hq:], sd[hs:])
                torch.cuda.synchronize()
                qw = backend.fuse_pairs(g, u, name=name)
                g.free()
                u.free()
                epi = "swiglu"
            else:
                qw = backend.weight_from_device(bits, N, K, qd, sd, name=name)
                if epilogues and lin in ("o_proj", "down_proj"):
                    epi = "add"
            torch.cuda.synchronize()              # qd / sd / w are released below
            st.weights.append(qw)
            st.nodes.append(QMatMul(w=name, x=f"in.{K}", y=f"out.{lin}", quant=bits, M=1, N=N, K=K))
            if epilogues:
                st.epilogues.append(epi)
            if norms:
                which = "input" if lin in ("q_proj", "k_proj", "v_proj", "qkv_proj") else "post_attention"
                if lin in NORMED and which not in layer_gamma:
                    layer_gamma[which] = (1.0 + 0.1 * torch.empty(K, dtype=torch.float32, device="cuda").normal_(generator=gen)).to(torch.float16)
                st.gammas.append(layer_gamma[which] if lin in NORMED else None)
            if layer in kept:
                st.planar[name] = (qd, sd)
            del w
    return st


def edges_for(stack: LinearStack, M: int, seed: int = 5, shapes: Dict[str, tuple] = None, xdtype=None):
    """Fresh seeded inputs (one per input width; f16 unless `xdtype` says otherwise) and f32
    outputs (one per linear kind)."""
    import torch
    shapes = shapes or synth.LLAMA3_8B_LINEARS
    edges = {}
    for i, K in enumerate(sorted({k for k, _ in shapes.values()})):
        x = torch.from_numpy(synth.activations(seed, M, K, stream=i)).cuda().to(xdtype or torch.float16)
        edges[f"in.{K}"] = x
    for lin in shapes:
        cols = shapes[lin][1] // 2 if (stack.epilogues and lin == "gate_up_proj") else shapes[lin][1]
        edges[f"out.{lin}"] = torch.empty((M, cols), dtype=torch.float32, device="cuda")
    if stack.epilogues:
        widths = sorted({shapes[lin][1] for lin in ("o_proj", "down_proj") if lin in shapes})
        for i, N in enumerate(widths):          # the residual stream entering o_proj / down_proj
            edges[f"res.{N}"] = torch.from_numpy(synth.activations(seed, M, N, stream=100 + i)).cuda()
    return edges


def plan(stack: LinearStack, edges):
    xs, ys = [edges[n.x] for n in stack.nodes], [edges[n.y] for n in stack.nodes]
    gammas = stack.gammas or None
    if not stack.epilogues:
        return stack.backend.plan_many(stack.weights, xs, ys, gammas=gammas, eps=stack.eps)
    res = [edges[f"res.{n.N}"] if e == "add" else None for n, e in zip(stack.nodes, stack.epilogues)]
    return stack.backend.plan_many(stack.weights, xs, ys, stack.epilogues, res, gammas=gammas, eps=stack.eps)


def stepper(stack, M: int, shapes: Dict[str, tuple] = None, xdtype=None):
    """One step of M rows as a call: step(stream).  The plan and its buffers live as long as the call does."""
    if isinstance(stack, (ExpertStack, CachedStack)):
        return stack.stepper(M, xdtype)
    edges = edges_for(stack, M, shapes=shapes, xdtype=xdtype)
    p = plan(stack, edges)

    def step(stream: int = 0) -> None:
        stack.backend.matmul_many(p, M, stream)
    step.edges = edges
    return step


@dataclass
class ExpertStack:
    """The decode-step stack of a model whose FFNs are mixtures of experts: per layer q/k/v and o as in LinearStack, a router
    (a Q8 linear, then Backend.route) and the experts' gate / up and down (matmul_experts, matmul_experts_sum), the
    residual added on the way back."""
    backend: Backend
    layers: int
    bits: int
    experts: int
    top_k: int
    hidden: int
    width: int
    qkv: List[QWeight] = field(default_factory=list)
    o: List[QWeight] = field(default_factory=list)
    router: List[QWeight] = field(default_factory=list)
    gate_up: List[QWeight] = field(default_factory=list)      # fuse_pairs of [experts * width, hidden] twice
    down: List[QWeight] = field(default_factory=list)         # [experts * hidden, width]

    @property
    def weights(self) -> List[QWeight]:
        return self.qkv + self.o + self.router + self.gate_up + self.down

    @property
    def weight_bytes(self) -> int:
        return sum(w.algorithmic_bytes for w in self.weights)

    @property
    def nodes(self) -> List[str]:
        """The calls of one step."""
        return ["qkv", "o", "router", "route", "gate_up", "down"] * self.layers

    def stepper(self, M: int, xdtype=None, seed: int = 5):
        import torch
        xdtype = xdtype or torch.float16
        be, dev = self.backend, f"cuda:{self.backend.device}"
        b = {"x": torch.from_numpy(synth.activations(seed, M, self.hidden)).to(dev).to(xdtype),
             "attn": torch.from_numpy(synth.activations(seed, M, self.hidden, stream=1)).to(dev).to(xdtype),
             "mid": torch.empty((M, self.hidden), dtype=xdtype, device=dev),
             "qkv": torch.empty((M, self.qkv[0].N), dtype=torch.float32, device=dev),
             "logits": torch.empty((M, self.experts), dtype=torch.float32, device=dev),
             "ids": torch.empty((M, self.top_k), dtype=torch.int32, device=dev),
             "weights": torch.empty((M, self.top_k), dtype=torch.float32, device=dev),
             "h": torch.empty((M * self.top_k, self.width), dtype=xdtype, device=dev),
             "y": torch.empty((M, self.hidden), dtype=xdtype, device=dev)}

        def step(stream: int = 0) -> None:
            for i in range(self.layers):
                be.matmul(self.qkv[i], b["x"], b["qkv"], stream=stream)
                be.matmul_ex(self.o[i], b["attn"], b["mid"], "add", b["x"], stream=stream)
                be.matmul(self.router[i], b["mid"], b["logits"], stream=stream)
                be.route(b["logits"], b["ids"], b["weights"], stream=stream)
                be.matmul_experts(self.gate_up[i], self.experts, b["mid"], b["ids"], b["h"], "swiglu", stream=stream)
                be.matmul_experts_sum(self.down[i], self.experts, b["h"], b["ids"], b["weights"], b["y"], b["mid"], stream=stream)
        step.edges = b
        return step


def build_experts(backend: Backend, layers: int = 4, bits: int = formats.Q4, experts: int = 128, top_k: int = 8, hidden: int = 2048,
                  width: int = 768, qkv: int = None, seed: int = 5) -> ExpertStack:
    """Random-init stack of expert layers with N(0, 0.02) weights quantised on the device, a stack of experts at a time."""
    import torch
    if width % 32 or hidden % 32 or not 1 <= top_k <= experts:
        raise CybqError(-2, "bad shape", "hidden and width must be multiples of 32, top_k in 1 .. experts")
    st = ExpertStack(backend, layers, bits, experts, top_k, hidden, width)
    dev = f"cuda:{backend.device}"
    gen = torch.Generator(device=dev)
    gen.manual_seed((synth.BASE_SEED ^ seed) & 0x7FFFFFFF)

    def tensor(quant: int, N: int, K: int, name: str = None) -> QWeight:
        q = torch.empty(N * K * quant // 8, dtype=torch.uint8, device=dev)
        s = torch.empty(N * (K // 32), dtype=torch.int16, device=dev)
        rows = max(16, (1 << 26) // K // 16 * 16)                     # a quarter of a gigabyte of fp32 at a time
        for r in range(0, N, rows):
            n = min(rows, N - r)
            w = torch.empty((n, K), dtype=torch.float32, device=dev).normal_(0.0, 0.02, generator=gen)
            backend.quantize(quant, w, n, K, q[r * K * quant // 8:], s[r * (K // 32):])
            torch.cuda.synchronize()
        out = backend.weight_from_device(quant, N, K, q, s, name=name)
        torch.cuda.synchronize()                                      # q and s are released
        return out

    for i in range(layers):
        st.qkv.append(tensor(bits, qkv or hidden * 5 // 4, hidden, tensor_name(i, "qkv_proj")))
        st.o.append(tensor(bits, hidden, hidden, tensor_name(i, "o_proj")))
        st.router.append(tensor(formats.Q8, experts, hidden, f"model.layers.{i}.mlp.gate.weight"))
        gate, up = tensor(bits, experts * width, hidden), tensor(bits, experts * width, hidden)
        st.gate_up.append(backend.fuse_pairs(gate, up, name=f"model.layers.{i}.mlp.experts.gate_up_proj.weight"))
        gate.free()
        up.free()
        st.down.append(tensor(bits, experts * hidden, width, f"model.layers.{i}.mlp.experts.down_proj.weight"))
    return st


@dataclass
class CachedStack:
    """Whole decoder layers of `conversations` conversations: the fused linears with their norms and epilogues, RoPE, the paged cache and its
    attention; hidden rows in, hidden rows out.  Conversation c's pages are its own, shuffled over the cache; its length is on the device."""
    backend: Backend
    layers: int
    bits: int
    hidden: int
    heads: int
    kv_heads: int
    head_dim: int
    context: int                # tokens a conversation has pages for
    window: int
    cache: KVCache
    tables: object              # int32 [conversations, pages of one]
    lengths: object             # int32 [conversations]
    rope: object                # fp32 [tokens of a conversation's pages, head_dim / 2, 2]: the table's length, not less
    eps: float = 1e-5
    qkv: List[QWeight] = field(default_factory=list)
    o: List[QWeight] = field(default_factory=list)
    gate_up: List[QWeight] = field(default_factory=list)      # fuse_pairs
    down: List[QWeight] = field(default_factory=list)
    norms: List[tuple] = field(default_factory=list)          # gammas in front of qkv and of gate_up

    @property
    def weights(self) -> List[QWeight]:
        return self.qkv + self.o + self.gate_up + self.down

    @property
    def weight_bytes(self) -> int:
        return sum(w.algorithmic_bytes for w in self.weights)

    @property
    def nodes(self) -> List[str]:
        """The calls of one step."""
        return ["qkv", "append", "attention", "o", "gate_up", "down"] * self.layers

    @property
    def conversations(self) -> int:
        return self.tables.shape[0]

    def set_lengths(self, tokens: int, count: Optional[int] = None) -> None:
        """The first `count` conversations (None: all) hold their first `tokens` tokens (0: they begin again)."""
        self.lengths[:count].fill_(tokens)

    def stepper(self, M: int, xdtype=None, count: int = 1, seed: int = 5):
        """step(stream, first): M new tokens, M / count for each of the conversations first .. first + count.  Tokens behind a conversation's
        pages are not stored: counting them is the caller's affair.  Its buffers are made on torch's current stream, which steps on another one
        have to wait for."""
        import torch
        if count < 1 or M % count:
            raise CybqError(-2, "bad shape", "the rows are shared by the conversations evenly")
        xdtype = xdtype or torch.float16
        be, dev, n = self.backend, f"cuda:{self.backend.device}", M // count
        qdtype = {"f16": torch.float16, "bf16": torch.bfloat16}.get(self.cache.kind, xdtype)
        heads, kvh, dim = self.heads, self.kv_heads, self.head_dim

        def rows(cols, dtype=xdtype):
            return torch.empty((M, cols), dtype=dtype, device=dev)
        b = {"x": torch.from_numpy(synth.activations(seed, M, self.hidden)).to(dev).to(xdtype), "qkv": rows((heads + 2 * kvh) * dim),
             "q": rows(heads * dim, qdtype).view(M, heads, dim), "attn": rows(heads * dim, qdtype), "mid": rows(self.hidden),
             "h": rows(self.down[0].K), "y": rows(self.hidden)}
        q, k, v = b["qkv"].view(M, heads + 2 * kvh, dim).split([heads, kvh, kvh], dim=1)
        starts = torch.arange(0, M + 1, n, dtype=torch.int32, device=dev)
        batches = {}

        def step(stream: int = 0, first: int = 0) -> None:
            if first not in batches:
                if not 0 <= first <= self.conversations - count:
                    raise CybqError(-1, "invalid argument", "no such conversations")
                batches[first] = be.cache_batch(starts, self.lengths[first:first + count], self.tables[first:first + count], M, n)
            batch, x = batches[first], b["x"]
            with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=be.device) if stream else torch.cuda.default_stream(be.device)):
                batch.keep[1].add_(n)
            for i in range(self.layers):
                be.matmul_norm(self.qkv[i], x, self.norms[i][0], self.eps, b["qkv"], stream=stream)
                be.cache_append(self.cache, i, batch, q, k, v, b["q"], self.rope, stream=stream)
                be.attention(self.cache, i, batch, b["q"], b["attn"].view(M, heads, dim), window=self.window, stream=stream)
                be.matmul_ex(self.o[i], b["attn"], b["mid"], "add", x, stream=stream)
                be.matmul_norm(self.gate_up[i], b["mid"], self.norms[i][1], self.eps, b["h"], "swiglu", stream=stream)
                be.matmul_ex(self.down[i], b["h"], b["y"], "add", b["mid"], stream=stream)
                x = b["y"]
        step.edges = b
        return step

    def free(self) -> None:
        for w in self.weights:
            w.free()
        self.cache.free()


def build_cached(backend: Backend, layers: int = 32, bits: int = formats.Q4, kind: str = "q8", conversations: int = 1, context: int = 4096,
                 heads: int = 32, kv_heads: int = 8, head_dim: int = 128, width: int = 14336, page: int = 64, window: int = 0,
                 base: float = 500000.0, seed: int = 5) -> CachedStack:
    """Random-init stack of whole layers (Llama-3-8B shapes unless told otherwise; hidden = heads * head_dim) with N(0, 0.02) weights
    quantised on the device, gammas 1 +- 0.1, and an empty cache of `kind` for `conversations` conversations of `context` tokens."""
    import torch
    hidden = heads * head_dim
    if context < 1 or conversations < 1 or width % 32 or kv_heads < 1 or heads % kv_heads:
        raise CybqError(-2, "bad shape", "width must be a multiple of 32, heads one of kv_heads, context and conversations at least 1")
    dev, per = f"cuda:{backend.device}", -(-context // page)
    gen = torch.Generator(device=dev)
    gen.manual_seed((synth.BASE_SEED ^ seed) & 0x7FFFFFFF)
    shuffled = torch.randperm(conversations * per, generator=gen, device=dev).to(torch.int32).view(conversations, per)
    angle = torch.arange(per * page, dtype=torch.float64, device=dev).unsqueeze(1) * base ** (
        -torch.arange(0, head_dim, 2, dtype=torch.float64, device=dev) / head_dim)
    st = CachedStack(backend, layers, bits, hidden, heads, kv_heads, head_dim, context, window,
                     backend.kv_cache(kind, layers, kv_heads, head_dim, page, conversations * per), shuffled,
                     torch.zeros(conversations, dtype=torch.int32, device=dev), torch.stack([angle.cos(), angle.sin()], dim=2).float())

    def tensor(N: int, K: int, name: str = None) -> QWeight:
        w = torch.empty((N, K), dtype=torch.float32, device=dev).normal_(0.0, 0.02, generator=gen)
        q = torch.empty(N * K * bits // 8, dtype=torch.uint8, device=dev)
        s = torch.empty(N * (K // 32), dtype=torch.int16, device=dev)
        backend.quantize(bits, w, N, K, q, s)
        out = backend.weight_from_device(bits, N, K, q, s, name=name)
        torch.cuda.synchronize(dev)                                      # w, q and s are released
        return out

    for i in range(layers):
        st.qkv.append(tensor((heads + 2 * kv_heads) * head_dim, hidden, tensor_name(i, "qkv_proj")))
        st.o.append(tensor(hidden, hidden, tensor_name(i, "o_proj")))
        gate, up = tensor(width, hidden), tensor(width, hidden)
        st.gate_up.append(backend.fuse_pairs(gate, up, name=tensor_name(i, "gate_up_proj")))
        gate.free()
        up.free()
        st.down.append(tensor(hidden, width, tensor_name(i, "down_proj")))
        st.norms.append(tuple((1.0 + 0.1 * torch.empty(hidden, device=dev).normal_(generator=gen)).half() for _ in range(2)))
    return st
