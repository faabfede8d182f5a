"""The paged key-value cache as cases to time: new tokens' rows rotated, quantised and written into their pages, then read
back (`store`: cache_append, cache_read), whole sequences read back (`read`: cache_read), and the attention of the new
tokens over all that is cached for their sequences (`attn`: attention).

Where `own` is false `run` computes the definitions with elementary torch operations in fp32 (the rotation and the
quantiser's quotients in fp64: which of two integers a value becomes hangs on their last bits); where it is true it makes
the calls of cyb_amd.Backend.

A batch is `starts` [B + 1], `lengths` [B] and `tables` [B, pages]: sequence b has starts[b + 1] - starts[b] new rows, the
last ones of its lengths[b] tokens; token j lies in page tables[b, j // page], slot j % page.  A page id of -1 is no page
(pages that have left the window are given back): its tokens are not seen.  Rows of a padded batch behind the last
sequence's stay as they were.

Caches of kind q8 and q4 hold integers in groups of 32 along a head with one half-precision scale, the weights' format:
d = f16(absmax / qmax), q = round(x / d), ties away from zero.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BITS = {"f16": 16, "bf16": 16, "q8": 8.5, "q4": 4.5}               # a value's share of its group's scale included
LIMIT = {"f16": 65504.0, "bf16": 3.3895313892515355e38, "q8": 57344.0, "q4": 57344.0}


def _case(kind, **kw):
    return dict({"kind": kind, "cache": "q8", "x": "f16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "seqs": 1, "length": 1,
                 "ragged": False, "new": 1, "mixed": False, "window": 0, "evicted": False, "pad": 0, "rot": 128, "style": "halves",
                 "out": "f16"}, **kw)


def listed():
    return [
        # one token of one conversation, heads of a Llama-3-8B layer: what every layer of a decode step does with its q, k and v
        _case("store", name="store_token", length=777),
        # a batch of conversations being decoded on a narrow model's heads, 4-bit cache, neighbouring dimensions as pairs, half
        # of a head rotated
        _case("store", name="store_batch_48_q4", cache="q4", x="bf16", heads=16, kv_heads=2, seqs=48, length=2500, ragged=True, rot=64,
              style="pairs", out="bf16"),
        # a chunk of a long prompt, its first tokens in a page that is half full
        _case("store", name="store_prompt_4096", x="bf16", length=4096 + 709, new=4096, out="bf16"),
        # one conversation answering: short, where latency counts, and long, where one token reads 200 MB
        _case("attn", name="attn_token_1000", length=1000),
        _case("attn", name="attn_token_100001", x="bf16", length=100001),
        # a batch of conversations of all lengths, the last rows of the batch padding
        _case("attn", name="attn_batch_48", seqs=48, length=8192, ragged=True, pad=3),
        # drafted tokens to be judged, seven heads to a kv head, a 4-bit cache and a window whose old pages are gone
        _case("attn", name="attn_draft_8x5_q4_window", cache="q4", x="bf16", heads=28, kv_heads=4, page=32, seqs=8, length=6000, ragged=True,
              new=5, window=2048, evicted=True),
        # a prompt from its first token on, short heads, a cache of 16 bits
        _case("attn", name="attn_prompt_2000_bf16", cache="bf16", x="bf16", heads=32, kv_heads=8, dim=64, rot=64, length=2000, new=2000),
        # a chunk of a long prompt next to sixteen conversations being decoded
        _case("attn", name="attn_mixed_512", seqs=17, length=16384, ragged=True, new=512, mixed=True),
        # the largest: a chunk in the middle of a long document
        _case("attn", name="attn_chunk_4096_of_32768", cache="f16", length=32768, new=4096),
        # a few short sequences read back, 4-bit cache; long ones, handed on to another program
        _case("read", name="read_short_q4", cache="q4", heads=16, kv_heads=2, page=32, seqs=3, length=300, ragged=True, out="f32"),
        _case("read", name="read_long", seqs=4, length=20011, ragged=True, out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["store", "store", "attn", "attn", "attn", "attn", "read"])
    cache = rng.choice(["f16", "bf16", "q8", "q8", "q8", "q4", "q4"])
    dim = rng.choice([64, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
    if dim == 256:
        kv_heads, group = min(kv_heads, 4), min(group, 8)
    c = _case(kind, cache=cache, x=cache if cache in TYPES else rng.choice(["f16", "bf16"]), heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
              page=rng.choice([32, 64, 64, 128, 256]), rot=rng.choice([dim, dim, dim // 2]), style=rng.choice(["halves", "halves", "pairs"]))
    if kind != "attn":
        c["x"] = rng.choice(["f16", "bf16", "f32"])
        c["out"] = rng.choice(["f16", "bf16", "f32"])
    seqs = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 128)])
    c["ragged"] = seqs > 1 and rng.random() < 0.8
    if kind == "read":
        c["seqs"], c["length"] = seqs, _log(rng, 1, max(64, min(40000, int(1.6e8 / (seqs * kv_heads * dim)))))
        return c
    shape = rng.choice(["token", "token", "draft", "prompt", "chunk", "mixed"])
    if shape == "token" or shape == "draft":
        c["new"] = 1 if shape == "token" else rng.randint(2, 12)
        c["seqs"] = seqs
        c["length"] = c["new"] + _log(rng, 1, max(256, min(120000, int(1.3e8 / (seqs * kv_heads * dim)))))
    else:
        c["seqs"] = {"prompt": rng.choice([1, 1, 2, 5]), "chunk": 1, "mixed": rng.randint(2, 24)}[shape]
        c["new"] = _log(rng, 13, 2048 if c["seqs"] > 1 and shape == "prompt" else 4096)
        c["mixed"] = shape == "mixed"
        c["ragged"] = c["seqs"] > 1
        chunks = c["seqs"] if shape == "prompt" else 1
        most = int(1.0e12 / (chunks * c["new"] * c["heads"] * dim * 4))           # no more multiplications than the largest has
        c["length"] = c["new"] if shape == "prompt" else c["new"] + _log(rng, 1, max(2, min(30000 if c["seqs"] == 1 else 12000, most)))
    if kind == "attn" and rng.random() < 0.3:
        c["window"] = _log(rng, 1, 4096)
        c["evicted"] = rng.random() < 0.5
    c["pad"] = rng.choice([0, 0, rng.randint(1, 5)])
    return c


# ---- inputs -------------------------------------------------------------------------------------------------

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + what) & 0x7FFFFFFF)
    return g


def _randn(shape, gen, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen)


def _layout(case, seed):
    """(new rows, tokens) of every sequence, on the host: another seed has the same lengths in another order."""
    r = np.random.default_rng(17)
    B, L, n = case["seqs"], case["length"], case["new"]
    lengths = np.full(B, L, dtype=np.int64)
    if case["ragged"]:
        least = max(1, L // 8) if case["mixed"] or case["kind"] == "read" else max(n, L // 8)
        if n == L and n > 1 and not case["mixed"]:              # prompts from their first tokens on
            least = max(1, L // 4)
        lengths[:-1] = np.random.default_rng(seed).permutation(r.integers(least, L + 1, B - 1))
    new = np.full(B, n, dtype=np.int64)
    if case["mixed"]:
        new[:-1] = 1
    if case["kind"] == "read":
        new = lengths.copy()
    return np.minimum(new, lengths), lengths


def _inputs(case, seed):
    new, lengths = _layout(case, seed)
    B, page, kvh, dim = case["seqs"], case["page"], case["kv_heads"], case["dim"]
    per = -(-lengths // page)
    width, pages = int(per.max()), int(per.sum())
    r = np.random.default_rng(seed * 104729 + 5)
    order = r.permutation(pages)
    tables = np.full((B, width), -1, dtype=np.int32)
    at = 0
    for b in range(B):
        tables[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
    full = tables.copy()                                     # as they were when the tokens were written
    if case["evicted"]:
        for b in range(B):
            first = int(lengths[b] - new[b]) - case["window"] + 1            # the first position that the first new row sees
            tables[b, :max(0, first) // page] = -1
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    s = {"starts": torch.from_numpy(starts).cuda(), "lengths": torch.from_numpy(lengths.astype(np.int32)).cuda(),
         "tables": torch.from_numpy(tables).cuda(), "full": torch.from_numpy(full).cuda(), "pages": pages,
         "new": new.tolist(), "len": lengths.tolist(), "rows": int(new.sum()) + case["pad"]}
    x = TYPES[case["x"]]
    # a few channels of the keys are much larger than the others, as they are behind a rotary embedding
    loud = 1.0 + 4.0 * (torch.rand((1, kvh, dim), generator=_gen(seed, 1), device="cuda") < 0.04).float()
    if case["kind"] == "store":
        # one buffer as the fused projection leaves it: q heads, k heads, v heads side by side
        h = case["heads"]
        qkv = _randn((s["rows"], h + 2 * kvh, dim), _gen(seed, 2))
        qkv[:, h:h + kvh] *= loud
        s["qkv"] = qkv.to(x)
        capacity = width * page
        freq = 10000.0 ** (-torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda") * 2.0 / case["rot"])
        angle = torch.arange(capacity, dtype=torch.float64, device="cuda").reshape(-1, 1) * freq
        s["rope"] = torch.stack((torch.cos(angle), torch.sin(angle)), dim=2).to(torch.float32).contiguous()
        return s
    total = int(lengths.sum())
    s["k"] = (_randn((total, kvh, dim), _gen(seed, 3)) * loud).to(x)
    s["v"] = _randn((total, kvh, dim), _gen(seed, 4)).to(x)
    if case["kind"] == "attn":
        # queries that agree with some of the keys: scores with a spread of 2 and a few far above
        s["q"] = _randn((s["rows"], case["heads"], dim), _gen(seed, 5), 1.3).to(x)
    return s


_backend = None


def _library():
    """One context for the life of the process, as a runtime keeps it."""
    global _backend
    if _backend is None:
        from cyb_amd import Backend
        torch.cuda.init()
        _backend = Backend(0)
    return _backend


def prepare(case, seed):
    """The inputs, the buffers that a program keeps for results, and the cache with what was written before."""
    a = _inputs(case, seed)
    st = {"case": case, "in": a}
    kvh, dim, rows = case["kv_heads"], case["dim"], a["rows"]
    out = TYPES[case["out"]]
    if case["kind"] == "attn":
        st["y"] = torch.zeros((rows, case["heads"], dim), dtype=TYPES[case["x"]], device="cuda")
    else:
        st["k"], st["v"] = (torch.zeros((rows, kvh, dim), dtype=out, device="cuda") for _ in range(2))
    if case["kind"] == "store":
        st["q"] = torch.zeros((rows, case["heads"], dim), dtype=out if case["out"] != "f32" else torch.bfloat16, device="cuda")
    if own:
        be = _library()
        st["cache"] = be.kv_cache(case["cache"], 1, kvh, dim, case["page"], a["pages"])
        st["batch"] = be.cache_batch(a["starts"], a["lengths"], a["tables"], rows, max(a["new"]))
        if case["kind"] != "store":
            starts = torch.from_numpy(np.concatenate([[0], np.cumsum(a["len"])]).astype(np.int32)).cuda()
            written = be.cache_batch(starts, a["lengths"], a["full"], sum(a["len"]), max(a["len"]))
            be.cache_append(st["cache"], 0, written, None, a["k"], a["v"])
    else:
        st["planes"] = [_empty_planes(case, a["pages"]) for _ in range(2)]
        if case["kind"] != "store":
            page, slot = _places(case, a["full"], [0] * case["seqs"], a["len"])
            for planes, x in zip(st["planes"], (a["k"], a["v"])):
                for i in range(0, x.shape[0], 1 << 15):
                    _plain_write(case, planes, page[i:i + (1 << 15)], slot[i:i + (1 << 15)], x[i:i + (1 << 15)].to(torch.float32))
    torch.cuda.synchronize()
    return st


# ---- the library's calls ------------------------------------------------------------------------------------

def _own(st):
    case, a = st["case"], st["in"]
    be, cache, batch = _library(), st["cache"], st["batch"]
    if case["kind"] == "attn":
        be.attention(cache, 0, batch, a["q"], st["y"], window=case["window"])
        return st["y"]
    if case["kind"] == "store":
        h, kvh, qkv = case["heads"], case["kv_heads"], a["qkv"]
        be.cache_append(cache, 0, batch, qkv[:, :h], qkv[:, h:h + kvh], qkv[:, h + kvh:], st["q"], rope=a["rope"], style=case["style"])
    be.cache_read(cache, 0, batch, st["k"], st["v"])
    return (st["q"], st["k"], st["v"]) if case["kind"] == "store" else (st["k"], st["v"])


# ---- the plain form -----------------------------------------------------------------------------------------

def _empty_planes(case, pages):
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    if case["cache"] in TYPES:
        return (torch.zeros(shape, dtype=TYPES[case["cache"]], device="cuda"),)
    return (torch.zeros(shape, dtype=torch.int8, device="cuda"),
            torch.zeros(shape[:3] + (case["dim"] // 32,), dtype=torch.float16, device="cuda"))


def _places(case, tables, first, count):
    """Page and slot of tokens first[b] .. first[b] + count[b] of every sequence, one after another."""
    at = [tables[b].long() for b in range(case["seqs"])]
    pos = [torch.arange(f, f + c, device="cuda") for f, c in zip(first, count)]
    return torch.cat([t[p // case["page"]] for t, p in zip(at, pos)]), torch.cat([p % case["page"] for p in pos])


def _plain_write(case, planes, page, slot, x):
    """x: fp32 rows of tokens, into their pages as the cache's kind holds them."""
    x = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).clamp(-LIMIT[case["cache"]], LIMIT[case["cache"]])
    if case["cache"] in TYPES:
        planes[0][page, slot] = x.to(TYPES[case["cache"]])
        return
    most = 127.0 if case["cache"] == "q8" else 7.0
    g = x.reshape(x.shape[:2] + (-1, 32))
    d = (g.abs().amax(dim=3).double() / most).to(torch.float32).to(torch.float16)
    r = (g.double() / d.double().unsqueeze(3)).to(torch.float32).double()
    q = torch.sign(r) * torch.floor(r.abs() + 0.5)
    q = torch.where(d.unsqueeze(3) == 0, 0.0, q).clamp(-most, most)
    planes[0][page, slot] = q.to(torch.int8).reshape(x.shape)
    planes[1][page, slot] = d


def _plain_values(planes, page, slot):
    """fp32 [tokens, kv heads, dim] of the tokens at these places; places without a page: zeros."""
    there = page >= 0
    v = planes[0][page.clamp(min=0), slot].to(torch.float32)
    if len(planes) == 2:
        d = planes[1][page.clamp(min=0), slot].to(torch.float32)
        v = (v.reshape(d.shape + (32,)) * d.unsqueeze(3)).reshape(v.shape)
    return torch.where(there.reshape(-1, 1, 1), v, 0.0)


def _plain_rotate(x, rope, style):
    """x [rows, heads, dim], rope [rows, rot / 2, 2] -> fp32; the first rot dimensions of a head turn."""
    rot = rope.shape[1] * 2
    c, s = (rope[:, :, i].double().unsqueeze(1) for i in range(2))
    x = x.double()
    if style == "halves":
        a, b = x[:, :, :rot // 2], x[:, :, rot // 2:rot]
        turned = torch.cat((a * c - b * s, b * c + a * s), dim=2)
    else:
        a, b = x[:, :, 0:rot:2], x[:, :, 1:rot:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), dim=3).reshape(x.shape[:2] + (rot,))
    return torch.cat((turned, x[:, :, rot:]), dim=2).to(torch.float32)


def _plain_read(st):
    case, a = st["case"], st["in"]
    n = sum(a["new"])
    page, slot = _places(case, a["tables"], [l - m for l, m in zip(a["len"], a["new"])], a["new"])
    for planes, out in zip(st["planes"], (st["k"], st["v"])):
        out[:n] = _plain_values(planes, page, slot).to(out.dtype)
    return st["k"], st["v"]


def _plain_store(st):
    case, a = st["case"], st["in"]
    n, h, kvh = sum(a["new"]), case["heads"], case["kv_heads"]
    first = [l - m for l, m in zip(a["len"], a["new"])]
    page, slot = _places(case, a["tables"], first, a["new"])
    rope = a["rope"][torch.cat([torch.arange(f, f + m, device="cuda") for f, m in zip(first, a["new"])])]
    st["q"][:n] = _plain_rotate(a["qkv"][:n, :h], rope, case["style"]).to(st["q"].dtype)
    _plain_write(case, st["planes"][0], page, slot, _plain_rotate(a["qkv"][:n, h:h + kvh], rope, case["style"]))
    _plain_write(case, st["planes"][1], page, slot, a["qkv"][:n, h + kvh:].to(torch.float32))
    return (st["q"],) + _plain_read(st)


def _plain_attn(st):
    case, a = st["case"], st["in"]
    kvh, dim = case["kv_heads"], case["dim"]
    group, row = case["heads"] // kvh, 0
    for b in range(case["seqs"]):
        n, L = a["new"][b], a["len"][b]
        lo = max(0, L - n - case["window"] + 1) if case["window"] else 0          # before it no row sees anything
        pos = torch.arange(lo, L, device="cuda")
        page, slot = a["tables"][b].long()[pos // case["page"]], pos % case["page"]
        k, v = (_plain_values(p, page, slot).transpose(0, 1).contiguous() for p in st["planes"])
        q = a["q"][row:row + n].to(torch.float32).reshape(n, kvh, group, dim).permute(1, 0, 2, 3).reshape(kvh, n * group, dim)
        mine = torch.arange(L - n, L, device="cuda").repeat_interleave(group).reshape(-1, 1)
        seen = (pos <= mine) & (page >= 0)
        if case["window"]:
            seen &= pos > mine - case["window"]
        out = torch.empty_like(q)
        step = max(1, (1 << 30) // (n * group * (L - lo)))
        for h in range(0, kvh, step):
            s = torch.bmm(q[h:h + step], k[h:h + step].transpose(1, 2).contiguous()) * (1.0 / math.sqrt(dim))
            s = torch.where(seen, s, -math.inf)
            top = s.amax(dim=2, keepdim=True)
            s = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            total = s.sum(dim=2, keepdim=True)
            out[h:h + step] = torch.bmm(s, v[h:h + step]) / torch.where(total == 0, 1.0, total)
        st["y"][row:row + n] = out.reshape(kvh, n, group, dim).permute(1, 0, 2, 3).reshape(n, kvh * group, dim).to(st["y"].dtype)
        row += n
    return st["y"]


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "read": _plain_read, "attn": _plain_attn}[state["case"]["kind"]](state)


# ---- work ---------------------------------------------------------------------------------------------------

def work(case):
    new, lengths = _layout(case, 0)
    rows, kvh, dim, h = int(new.sum()), case["kv_heads"], case["dim"], case["heads"]
    held = 2 * kvh * dim * BITS[case["cache"]] / 8         # bytes of a token's keys and values
    if case["kind"] == "read":
        return {"bytes": int(rows * (held + 2 * kvh * dim * SIZE[case["out"]])), "flops": rows * 2 * kvh * dim}
    if case["kind"] == "store":
        return {"bytes": int(rows * ((h + 2 * kvh) * dim * SIZE[case["x"]] + h * dim * 2 + held + 2 * kvh * dim * SIZE[case["out"]]
                                     + case["rot"] * 4)), "flops": rows * ((h + kvh) * case["rot"] * 3 + 6 * kvh * dim)}
    tokens = pairs = 0
    for n, L in zip(new.tolist(), lengths.tolist()):
        w = case["window"] or L
        tokens += min(L, n - 1 + w)
        p = np.arange(L - n, L)
        pairs += int(np.minimum(p + 1, w).sum())
    return {"bytes": int(tokens * held + rows * 2 * h * dim * SIZE[case["x"]]), "flops": 4 * pairs * h * dim}


# ---- the definition in 64 bits ------------------------------------------------------------------------------

def _held(kind, x):
    """float64 of what a cache of this kind holds for fp32 x [..., dim]: the roundings are part of the definition."""
    limit = LIMIT[kind]
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(min=-limit, max=limit)
    if kind in TYPES:
        return x.to(TYPES[kind]).double()
    steps = {"q8": 127, "q4": 7}[kind]
    groups = x.double().unflatten(-1, (-1, 32))
    scale = (groups.abs().max(dim=-1, keepdim=True).values / steps).float().half().double()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    units = (groups / safe).float().double()
    whole = units.trunc()
    whole = whole + torch.where((units - whole).abs() >= 0.5, units.sign(), torch.zeros_like(units))
    return (whole.clamp(-steps, steps) * scale).flatten(-2)


def _turn(x, positions, rope, style):
    """float64 rotation of x [rows, heads, dim], as complex numbers."""
    table = torch.view_as_complex(rope.double())[positions].unsqueeze(1)
    rot = rope.shape[1] * 2
    x = x.double()
    head, rest = x[..., :rot], x[..., rot:]
    pairs = head.unflatten(-1, (2, rot // 2)).transpose(-1, -2) if style == "halves" else head.unflatten(-1, (rot // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * table)
    z = z.transpose(-1, -2) if style == "halves" else z
    return torch.cat((z.flatten(-2), rest), dim=-1)


def exact(case, seed):
    a = _inputs(case, seed)
    kvh, dim, h = case["kv_heads"], case["dim"], case["heads"]
    rows, n = a["rows"], sum(a["new"])
    if case["kind"] == "read":
        return tuple(_held(case["cache"], x.float()) for x in (a["k"], a["v"]))
    if case["kind"] == "store":
        where = torch.tensor([l - m + i for l, m in zip(a["len"], a["new"]) for i in range(m)], device="cuda")
        q, k, v = (torch.zeros((rows, w, dim), dtype=torch.float64, device="cuda") for w in (h, kvh, kvh))
        q[:n] = _turn(a["qkv"][:n, :h], where, a["rope"], case["style"])
        k[:n] = _held(case["cache"], _turn(a["qkv"][:n, h:h + kvh], where, a["rope"], case["style"]).float())
        v[:n] = _held(case["cache"], a["qkv"][:n, h + kvh:].float())
        return q, k, v
    y = torch.zeros((rows, h, dim), dtype=torch.float64, device="cuda")
    row = token = 0
    for b, (m, L) in enumerate(zip(a["new"], a["len"])):
        here = (a["tables"][b].repeat_interleave(case["page"])[:L] >= 0)
        there = torch.arange(L, device="cuda")
        for g in range(kvh):
            k, v = (_held(case["cache"], x[token:token + L, g].float()) for x in (a["k"], a["v"]))
            for head in range(g * h // kvh, (g + 1) * h // kvh):
                for i in range(0, m, 2048):
                    part = min(2048, m - i)
                    own_place = torch.arange(L - m + i, L - m + i + part, device="cuda")
                    back = own_place[:, None] - there[None, :]               # how far back a token lies
                    hidden = (back < 0) | ~here
                    if case["window"]:
                        hidden |= back >= case["window"]
                    s = a["q"][row + i:row + i + part, head].double() @ k.t().contiguous() / dim ** 0.5
                    s.masked_fill_(hidden, -math.inf)
                    y[row + i:row + i + part, head] = torch.nan_to_num(torch.softmax(s, dim=1)) @ v
        row += m
        token += L
    return y
