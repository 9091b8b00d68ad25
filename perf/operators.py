"""The operators of the 8-bit KV cache and of scaled rotary positions: cases, inputs, plain forms, exact values.

    rope       rotary positions from a frequency table: interleaved or half layout, all of a head or its first part
    write      the same for q and k, with k and v quantised into the cache's slots on the way
    read       rows of the cache read back
    attention  paged, variable-length, grouped, causal attention over the cache

A cache is a pool of E4M3 codes, [slots, kv_heads * head_dim], and a float32 scale for each head of each slot,
[kv_heads, slots]: value = code * scale, scale = max(largest magnitude / 448, 2^-126).
"""
import math
import random

import torch

own = False

E4M3_MAX, LEAST_SCALE = 448.0, 2.0 ** -126
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one request, the step of a chat: nothing but latency
        dict(name="rope_one_token", op="rope", tokens=1, heads=32, kv_heads=8, head_dim=128, rotary=128, half=False,
             type="bf16", farthest=8192),
        # a chunk of a prompt of a model that rotates half of each head, at positions of a long context
        dict(name="rope_chunk_partial", op="rope", tokens=8192, heads=32, kv_heads=8, head_dim=128, rotary=64, half=True,
             type="bf16", farthest=131072),
        # a decode step of a full batch
        dict(name="write_decode_64", op="write", tokens=64, heads=32, kv_heads=8, head_dim=128, rotary=128, half=False,
             type="bf16", farthest=131072, slots=65536),
        # a prompt of a small model with float32 activations, no round number anywhere
        dict(name="write_odd_777_f32", op="write", tokens=777, heads=14, kv_heads=2, head_dim=64, rotary=64, half=True,
             type="f32", farthest=32768, slots=5000),
        # a long prompt
        dict(name="write_prompt_8192", op="write", tokens=8192, heads=32, kv_heads=8, head_dim=128, rotary=128, half=False,
             type="bf16", farthest=131072, slots=32768),
        # a request's cache taken out, to be kept or sent elsewhere
        dict(name="read_1000", op="read", rows=1000, kv_heads=8, head_dim=128, type="bf16", slots=16384),
        dict(name="read_40001_f32", op="read", rows=40001, kv_heads=8, head_dim=128, type="f32", slots=65536),
        # one request's decode step
        dict(name="decode_1x1000", op="attention", requests=1, shortest=1000, longest=1000, new=1, heads=32, kv_heads=8,
             head_dim=128, page=16, type="bf16", ragged=0),
        # a decode batch whose requests have come differently far
        dict(name="decode_64_ragged", op="attention", requests=64, shortest=100, longest=8192, new=1, heads=32, kv_heads=8,
             head_dim=128, page=16, type="bf16", ragged=1),
        # one request at the end of a long context
        dict(name="decode_1x131072", op="attention", requests=1, shortest=131071, longest=131071, new=1, heads=32, kv_heads=8,
             head_dim=128, page=256, type="bf16", ragged=0),
        # a prompt of its own
        dict(name="prompt_4096", op="attention", requests=1, shortest=4096, longest=4096, new=4096, heads=32, kv_heads=8,
             head_dim=128, page=16, type="bf16", ragged=0),
        # a mixed batch of a small model: chunks of prompts beside decoding requests, pages that are no power of two
        dict(name="mixed_12_odd", op="attention", requests=12, shortest=1, longest=2900, new=500, heads=14, kv_heads=2,
             head_dim=64, page=24, type="bf16", ragged=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "attention", "attention", "attention"])
    head_dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([n for n in (1, 2, 4, 4, 5, 7, 8) if n * kv_heads <= 40])
    kind = rng.choice(["bf16", "bf16", "f32"])
    if op == "read":
        slots = _log(rng, 2000, 65536)
        return dict(op=op, rows=_log(rng, 1, min(slots, 40000)), kv_heads=kv_heads, head_dim=head_dim, type=kind, slots=slots)
    if op in ("rope", "write"):
        tokens = _log(rng, 1, 8192 * 32 // max(32, heads))
        case = dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary=rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4]), half=rng.random() < 0.5, type=kind,
                    farthest=_log(rng, 8192, 131072))
        if kind == "f32":
            case["tokens"] = max(1, tokens // 2)
        if op == "write":
            case["slots"] = case["tokens"] + _log(rng, 16, 20000)
        return case
    page = rng.choice([16, 16, 32, 64, 256, rng.randint(1, 100)])
    what = rng.choice(["decode", "decode", "prompt", "mixed"])
    if what == "decode":
        requests = _log(rng, 1, 64)
        longest = _log(rng, 64, min(131072, 260000 // requests))
        shortest, new = rng.randint(1, longest), 1
    elif what == "prompt":
        requests = rng.choice([1, 1, 2])
        longest = _log(rng, 20, 4000 * 32 // max(32, heads) // requests)
        shortest, new = longest, rng.choice([longest, max(1, longest // 2)])
    else:
        requests = rng.randint(2, 12)
        longest = _log(rng, 100, 4000)
        shortest, new = rng.randint(1, longest), rng.randint(1, min(longest, 600))
    return dict(op="attention", requests=requests, shortest=shortest, longest=longest, new=new, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, type="bf16", ragged=rng.randint(1, 1000))


def _lengths(case):
    """Positions and new tokens of each request of an attention case."""
    rng = random.Random(case["ragged"])
    n = case["requests"]
    lens = [case["longest"]] + [rng.randint(case["shortest"], case["longest"]) for _ in range(n - 1)]
    if case["new"] == 1:
        return lens, [1] * n
    # the first request brings the most tokens; of the others every second one is decoding
    news = [min(case["new"], lens[0])] + [1 if i % 2 else rng.randint(1, min(case["new"], lens[i])) for i in range(1, n)]
    return lens, news


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "read":
        row = case["kv_heads"] * case["head_dim"]
        return {"bytes": case["rows"] * (row + 4 * case["kv_heads"] + 4 + row * size), "flops": case["rows"] * row}
    if case["op"] in ("rope", "write"):
        t, hd = case["tokens"], case["head_dim"]
        q, k = t * case["heads"] * hd, t * case["kv_heads"] * hd
        flops = 3 * t * (case["heads"] + case["kv_heads"]) * case["rotary"]
        if case["op"] == "rope":
            return {"bytes": 2 * (q + k) * size + 4 * t, "flops": flops}
        return {"bytes": (2 * q + 2 * k) * size + 2 * k + 8 * t * case["kv_heads"] + 8 * t, "flops": flops + 4 * k}
    lens, news = _lengths(case)
    row = case["heads"] * case["head_dim"]
    pairs = sum(n * (l - n) + n * (n + 1) // 2 for l, n in zip(lens, news))
    pages = sum(-(-l // case["page"]) for l in lens)
    return {"bytes": sum(lens) * case["kv_heads"] * (2 * case["head_dim"] + 8) + 2 * sum(news) * row * size + 4 * pages,
            "flops": 4 * row * pairs}


# ---- inputs --------------------------------------------------------------------------------------

def _quantised(x, kv_heads):
    """[slots, row] -> E4M3 codes [slots, row] and scales [kv_heads, slots]: how a cache was filled."""
    h = x.view(x.shape[0], kv_heads, -1)
    scale = (h.abs().amax(-1) / torch.tensor(E4M3_MAX, device=x.device)).clamp_min(LEAST_SCALE)
    return (h / scale[..., None]).to(torch.float8_e4m3fn).reshape(x.shape), scale.t().contiguous()


def _frequencies(rotary):
    """theta = 500000, stretched for a long context by wavelength: short waves as they are, long ones slowed eightfold."""
    i = torch.arange(rotary // 2, dtype=torch.float64)
    f = 500000.0 ** (-2.0 * i / rotary)
    turns = 8192.0 * f / (2.0 * math.pi)
    keep = ((turns - 1.0) / 3.0).clamp(0.0, 1.0)
    return (f * (keep + (1.0 - keep) / 8.0)).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kv_heads, hd = case["kv_heads"], case["head_dim"]
    row = kv_heads * hd
    # some channels of keys are much larger than the others, as in trained models
    loud = torch.where(torch.rand(row, generator=g, device="cuda") < 0.05, 6.0, 1.0)
    if case["op"] == "read":
        codes, scales = _quantised(rand(case["slots"], row) * loud, kv_heads)
        rows = torch.randperm(case["slots"], generator=g, device="cuda")[: case["rows"]].to(torch.int32)
        return dict(case=case, codes=codes, scales=scales, rows=rows, out=torch.zeros(case["rows"], row, dtype=kind, device="cuda"))
    if case["op"] in ("rope", "write"):
        t, heads = case["tokens"], case["heads"]
        first = int(torch.randint(0, max(1, case["farthest"] - t), (1,), generator=g, device="cuda"))
        s = dict(case=case, q=rand(t, heads * hd).to(kind), k=(rand(t, row) * loud).to(kind),
                 positions=torch.arange(first, first + t, device="cuda", dtype=torch.int32),
                 freq=_frequencies(case["rotary"]).cuda(), magnitude=1.1)
        s["q_out"] = torch.zeros_like(s["q"])
        if case["op"] == "rope":
            return s | dict(k_out=torch.zeros_like(s["k"]))
        n = case["slots"]
        return s | dict(
            v=rand(t, row).to(kind), slots=torch.randperm(n, generator=g, device="cuda")[:t].to(torch.int32),
            k_codes=torch.zeros(n, row, device="cuda").to(torch.float8_e4m3fn), k_scales=torch.zeros(kv_heads, n, device="cuda"),
            v_codes=torch.zeros(n, row, device="cuda").to(torch.float8_e4m3fn), v_scales=torch.zeros(kv_heads, n, device="cuda"))
    lens, news = _lengths(case)
    page, most = case["page"], -(-max(lens) // case["page"])
    pages = sum(-(-l // page) for l in lens) + 3
    k_codes, k_scales = _quantised(rand(pages * page, row) * loud, kv_heads)
    v_codes, v_scales = _quantised(rand(pages * page, row), kv_heads)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), most, dtype=torch.int32, device="cuda")
    at = 0
    for r, l in enumerate(lens):
        n = -(-l // page)
        table[r, :n] = order[at: at + n]
        at += n
    q = rand(sum(news), case["heads"] * hd).to(kind)
    starts = torch.tensor([0] + news, device="cuda").cumsum(0).to(torch.int32)
    return dict(case=case, q=q, out=torch.zeros_like(q), k_codes=k_codes, k_scales=k_scales, v_codes=v_codes, v_scales=v_scales,
                table=table, starts=starts, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), longest=max(lens),
                most_new=max(news))


# ---- plain forms ---------------------------------------------------------------------------------

def _rotated(x, s):
    """[tokens, heads * head_dim] rotated, in 32 bits; the angles, which lose their fraction far out, in 64."""
    case, half = s["case"], s["case"]["rotary"] // 2
    h = x.float().view(x.shape[0], -1, case["head_dim"])
    angle = s["positions"].double()[:, None] * s["freq"].double()
    cos = (angle.cos() * s["magnitude"]).float()[:, None]
    sin = (angle.sin() * s["magnitude"]).float()[:, None]
    part, rest = h[..., : 2 * half], h[..., 2 * half:]
    if case["half"]:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, rest], -1).view(x.shape)


def _write(x, codes, scales, slots):
    c, s = _quantised(x, scales.shape[0])
    codes.view(torch.uint8)[slots] = c.view(torch.uint8)
    scales[:, slots] = s


def _plain_attention(s):
    case = s["case"]
    hd, kv_heads, page = case["head_dim"], case["kv_heads"], case["page"]
    group = case["heads"] // kv_heads
    at = torch.arange(s["longest"], device="cuda")
    slot = s["table"].long()[:, at // page] * page + at % page                                   # [request, position]

    def values(codes, scales):                                                                   # [request, head, position, dim]
        x = codes.view(torch.uint8)[slot].view(torch.float8_e4m3fn).float().view(*slot.shape, kv_heads, hd)
        return (x * scales.t()[slot][..., None]).transpose(1, 2)

    i = torch.arange(s["most_new"], device="cuda")
    starts, new = s["starts"].long()[:-1], s["starts"].long().diff()
    there = i < new[:, None]
    token = (starts[:, None] + i).clamp_max(s["q"].shape[0] - 1)
    q = s["q"][token].float().view(len(new), -1, kv_heads, group, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = q @ values(s["k_codes"], s["k_scales"]).transpose(-1, -2) / math.sqrt(hd)             # [request, head, (of group, new), position]
    seen = at < (s["lens"][:, None] - new[:, None] + i + 1)[..., None]                           # [request, new, position]
    seen = seen[:, None, None].expand(-1, 1, group, -1, -1).flatten(2, 3)
    score = score.masked_fill(~seen, -math.inf)
    p = (score - score.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    o = (p @ values(s["v_codes"], s["v_scales"])) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.unflatten(2, (group, -1)).permute(0, 3, 1, 2, 4).flatten(2)
    s["out"][token[there]] = o[there].to(s["out"].dtype)
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    s, op = state, state["case"]["op"]
    if op == "attention":
        return _plain_attention(s)
    if op == "read":
        kv_heads, rows = s["case"]["kv_heads"], s["rows"].long()
        x = s["codes"].view(torch.uint8)[rows].view(torch.float8_e4m3fn).float().view(len(rows), kv_heads, -1)
        s["out"].copy_((x * s["scales"].t()[rows][..., None]).view(len(rows), -1))
        return s["out"]
    s["q_out"].copy_(_rotated(s["q"], s))
    if op == "rope":
        s["k_out"].copy_(_rotated(s["k"], s))
        return [s["q_out"], s["k_out"]]
    slots = s["slots"].long()
    _write(_rotated(s["k"], s), s["k_codes"], s["k_scales"], slots)
    _write(s["v"].float(), s["v_codes"], s["v_scales"], slots)
    return [s["q_out"], s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]]


# ---- the framework's calls -----------------------------------------------------------------------

_backends = {}
LEGACY_STREAM = 1          # the handle that names torch's default stream; 0 asks for a stream of the context's own


def _backend():
    """A context on torch's current stream: its calls come after what torch has put there and before what it puts there next."""
    from llm_rs_b200 import CudaBackend
    at = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream or LEGACY_STREAM
    if at not in _backends:
        _backends[at] = CudaBackend(*at)
    return _backends[at]


def _buffers(backend, state):
    """The state's tensors as buffers of the framework, which a program that keeps its data there has from the start."""
    from llm_rs_b200 import DType
    kinds = {torch.bfloat16: DType.BF16, torch.float32: DType.F32, torch.int32: DType.I32, torch.float8_e4m3fn: DType.E4M3}
    return {n: backend.wrap(t.data_ptr(), t.shape[::-1], kinds[t.dtype], keepalive=t)
            for n, t in state.items() if isinstance(t, torch.Tensor)}


def _run_own(state):
    s, case = state, state["case"]
    if "buffers" not in s:                              # the context and the buffers, as a program keeps them
        s["backend"] = _backend()
        s["buffers"] = _buffers(s["backend"], s)
    be, b = s["backend"], s["buffers"]
    if case["op"] == "attention":
        be.attention_quant(b["out"], b["q"], b["k_codes"], b["k_scales"], b["v_codes"], b["v_scales"], b["table"],
                           b["starts"], b["lens"], case["heads"], case["kv_heads"], case["head_dim"], case["page"],
                           s["table"].shape[1])
        return s["out"]
    if case["op"] == "read":
        be.gather_quant(b["out"], b["codes"], b["scales"], b["rows"], case["rows"])
        return s["out"]
    if case["op"] == "rope":
        be.rope_scaled(b["q_out"], b["k_out"], b["q"], b["k"], b["positions"], b["freq"], case["head_dim"],
                       s["magnitude"], split_half=case["half"])
        return [s["q_out"], s["k_out"]]
    be.rope_scatter_kv_quant(b["q_out"], b["q"], b["k"], b["v"], b["positions"], b["freq"], case["head_dim"],
                             s["magnitude"], b["k_codes"], b["k_scales"], b["v_codes"], b["v_scales"], b["slots"],
                             split_half=case["half"])
    return [s["q_out"], s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]]


# ---- exact values --------------------------------------------------------------------------------

def _exact_rotation(x, s):
    """Each pair as a complex number times magnitude * e^(i angle)."""
    case = s["case"]
    n, half = x.shape[0], case["rotary"] // 2
    turn = torch.polar(torch.full((n, half), s["magnitude"], dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["freq"].double()))
    y = x.double().view(n, -1, case["head_dim"]).clone()
    first = slice(0, half) if case["half"] else slice(0, 2 * half, 2)
    second = slice(half, 2 * half) if case["half"] else slice(1, 2 * half, 2)
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_cache(y, s, slots):
    """Codes before their rounding, and scales, of heads y [token, head, dim]."""
    scale = torch.maximum(y.abs().max(-1).values / 448, torch.tensor(2.0 ** -126, dtype=torch.float64, device="cuda"))
    codes = torch.zeros(s["case"]["slots"], y.shape[1] * y.shape[2], dtype=torch.float64, device="cuda")
    scales = torch.zeros(y.shape[1], s["case"]["slots"], dtype=torch.float64, device="cuda")
    codes.index_copy_(0, slots, (y / scale.unsqueeze(-1)).reshape(y.shape[0], -1))
    scales.index_copy_(1, slots, scale.T.contiguous())
    return codes, scales


def _exact_values(codes, scales):
    return codes.double().view(codes.shape[0], scales.shape[0], -1) * scales.double().T.unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "read":
        return _exact_values(s["codes"], s["scales"]).index_select(0, s["rows"].long()).reshape(case["rows"], -1)
    if case["op"] in ("rope", "write"):
        q, k = _exact_rotation(s["q"], s).reshape(s["q"].shape), _exact_rotation(s["k"], s)
        if case["op"] == "rope":
            return [q, k.reshape(s["k"].shape)]
        slots = s["slots"].long()
        return [q, *_exact_cache(k, s, slots),
                *_exact_cache(s["v"].double().view(case["tokens"], case["kv_heads"], -1), s, slots)]
    lens, news = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    keys, vals = _exact_values(s["k_codes"], s["k_scales"]), _exact_values(s["v_codes"], s["v_scales"])
    out, t0 = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for r, (l, n) in enumerate(zip(lens, news)):
        p = torch.arange(l, device="cuda")
        where = s["table"][r].long()[p // case["page"]] * case["page"] + p % case["page"]
        later = p[None, :] > (l - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(case["kv_heads"]):
            at = slice(h * group * case["head_dim"], (h + 1) * group * case["head_dim"])
            q = s["q"][t0: t0 + n, at].double().view(n, group, -1)
            w = torch.einsum("ngd,ld->gnl", q, keys[where, h]) * case["head_dim"] ** -0.5
            w = torch.softmax(torch.where(later, -torch.inf, w), -1)
            out[t0: t0 + n, at] = torch.einsum("gnl,ld->ngd", w, vals[where, h]).reshape(n, -1)
        t0 += n
    return out
