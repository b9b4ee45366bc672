"""The operators of the 8-bit paged cache, as cases that can be timed and checked.

The cache holds a row of keys or values (one token, one kv head) as `hd` numbers in e4m3 and one scale byte b that stands for
2^(b - 127).  With e the smallest integer of [-100, 119] for which max|x| <= 448 * 2^e, the row's numbers are x * 2^-e rounded to e4m3 and
b = e + 127.  Four operators:

  store    `quantise_kv`: the rows of a step's new tokens into their places in the pages, then `dequantise_kv` of the same rows, as
           the numbers that attention will see
  read     `dequantise_kv`: whole sequences back out of their pages
  single   `attention_quantised` with one new token per sequence (decoding)
  chunk    `attention_quantised` with many new tokens per sequence: prompts, and chunks of prompts behind keys that are cached

Attention's position p sees the keys j <= p, with a window w those with p - j < w and beside them the first `keep_first`; a sink is a logit
per head that joins the softmax's denominator; a soft cap c turns a score s into c * tanh(s / c).  Pages hold 64 tokens and lie in the pool in no order.
Head layouts (query heads, kv heads, head size) are those of the Qwen2 presets; windows and kept first keys those of the Kebesun presets.
"""
from __future__ import annotations

import math
import random
from typing import Any, Dict, List

import torch

own = False

PAGE = 64
LAYOUTS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128)}


def _case(kind: str, layout: str, seqs: int, new: int, cached: int, name: str = "", **more: Any) -> Dict[str, Any]:
    """`seqs` sequences of `cached` keys, `new` tokens each; with `ragged` both are the largest of unequal ones."""
    c: Dict[str, Any] = dict(kind=kind, layout=layout, seqs=seqs, new=new, cached=cached, ragged=False, dtype="bfloat16",
                             window=0, keep_first=0, sinks=False, softcap=0.0)
    c.update(more)
    return dict(c, name=name) if name else c


def listed() -> List[Dict[str, Any]]:
    return [
        # what a decode step of the headline workload writes: one layer's rows of eight sequences
        _case("store", "0.5b", 8, 1, 2048, "store, 8 single tokens"),
        # one layer's rows of a long prompt of an odd length
        _case("store", "7b", 1, 8191, 0, "store, prompt of 8191"),
        # a step of ragged prompts whose projections are still float32
        _case("store", "1.5b", 12, 700, 333, "store, ragged prompts, float32", ragged=True, dtype="float32"),
        # looking at what one short conversation has in the cache
        _case("read", "0.5b", 1, 0, 300, "read, 300 tokens, float32", dtype="float32"),
        # handing a batch's caches to something that wants ordinary rows
        _case("read", "7b", 16, 0, 16000, "read, 16 ragged sequences", ragged=True),
        # one user's answer: latency
        _case("single", "0.5b", 1, 1, 1999, "single, batch 1, 2000 keys"),
        # few users far into long documents: the longest rows the presets' positions allow, keys shared out over the GPU
        _case("single", "1.5b", 2, 1, 32700, "single, batch 2, 32701 keys"),
        # a server's full batch, ragged
        _case("single", "7b", 64, 1, 8191, "single, batch 64, ragged", ragged=True),
        # layers with a window, kept first keys and sinks, a large batch
        _case("single", "0.5b", 48, 1, 5000, "single, batch 48, window", ragged=True, window=1024, keep_first=4, sinks=True),
        # a chunk of a long document: the largest
        _case("chunk", "7b", 1, 2048, 14000, "chunk of 2048 behind 14000"),
        # a prompt from nothing, odd length
        _case("chunk", "0.5b", 1, 4095, 0, "chunk, prompt of 4095"),
        # a server's step of ragged turns of running conversations, windowed layers with sinks and a soft cap
        _case("chunk", "1.5b", 12, 600, 3000, "chunk, batch 12, ragged, window", ragged=True, window=1024, keep_first=4, sinks=True,
              softcap=30.0),
    ]


def _spread(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> Dict[str, Any]:
    kind = rng.choice(["store", "read", "single", "single", "chunk", "chunk"])
    layout = rng.choice(sorted(LAYOUTS))
    heads, kv_heads, hd = LAYOUTS[layout]
    more: Dict[str, Any] = {}
    if kind in ("store", "read"):
        more["dtype"] = rng.choice(["bfloat16", "bfloat16", "float32"])
    else:
        if rng.random() < 0.4:
            more.update(window=_spread(rng, 1, 4096), keep_first=rng.choice([0, 1, 4, 100]))
        more.update(sinks=rng.random() < 0.3, softcap=30.0 if rng.random() < 0.2 else 0.0)
    if kind == "store":
        seqs = _spread(rng, 1, 64)
        new, cached = _spread(rng, 1, max(1, 8191 // seqs)), rng.choice([0, rng.randint(1, 4000)])
    elif kind == "read":
        seqs = _spread(rng, 1, 64)
        new, cached = 0, _spread(rng, 1, min(32768, 256000 // seqs))
    elif kind == "single":
        seqs = _spread(rng, 1, 64)
        new, cached = 1, _spread(rng, 1, min(32767, 520000 // seqs))
    else:
        seqs = _spread(rng, 1, 16)
        new = _spread(rng, 2, 4096 // seqs)
        cached = rng.choice([0, _spread(rng, 1, min(16000, 30_000_000 // (seqs * new)))])
    return _case(kind, layout, seqs, new, cached, ragged=seqs > 1 and rng.random() < 0.6, **more)


def _lengths(case: Dict[str, Any]) -> List[List[int]]:
    """(cached keys, new tokens) of each sequence; every seed has the same ones in another order."""
    n, new, cached = case["seqs"], case["new"], case["cached"]
    if not case["ragged"]:
        return [[cached, new]] * n
    rng = random.Random(cached * 1000 + new * 10 + n)
    return [[cached, new]] + [[rng.randint(min(1, cached), cached), rng.randint(min(1, new), new)] for _ in range(n - 1)]


def _shapes(case: Dict[str, Any]) -> List[List[int]]:
    """The same, and for each sequence how many of its keys are visible to one of its new tokens at least."""
    out = []
    for cached, new in _lengths(case):
        w = case["window"] or cached + new
        first_of_window = max(0, cached - w + 1)
        out.append([cached, new, cached + new - first_of_window + min(case["keep_first"] if case["window"] else 0, first_of_window)])
    return out


# --------------------------------------------------------------------------- what a program has before the call

def _plain_quantise(x: torch.Tensor):
    """Rows [..., hd] -> (e4m3 numbers, scale bytes), float32 arithmetic in which every step but the last rounding is exact."""
    x = x.float()
    mantissa, exponent = torch.frexp(x.abs().amax(dim=-1))               # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(-100, 119)    # 448 = 0.875 * 2^9
    codes = torch.ldexp(x, -e[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _plain_values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(codes.float(), scale.int()[..., None] - 127)


def prepare(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    dev = torch.device("cuda")
    heads, kv_heads, hd = LAYOUTS[case["layout"]]
    dtype = getattr(torch, case["dtype"])
    gen = torch.Generator(device=dev).manual_seed(seed)
    order = random.Random(seed)
    lengths = list(_lengths(case))
    order.shuffle(lengths)
    n_seqs = len(lengths)
    total = [c + n for c, n in lengths]
    width = max((t + PAGE - 1) // PAGE for t in total)
    used = sum((t + PAGE - 1) // PAGE for t in total)
    n_pages = used + 3
    pages = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed))[:used].tolist()
    table = torch.full((n_seqs, width), -1, dtype=torch.int32)
    at = 0
    for s, t in enumerate(total):
        n = (t + PAGE - 1) // PAGE
        table[s, :n] = torch.tensor(pages[at:at + n], dtype=torch.int32)
        at += n
    if case["window"]:                # pages that the window has passed were given back, but for those of kept first keys
        for s, (c, n) in enumerate(lengths):
            kept = (case["keep_first"] + PAGE - 1) // PAGE
            table[s, kept:max(kept, max(0, c - case["window"] + 1) // PAGE)] = -1

    def rows(*shape: int) -> torch.Tensor:
        """Keys or values: normal numbers, channels of unequal size, a few of them large, and rows of unequal size."""
        x = torch.randn(*shape, generator=gen, device=dev)
        channels = 0.3 + torch.rand(shape[-1], generator=gen, device=dev)
        channels[torch.randint(0, shape[-1], (2,), generator=gen, device=dev)] *= 6.0
        return x * channels * torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=gen, device=dev))

    state: Dict[str, Any] = dict(case=case)
    shape = (1, n_pages, kv_heads, PAGE, hd)
    k_pool, k_scale = _plain_quantise(rows(*shape).to(torch.bfloat16))
    v_pool, v_scale = _plain_quantise(rows(*shape).to(torch.bfloat16))
    state.update(k_pool=k_pool, v_pool=v_pool, k_scale=k_scale, v_scale=v_scale, table=table.to(dev))
    # which rows a call is about: the new tokens, or with `read` all that is cached
    spans = [(0, c) for c, _ in lengths] if case["kind"] == "read" else [(c, n) for c, n in lengths]
    n_rows = sum(n for _, n in spans)
    positions = torch.cat([torch.arange(a, a + n, dtype=torch.int32) for a, n in spans])
    tok_seq = torch.cat([torch.full((n,), s, dtype=torch.int32) for s, (_, n) in enumerate(spans)])
    cu = torch.tensor([0] + [n for _, n in spans]).cumsum(0).int()
    start = torch.tensor([a for a, _ in spans], dtype=torch.int32)
    state.update(positions=positions.to(dev), tok_seq=tok_seq.to(dev), cu=cu.to(dev), start=start.to(dev),
                 n_seqs=n_seqs, max_q=max(n for _, n in spans), max_kv=max(total))
    if case["kind"] == "store":
        state.update(k=rows(n_rows, kv_heads, hd).to(dtype), v=rows(n_rows, kv_heads, hd).to(dtype))
    if case["kind"] in ("store", "read"):
        state.update(k_out=torch.empty(n_rows, kv_heads, hd, dtype=dtype, device=dev),
                     v_out=torch.empty(n_rows, kv_heads, hd, dtype=dtype, device=dev))
    else:
        q = torch.randn(n_rows, heads * hd, generator=gen, device=dev) * 1.5
        state.update(q=q.to(dtype), out=torch.empty(n_rows, heads * hd, dtype=dtype, device=dev), scale=hd ** -0.5,
                     sinks=torch.randn(heads, generator=gen, device=dev) if case["sinks"] else None)
    return state


# --------------------------------------------------------------------------- one pass

def _plain_store(s: Dict[str, Any]) -> None:
    pos, seq = s["positions"].long(), s["tok_seq"].long()
    page, at = s["table"][seq, pos // PAGE].long(), pos % PAGE
    k, ks = _plain_quantise(s["k"])
    v, vs = _plain_quantise(s["v"])
    s["k_pool"].view(torch.uint8)[0, page, :, at] = k.view(torch.uint8)
    s["v_pool"].view(torch.uint8)[0, page, :, at] = v.view(torch.uint8)
    s["k_scale"][0, page, :, at] = ks
    s["v_scale"][0, page, :, at] = vs


def _plain_read(s: Dict[str, Any]):
    pos, seq = s["positions"].long(), s["tok_seq"].long()
    page, at = s["table"][seq, pos // PAGE].long(), pos % PAGE
    dtype = s["k_out"].dtype
    k = _plain_values(s["k_pool"].view(torch.uint8)[0, page, :, at].view(torch.float8_e4m3fn), s["k_scale"][0, page, :, at])
    v = _plain_values(s["v_pool"].view(torch.uint8)[0, page, :, at].view(torch.float8_e4m3fn), s["v_scale"][0, page, :, at])
    return k.to(dtype), v.to(dtype)


def _plain_attention(s: Dict[str, Any]) -> torch.Tensor:
    """Sequences side by side, padded to the longest: keys [seqs, kv heads, keys, hd], queries [seqs, kv heads, group * tokens, hd]."""
    case = s["case"]
    heads, kv_heads, hd = LAYOUTS[case["layout"]]
    group, n_seqs, max_q = heads // kv_heads, s["n_seqs"], s["max_q"]
    dev = s["q"].device
    page = s["table"].long().clamp(min=0)
    n_keys = page.shape[1] * PAGE
    k = _plain_values(s["k_pool"].view(torch.uint8)[0, page].view(torch.float8_e4m3fn), s["k_scale"][0, page])
    v = _plain_values(s["v_pool"].view(torch.uint8)[0, page].view(torch.float8_e4m3fn), s["v_scale"][0, page])
    k = k.permute(0, 2, 1, 3, 4).reshape(n_seqs, kv_heads, n_keys, hd)
    v = v.permute(0, 2, 1, 3, 4).reshape(n_seqs, kv_heads, n_keys, hd)
    row = torch.arange(max_q, device=dev)
    q = s["q"].float().view(-1, kv_heads, group, hd)[(s["cu"][:-1, None] + row).long().clamp(max=s["q"].shape[0] - 1)]
    q = q.permute(0, 2, 3, 1, 4).reshape(n_seqs, kv_heads, group * max_q, hd)
    score = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(n_seqs, kv_heads, group, max_q, n_keys)
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    p, j = (s["start"][:, None] + row)[:, :, None], torch.arange(n_keys, device=dev)
    seen = (j <= p) & (s["table"] >= 0).repeat_interleave(PAGE, dim=1)[:, None, :]
    if case["window"]:
        seen = seen & ((p - j < case["window"]) | (j < case["keep_first"]))
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = torch.exp(score - top)
    total = w.sum(dim=-1, keepdim=True)
    if case["sinks"]:
        total = total + torch.exp(s["sinks"].view(1, kv_heads, group, 1, 1) - top)
    o = torch.matmul(w.view(n_seqs, kv_heads, group * max_q, n_keys), v).view(n_seqs, kv_heads, group, max_q, hd) / total
    seq = s["tok_seq"].long()
    return o[seq, :, :, s["positions"].long() - s["start"].long()[seq]].reshape(-1, heads * hd).to(s["q"].dtype)


def run(state: Dict[str, Any]) -> Any:
    s, case = state, state["case"]
    if own:
        from mini_llama_cpp_release_b200 import kernels
        heads, kv_heads, hd = LAYOUTS[case["layout"]]
        kv = kernels.QuantisedKVView(s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], 0, s["table"], PAGE, kv_heads, hd)
        if case["kind"] == "store":
            kernels.quantise_kv(s["k"], s["v"], s["positions"], s["tok_seq"], kv)
        if case["kind"] in ("store", "read"):
            kernels.dequantise_kv(s["k_out"], s["v_out"], s["positions"], s["tok_seq"], kv)
            return s["k_out"], s["v_out"]
        kernels.attention_quantised(s["q"], s["out"], s["cu"], s["start"], s["n_seqs"], s["max_q"], s["max_kv"], heads, kv, s["scale"],
                                    case["window"], sinks=s["sinks"], keep_first=case["keep_first"], softcap=case["softcap"])
        return s["out"]
    if case["kind"] == "store":
        _plain_store(s)
    if case["kind"] in ("store", "read"):
        return _plain_read(s)
    return _plain_attention(s)


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case: Dict[str, Any]) -> Dict[str, float]:
    heads, kv_heads, hd = LAYOUTS[case["layout"]]
    item = 4 if case["dtype"] == "float32" else 2
    shapes = _shapes(case)
    new = sum(n for _, n, _ in shapes)
    if case["kind"] == "store":
        rows = 2 * new * kv_heads                     # read, written as codes, read back and written as numbers
        return {"bytes": float(rows * (hd * item + 2 * (hd + 1) + hd * item)), "flops": 0.0}
    if case["kind"] == "read":
        rows = 2 * sum(c for c, _, _ in shapes) * kv_heads
        return {"bytes": float(rows * (hd + 1 + hd * item)), "flops": 0.0}
    keys = sum(k for _, _, k in shapes)
    pairs = 0                                         # (new token, key that it sees)
    for cached, n, _ in shapes:
        for p in range(cached, cached + n):
            w = min(case["window"] or p + 1, p + 1)
            pairs += w + (min(case["keep_first"], p + 1 - w) if case["window"] else 0)
    return {"bytes": float(2 * keys * kv_heads * (hd + 1) + 2 * new * heads * hd * item), "flops": 4.0 * pairs * heads * hd}


# --------------------------------------------------------------------------- the definition, in 64 bits

def _e4m3_numbers(dev: torch.device) -> torch.Tensor:
    """What each of the 256 bytes stands for."""
    out = []
    for b in range(256):
        exponent, fraction = (b >> 3) & 15, b & 7
        x = math.ldexp(fraction, -9) if exponent == 0 else math.ldexp(8 + fraction, exponent - 10)
        out.append(math.nan if b & 127 == 127 else -x if b & 128 else x)
    return torch.tensor(out, dtype=torch.float64, device=dev)


def _exact_rows(x: torch.Tensor) -> torch.Tensor:
    """What the cache makes of the rows x [..., hd], by the format's definition."""
    x = x.double()
    amax = x.abs().amax(dim=-1, keepdim=True)
    e = torch.ceil(torch.log2(amax / 448.0)).clamp(-100, 119)
    e = torch.where((448.0 * torch.exp2(e) < amax) & (e < 119), e + 1, e)            # log2 may be a bit off either way
    e = torch.where((448.0 * torch.exp2(e - 1) >= amax) & (e > -100), e - 1, e)
    y = x * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(y / step) * step * torch.exp2(e)                              # round: halves go to the even multiple


def exact(case: Dict[str, Any], seed: int) -> Any:
    s = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_rows(s["k"]), _exact_rows(s["v"])
    heads, kv_heads, hd = LAYOUTS[case["layout"]]
    numbers = _e4m3_numbers(s["k_pool"].device)

    def sequence(b: int, n: int):
        """Keys and values [n, kv heads, hd] of sequence b; zeros where its page is gone."""
        n_pages = (n + PAGE - 1) // PAGE
        page = s["table"][b, :n_pages].long()
        both = []
        for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])):
            x = numbers[pool.view(torch.uint8)[0, page.clamp(min=0)].long()] * torch.exp2(scale[0, page.clamp(min=0)].double() - 127.0)[..., None]
            both.append((x * (page >= 0).view(-1, 1, 1, 1)).transpose(1, 2).reshape(n_pages * PAGE, kv_heads, hd)[:n])
        return both

    cu, start = s["cu"].tolist(), s["start"].tolist()
    if case["kind"] == "read":
        both = [sequence(b, cu[b + 1] - cu[b]) for b in range(s["n_seqs"])]
        return torch.cat([k for k, _ in both]), torch.cat([v for _, v in both])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(s["n_seqs"]):
        n, n_new = start[b] + cu[b + 1] - cu[b], cu[b + 1] - cu[b]
        k, v = sequence(b, n)
        p = torch.arange(start[b], n, device=out.device)[:, None]
        j = torch.arange(n, device=out.device)[None, :]
        seen = j <= p
        if case["window"]:
            seen &= (p - j < case["window"]) | (j < case["keep_first"])
        for h in range(heads):
            q = s["q"][cu[b]:cu[b + 1], h * hd:(h + 1) * hd].double()
            score = q @ k[:, h // (heads // kv_heads)].T * s["scale"]
            if case["softcap"]:
                score = case["softcap"] * torch.tanh(score / case["softcap"])
            score[~seen] = -math.inf
            if case["sinks"]:
                score = torch.cat([score, s["sinks"][h].double().expand(n_new, 1)], dim=1)
            w = torch.softmax(score, dim=1)[:, :n]
            out[cu[b]:cu[b + 1], h * hd:(h + 1) * hd] = w @ v[:, h // (heads // kv_heads)]
    return out
