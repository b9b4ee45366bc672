"""The 8-bit cache without a GPU: options, sizes, views, the format's plain form."""
import math

import pytest
import torch

import plain_quantised as plain
from mini_llama_cpp_release_b200 import EngineConfig, cli
from mini_llama_cpp_release_b200.cache.paged import PagedCache
from mini_llama_cpp_release_b200.kernels import KernelError, QuantisedKVView, attention_q8_plan, attention_q8_tcgen05_plan, quantise_kv
from mini_llama_cpp_release_b200.parts.base import CacheNeed


def test_engine_option():
    for name in ("float8_e4m3", "fp8", torch.float8_e4m3fn):
        assert EngineConfig(cache_dtype=name).cache_dtype == torch.float8_e4m3fn
    assert EngineConfig().cache_dtype == torch.bfloat16 and EngineConfig(dtype="fp32").cache_dtype == torch.float32
    assert EngineConfig(cache_dtype="bf16").cache_dtype == torch.bfloat16
    for bad in (dict(dtype="fp32", cache_dtype="fp8"), dict(cache_dtype="float32"), dict(dtype="fp32", cache_dtype="bf16"), dict(cache_dtype="e5m2"), dict(cache_dtype=8)):
        with pytest.raises(ValueError):
            EngineConfig(**bad)


def test_command_line_option():
    import argparse
    ap = argparse.ArgumentParser()
    cli.add_engine_options(ap)
    assert cli.engine_config(ap.parse_args(["--cache-dtype", "fp8"]), 64).cache_dtype == torch.float8_e4m3fn
    assert cli.engine_config(ap.parse_args([]), 64).cache_dtype == torch.bfloat16
    with pytest.raises(SystemExit, match="8-bit cache"):
        cli.engine_config(ap.parse_args(["--cache-dtype", "fp8", "--dtype", "float32"]), 64)


def needs():
    return [CacheNeed("all", 2, 64), CacheNeed("window", 1, 128, 100, 4), CacheNeed("all", 2, 64), CacheNeed("all", 1, 48, shared_kv=True)]


def test_pools_and_views():
    c = PagedCache(needs(), [None] * 4, [None] * 4, 640, 4, torch.float8_e4m3fn, torch.device("cpu"))
    assert c.quantised and [tuple(p.shape) for p in c.k_pools] == [(2, 10, 2, 64, 64), (1, 10, 1, 64, 128), (1, 10, 1, 64, 48)]
    assert [tuple(s.shape) for s in c.v_scales] == [(2, 10, 2, 64), (1, 10, 1, 64), (1, 10, 1, 64)]
    assert c.v_pools[2] is c.k_pools[2] and c.v_scales[2] is c.k_scales[2] and c.v_scales[0] is not c.k_scales[0]
    assert c.bytes_per_token() == 2 * 2 * 2 * 65 + 2 * 129 + 49
    assert c.bytes() == 640 * c.bytes_per_token()
    tables = [torch.zeros(1, 3, dtype=torch.int32)] * 3
    v = c.view(2, tables)
    assert isinstance(v, QuantisedKVView) and v.entry_offset == 10 * 2 * 64 * 64 and v.k_scale is c.k_scales[0] and v.pages_per_seq == 3
    wide = PagedCache(needs(), [None] * 4, [None] * 4, 640, 4, torch.bfloat16, torch.device("cpu"))
    assert not wide.quantised and wide.k_scales == [None] * 3 and wide.bytes_per_token() == 2 * (2 * 2 * 2 * 64 + 2 * 128 + 48)
    assert wide.bytes() == 640 * wide.bytes_per_token()


@pytest.mark.parametrize("head_dim,page", [(40, 64), (272, 64), (64, 32)])
def test_sizes_it_does_not_take(head_dim, page):
    with pytest.raises(ValueError, match="8-bit cache"):
        PagedCache([CacheNeed("all", 1, head_dim)], [None], [None], 640, 4, torch.float8_e4m3fn, torch.device("cpu"), page)


def test_a_cache_on_the_host_is_refused():
    c = PagedCache(needs()[:1], [None], [None], 640, 4, torch.float8_e4m3fn, torch.device("cpu"))
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(KernelError, match="CUDA"):
        quantise_kv(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), i, i, c.view(0, [torch.zeros(1, 1, dtype=torch.int32)]))


def test_plans_cover_every_key():
    for q_len in (1, 2, 5, 40, 700):
        for seqs in (1, 3, 64, 300):
            for keys in (1, 64, 65, 2000, 131072):
                for heads, kv_heads, hd in ((14, 2, 64), (28, 4, 128), (8, 8, 16), (40, 1, 256), (64, 1, 64)):
                    for mask in (dict(), dict(window=100), dict(window=5000, keep_first=70), dict(chunk=256)):
                        rows, n, per, cluster = attention_q8_plan(q_len, seqs, max(keys, q_len), heads, kv_heads, hd, 148, **mask)
                        tiles = (max(keys, q_len) + 63) // 64
                        assert rows in (8, 16, 64) and n >= 1 and per >= 0
                        assert per == 0 or n * per >= tiles or mask, (q_len, seqs, keys)
                        assert not cluster or (1 < n <= 8 and rows != 64)
                        p = attention_q8_tcgen05_plan(q_len, seqs, max(keys, q_len), heads, kv_heads, hd, 148, **mask)
                        assert p is None or p[0] >= 1 and (p[0] > 1) == (p[1] > 0) and p[1] <= q_len


def test_the_plain_form_of_the_format():
    values = plain.code_values()
    assert values[0x7e] == 448 and values[1] == 2.0 ** -9 and values[8] == 2.0 ** -6 and math.isnan(values[0x7f]) and values[0xff].isnan()
    x = torch.tensor([[448.0, 1.0], [449.0, -449.0], [0.0, 0.0], [math.inf, 1.0], [1e-45, 0.0], [3.4e38, -3.4e38]])
    codes, scale = plain.quantise(x)
    assert scale.tolist() == [127, 128, 27, 255, 27, 246]
    back = plain.values(codes, scale)
    assert back[0].tolist() == [448, 1] and back[1].tolist() == [448, -448] and back[2].tolist() == [0, 0] and back[3].isnan().all()
    # 3.4e38 is 511.6 times 2^119: it saturates at 448
    assert back[5].tolist() == [448 * 2.0 ** 119, -448 * 2.0 ** 119]
    # a rounding is off by at most half a step: 2^-4 of the number, or half of the smallest step of its row
    x = torch.randn(400, 64, dtype=torch.float64) * torch.exp2(torch.randint(-30, 30, (400, 1)).double())
    codes, scale = plain.quantise(x)
    step = torch.exp2(scale.double() - 127)[:, None] * 2.0 ** -9
    assert ((plain.values(codes, scale) - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, step / 2)).all()


def test_argument_lists_are_the_kernels():
    """The declared argument types of each entry point against its C signature, one by one."""
    import os
    import re
    from ctypes import c_float, c_int, c_longlong, c_void_p
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    root = os.path.dirname(bindings._build.__file__)
    names = {"P": c_void_p, "I": c_int, "F": c_float, "LL": c_longlong}
    with open(bindings.__file__) as f:
        text = f.read()
    for entry, source in (("mlc_attention_q8", "attention_q8.cu"), ("mlc_attention_q8_tcgen05", "attention_q8_tcgen05.cu"),
                          ("mlc_quantise_kv", "kv_quantise.cu"), ("mlc_dequantise_kv", "kv_quantise.cu")):
        with open(os.path.join(root, source)) as f:
            signature = re.search(r'extern "C" int ' + entry + r"\(([^)]*)\) \{", f.read()).group(1)
        want = [c_void_p if "*" in a else c_longlong if a.startswith("long long") else c_float if a.startswith("float") else c_int
                for a in (x.strip() for x in signature.replace("\n", " ").split(","))]
        declared = (re.search(rf'"{entry}": \[([^\]]*)\]', text) or re.search(rf"lib\.{entry}\.argtypes = \[([^\]]*)\]", text)).group(1)
        got = []
        for a in (x.strip() for x in declared.split(",")):
            got += bindings.QUANTISED_ARGS if a == "*QUANTISED_ARGS" else [names[a]]
        assert got == want, entry


def test_partial_results_stay_small():
    """Whatever the sizes and however far a bound lies above the lengths, splits that a second kernel joins need no more than 2 GiB."""
    for heads, kv_heads, hd in ((14, 2, 64), (28, 4, 128), (12, 4, 48), (32, 4, 256), (64, 8, 128), (8, 8, 16)):
        for q_len, seqs, keys in ((1, 1, 1 << 20), (1, 400, 1 << 20), (1, 4000, 65536), (3, 64, 200000), (16384, 1, 100000), (8192, 1, 30000), (1024, 16, 16000),
                                  (300, 2, 1 << 20), (40, 1, 1 << 20)):
            rows, n, per, cluster = attention_q8_plan(q_len, seqs, keys, heads, kv_heads, hd, 148)
            if n > 1 and not cluster:
                assert q_len * seqs * heads * n * (hd + 2) * 4 <= 2 << 30, (heads, hd, q_len, seqs, keys, n)
            p = attention_q8_tcgen05_plan(q_len, seqs, keys, heads, kv_heads, hd, 148)
            if p is not None and p[0] > 1:
                assert seqs * p[1] * (128 // min(heads // kv_heads, 128)) * heads * p[0] * (hd + 2) * 4 <= 2 << 30, (heads, hd, q_len, seqs, keys, p)


def test_warps_come_whole_to_the_clusters_barriers():
    """`barrier.cluster` in its aligned form is for whole warps: behind a loop that lanes leave one by one they are brought together first."""
    import os
    import re
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    with open(os.path.join(os.path.dirname(bindings._build.__file__), "attention_q8.cu")) as f:
        code = [line for line in (re.sub(r"//.*", "", x).strip() for x in f) if line]
    before = [code[i - 1] for i, line in enumerate(code) if line == "cluster_sync_all();"]
    assert len(before) == 2 and all(line == "__syncwarp();" for line in before)


@pytest.mark.parametrize("bad", [dict(scale=math.inf), dict(scale=math.nan), dict(scale=0.0), dict(softcap=math.inf), dict(softcap=1e6), dict(softcap=-1.0),
                                 dict(softcap=math.nan), dict(window=-1), dict(chunk=-1), dict(keep_first=-1), dict(window=4, chunk=4)], ids=str)
def test_attention_options_that_have_no_answer(bad):
    from mini_llama_cpp_release_b200.kernels import attention_quantised
    c = PagedCache(needs()[:1], [None], [None], 640, 4, torch.float8_e4m3fn, torch.device("cpu"))
    view = c.view(0, [torch.zeros(1, 1, dtype=torch.int32)])
    q = torch.zeros(1, 2 * 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(KernelError, match="softcap"):
        attention_quantised(q, q, i, i, 1, 1, 1, 2, view, **{**dict(scale=0.125), **bad})
    with pytest.raises(KernelError, match="CUDA"):
        attention_quantised(q, q, i, i, 1, 1, 1, 2, view, 0.125, softcap=2048.0)


def test_what_a_soft_cap_rounds():
    """cap * (1 - q), q = 2 / (1 + e^2y), in float32, the quotient two units off as a fast division may be, for scores of every size.  q <= 2: its two units are 2^-22 at most,
    the exponential and the sum below it are rounded to 2^-24 of themselves and move q by 2^-23 each at most, the difference is rounded by 2^-24: together less than
    cap * 2^-21.  So caps up to 2,048 stay within 2^-10, and one of a million would move a score by tenths."""
    worst = {}
    for cap in (0.5, 30.0, 2048.0, 1e6):
        score = torch.linspace(-3.0, 3.0, 20001, dtype=torch.float64) * min(cap, 64.0) / 3.0
        quotient = 2.0 / (1.0 + torch.exp(2.0 * score / cap).float())
        for units in (-2, 0, 2):
            got = cap * (1.0 - quotient * (1.0 + units * 2.0 ** -24)).double()
            worst[cap] = max(worst.get(cap, 0.0), float((got - cap * torch.tanh(score / cap)).abs().max()))
        assert worst[cap] < cap * 2.0 ** -21
    assert worst[2048.0] <= 2.0 ** -10 and worst[1e6] > 0.1


def test_a_wait_that_ran_out_keeps_the_warp_together():
    """What follows the row threads' waits (tensor memory, shuffles) is for whole warps.  So either the warp decides together whether a wait ran out, or the thread
    stays: it waits no more (`if (ok) ok = ...`) and no loop over tiles is left by some lanes only."""
    import os
    import re
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    root = os.path.dirname(bindings._build.__file__)
    for source, code in (("attention_q8_tcgen05.cu", "76"), ("attention_q8.cu", "72")):
        with open(os.path.join(root, source)) as f:
            lines = [re.sub(r"//.*", "", x).strip() for x in f]
        waits = [i for i, x in enumerate(lines) if "mbar_wait(" in x and f"a.status, {code})" in x]
        assert waits
        for i in waits:
            if "__all_sync(0xffffffffu, mbar_wait(" not in lines[i]:
                assert lines[i].startswith("if (ok) ok = mbar_wait(") or lines[i + 1] == "}", lines[i]
                assert lines[i + 1] != "if (!ok) break;", lines[i]


def test_places_of_the_pages_that_are_written_out():
    """Every page that some new token sees has a place of its own below the number that is asked for, wherever the sequence stands; under a mask that number follows the
    mask and not the page list."""
    import random
    from mini_llama_cpp_release_b200.kernels import attention_q8_places
    rng = random.Random(1)
    for _ in range(4000):
        kind = rng.choice(["all", "window", "kept", "chunk"])
        size, keep = rng.randint(1, 700), rng.randint(1, 300) if kind == "kept" else 0
        mask = {} if kind == "all" else dict(chunk=size) if kind == "chunk" else dict(window=size, keep_first=keep)
        heads, kv_heads = rng.choice([(14, 2), (12, 2), (28, 4), (4, 4), (40, 2), (300, 1)])
        block = 128 // min(heads // kv_heads, 128)
        start, new = rng.randint(0, 4000), rng.randint(1, 300)
        end = start + -(-new // block) * block                              # rows of the last block that do not exist take part in the walk
        last = max(0, (start + new + 63) // 64 + rng.randint(-3, 40) - 1)   # of the page list, which may end before the sequence or go on behind it
        lowest = 0 if kind == "all" else start // size * size if kind == "chunk" else max(0, start - size + 1)
        n = attention_q8_places(rng.randint(new, end - start), last + 1, heads, kv_heads, **mask)
        seen = [t for t in range(min((end - 1) // 64, last) + 1) if 64 * t + 63 >= lowest or t < -(-keep // 64)]
        first = min(lowest // 64, last)                                     # the kernels' rule, csrc/attention_q8_tcgen05.cu (Q8Places)
        head = min(first, -(-keep // 64))
        places = [t if t < head else t - (first - head) for t in seen]
        assert len(set(places)) == len(places) and all(0 <= x < n for x in places), (mask, start, new, last)
        assert n <= last + 1 and (kind == "all" or n <= (size + end - start) // 64 + 2 + -(-keep // 64))


def test_scratch_memory_for_pages_written_out(monkeypatch):
    """Several sequences take half a GiB at most, one as much as it needs up to the limit, in equal groups; fewer at a time where there is no room."""
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    made = []

    def empty(n, dtype, device):
        if 2 * n > room:
            raise torch.OutOfMemoryError("no room")
        made.append(n)
        return n

    monkeypatch.setattr(bindings.torch, "empty", empty)
    for per_seq, n_seqs, room, want in ((1000, 7, 1 << 40, 7), (1 << 26, 128, 1 << 40, 4), (1 << 26, 9, 1 << 40, 3), (1 << 26, 5, 1 << 40, 3), (1 << 30, 3, 1 << 40, 1), (1 << 32, 1, 1 << 40, 1),
                                        ((1 << 32) + 1, 1, 1 << 40, 0), (1 << 26, 128, 1 << 28, 2), (1 << 26, 128, 1 << 27, 1), (1 << 26, 128, (1 << 27) - 1, 0)):
        del made[:]
        at_once, tensor = bindings._expanded_pages(per_seq, n_seqs, torch.device("cpu"))
        assert at_once == want and (tensor == want * per_seq if want else tensor is None) and len(made) == bool(want), (per_seq, n_seqs, room)
        assert want <= 1 or 2 * want * per_seq <= bindings.EXPANDED_AT_ONCE


@pytest.mark.parametrize("name,want", [("A", "256 B in bfloat16, 512 B in float32, 136 B in float8_e4m3"), ("kebesun/big_latent", "not in 8 bits")])
def test_inspect_says_what_a_token_takes_in_8_bits(name, want, capsys):
    import helpers
    folder = helpers.model_folder(name) if "/" not in name else __import__(name.split("/")[0] + "_helpers").folder_of(name.split("/")[1])
    assert cli.main(["inspect", folder]) == 0
    assert want in capsys.readouterr().out


def test_lengths_of_masks_past_32_bits(monkeypatch):
    """A window, kept keys or a chunk longer than any sequence reaches the kernels as the longest length that 32 bits hold with a page above it, not as its low bits."""
    import types
    import mini_llama_cpp_release_b200.kernels.bindings as bindings
    seen = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: seen.append((name, a)) or 0

    for patch in (("_on_device", lambda *a: None), ("_sm_count", lambda d: 148), ("_stream", lambda: 0), ("gemm_status", lambda d: torch.zeros(1, dtype=torch.int32))):
        monkeypatch.setattr(bindings, *patch)
    monkeypatch.setitem(bindings._attn_q8_libs, 64, Lib())
    kv = types.SimpleNamespace(check=lambda: -7, args=(0, 0, 0, 0, 0, 1, 3, 0, 3, 64), kv_heads=2, head_dim=64, page_size=64, page_table=torch.zeros(1, 3, dtype=torch.int32))
    i = torch.zeros(2, dtype=torch.int32)
    for n in (1, 40):
        q = torch.zeros(n, 14 * 64, dtype=torch.bfloat16)
        for mask in (dict(window=(1 << 32) + 5), dict(window=3, keep_first=(1 << 31) - 1), dict(chunk=1 << 40), dict(window=1 << 31, keep_first=1 << 33)):
            del seen[:]
            bindings.attention_quantised(q, q, i, i, 1, n, 190, 14, kv, 0.125, **mask)
            name, a = seen[0]
            assert name == ("mlc_attention_q8" if n == 1 else "mlc_attention_q8_tcgen05")
            assert a[11:14] == tuple(min(mask.get(k, 0), (1 << 31) - 256) for k in ("window", "keep_first", "chunk"))
            assert all(x + 128 < 1 << 31 for x in a[11:14])
