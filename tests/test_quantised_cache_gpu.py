"""The 8-bit cache's rows: stored and read back bit for bit as the format's definition says."""
import math

import pytest
import torch

import plain_quantised as plain

pytestmark = pytest.mark.gpu


def kernels():
    from mini_llama_cpp_release_b200 import kernels as k
    return k


def make_cache(kv_heads, hd, n_pages, entries=1, shared=False, page_size=64, fill=0xA5):
    dev = "cuda"
    k = torch.full((entries, n_pages, kv_heads, page_size, hd), fill, dtype=torch.uint8, device=dev)
    v = k if shared else k.clone()
    ks = torch.full((entries, n_pages, kv_heads, page_size), 77, dtype=torch.uint8, device=dev)
    vs = ks if shared else ks.clone()
    return k, v, ks, vs


def view(cache, entry, table):
    k, v, ks, vs = cache
    e4 = torch.float8_e4m3fn
    vv = k.view(e4)
    return kernels().QuantisedKVView(vv, vv if v is k else v.view(e4), ks, vs, entry * k[0].numel(), table, k.shape[3], k.shape[2], k.shape[4])


def special_rows(n, kv_heads, hd, dtype, seed):
    """Rows of every size, with ties, maxima at the borders of the scale, zeros, and numbers far below the row's largest."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, kv_heads, hd, generator=g)
    x = x * torch.exp2(torch.randint(-20, 20, (n, kv_heads, 1), generator=g).float())
    x = x * torch.exp2(-torch.randint(0, 14, (n, kv_heads, hd), generator=g).float())
    grid = torch.randint(-896, 897, (n, kv_heads, hd), generator=g).float() / 16.0          # many exact ties of e4m3
    pick = torch.arange(n) % 4
    x = torch.where((pick == 1)[:, None, None], grid, x)
    x[:, :, 0] = torch.where((pick == 2)[:, None], torch.tensor(448.0), x[:, :, 0])
    x[:, :, hd - 1] = torch.where((pick == 3)[:, None], torch.tensor(-450.0), x[:, :, hd - 1])
    if n > 8:
        x[5] = 0.0
        x[6] = -0.0
        x[7] = 2.0 ** -126 * torch.randn(kv_heads, hd, generator=g)
        x[8] = 3.0e38 * torch.rand(kv_heads, hd, generator=g)
    return x.to(dtype)


@pytest.mark.parametrize("hd", [16, 48, 64, 128, 256, 512])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,kv_heads", [(1, 1), (3, 2), (257, 5)])
def test_stored_and_read_back_as_defined(hd, dtype, n, kv_heads):
    K = kernels()
    g = torch.Generator().manual_seed(hd + n)
    k, v = special_rows(n, kv_heads, hd, dtype, 1), special_rows(n, kv_heads, hd, dtype, 2)
    # two sequences whose tokens are mixed, the second from an odd position on
    tok_seq = torch.randint(0, 2, (n,), generator=g).int()
    start = [0, 61]
    positions = torch.tensor([start[s] + int((tok_seq[:i] == s).sum()) for i, s in enumerate(tok_seq.tolist())]).int()
    n_pages = 13
    table = torch.full((2, 6), -1, dtype=torch.int32)
    table.view(-1)[:12] = torch.randperm(n_pages, generator=g)[:12].int()
    cache = make_cache(kv_heads, hd, n_pages, entries=3)
    before = [t.clone() for t in cache]
    kv = view(cache, 1, table.cuda())
    K.quantise_kv(k.cuda(), v.cuda(), positions.cuda(), tok_seq.cuda(), kv)
    page, at = table[tok_seq.long(), positions.long() // 64].long(), positions.long() % 64
    for x, pool, scale, b_pool, b_scale in ((k, cache[0], cache[2], before[0], before[2]), (v, cache[1], cache[3], before[1], before[3])):
        codes, byte = plain.quantise(x)
        want_pool, want_scale = b_pool.cpu(), b_scale.cpu()
        want_pool[1, page, :, at] = codes
        want_scale[1, page, :, at] = byte
        assert torch.equal(scale.cpu(), want_scale)
        assert torch.equal(pool.cpu(), want_pool)              # and nothing else was written
    for out_dtype in (torch.bfloat16, torch.float32):
        k_out, v_out = (torch.empty(n, kv_heads, hd, dtype=out_dtype, device="cuda") for _ in range(2))
        K.dequantise_kv(k_out, v_out, positions.cuda(), tok_seq.cuda(), kv)
        for x, got in ((k, k_out), (v, v_out)):
            assert torch.equal(got.cpu().double(), plain.values(*plain.quantise(x)))       # exact in either type


def test_every_code_reads_as_its_number():
    K = kernels()
    cache = make_cache(1, 256, 1)
    cache[0][0, 0, 0, :] = torch.arange(256, dtype=torch.uint8, device="cuda")
    cache[2][0, 0, 0, :] = torch.arange(64, dtype=torch.uint8, device="cuda") * 3 + 27
    pos = torch.arange(64, dtype=torch.int32, device="cuda")
    out = torch.empty(64, 1, 256, device="cuda")
    K.dequantise_kv(out, torch.empty_like(out), pos, torch.zeros_like(pos), view(cache, 0, torch.zeros(1, 1, dtype=torch.int32, device="cuda")))
    want = plain.values(cache[0][0, 0, 0].cpu(), cache[2][0, 0, 0].cpu()).float()
    assert torch.equal(torch.nan_to_num(out[:, 0].cpu(), nan=7.0), torch.nan_to_num(want, nan=7.0))


def test_rows_that_are_not_finite():
    K = kernels()
    x = torch.randn(6, 2, 64)
    x[1, 0, 3] = math.nan
    x[2, 1, 63] = math.inf
    x[4, 0, 0] = -math.inf
    cache = make_cache(2, 64, 2)
    pos = torch.arange(6, dtype=torch.int32, device="cuda")
    kv = view(cache, 0, torch.ones(1, 1, dtype=torch.int32, device="cuda"))
    for dtype in (torch.float32, torch.bfloat16):
        K.quantise_kv(x.to(dtype).cuda(), x.to(dtype).cuda(), pos, torch.zeros_like(pos), kv)
        bad = ~torch.isfinite(x).all(-1)
        assert torch.equal(cache[2][0, 1, :, :6].cpu().T == 255, bad)
        assert not cache[0][0, 1, :, :6].cpu().transpose(0, 1)[bad].any()
        out = torch.empty(6, 2, 64, device="cuda")
        K.dequantise_kv(out, torch.empty_like(out), pos, torch.zeros_like(pos), kv)
        assert torch.equal(torch.isnan(out.cpu()).all(-1), bad) and torch.equal(torch.isnan(out.cpu()).any(-1), bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_and_unaligned_rows(dtype):
    """Keys and values as columns of one projection, also where a row starts at no multiple of 16 bytes."""
    K = kernels()
    n, kv_heads, hd = 37, 2, 64
    for first, pad in ((64, 0), (3, 5)):
        width = first + 2 * kv_heads * hd + pad
        proj = special_rows(n, 1, width, dtype, 9).view(n, width).cuda()
        k = proj[:, first:first + kv_heads * hd].unflatten(1, (kv_heads, hd))
        v = proj[:, first + kv_heads * hd:first + 2 * kv_heads * hd].unflatten(1, (kv_heads, hd))
        cache = make_cache(kv_heads, hd, 1)
        pos = torch.arange(n, dtype=torch.int32, device="cuda")
        kv = view(cache, 0, torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
        K.quantise_kv(k, v, pos, torch.zeros_like(pos), kv)
        for x, pool, scale in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
            codes, byte = plain.quantise(x.cpu())
            assert torch.equal(pool[0, 0, :, :n].cpu().transpose(0, 1), codes)
            assert torch.equal(scale[0, 0, :, :n].cpu().T, byte)
        out = torch.zeros(n, width, dtype=dtype, device="cuda")
        ko = out[:, first:first + kv_heads * hd].unflatten(1, (kv_heads, hd))
        vo = out[:, first + kv_heads * hd:first + 2 * kv_heads * hd].unflatten(1, (kv_heads, hd))
        K.dequantise_kv(ko, vo, pos, torch.zeros_like(pos), kv)
        assert torch.equal(ko.cpu().double(), plain.values(*plain.quantise(k.cpu())))
        assert torch.equal(vo.cpu().double(), plain.values(*plain.quantise(v.cpu())))
        assert not out[:, :first].any() and not out[:, width - pad:].any()


def test_missing_pages_and_sequences_without_a_list():
    """A token whose page is missing (negative, beyond the pool, beyond the list, of no sequence) is left out, and reads as zeros."""
    K = kernels()
    x = torch.randn(6, 1, 64)
    cache = make_cache(1, 64, 2)
    before = [t.clone() for t in cache]
    table = torch.tensor([[-1, 0, 2], [1, -5, 0]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, 130, 192, 70, 5, 5], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 0, 0, 1, 2, -1], dtype=torch.int32, device="cuda")
    kv = view(cache, 0, table)
    K.quantise_kv(x.cuda(), x.cuda(), pos, seq, kv)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    out = torch.ones(6, 1, 64, device="cuda")
    v_out = torch.ones(6, 1, 64, device="cuda")
    K.dequantise_kv(out, v_out, pos, seq, kv)
    assert not out.any() and not v_out.any()


def test_values_that_are_the_key_rows():
    K = kernels()
    x = special_rows(70, 1, 128, torch.bfloat16, 4)
    cache = make_cache(1, 128, 3, shared=True)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    pos = torch.arange(70, dtype=torch.int32, device="cuda")
    kv = view(cache, 0, table)
    K.quantise_kv(x.cuda(), None, pos, torch.zeros_like(pos), kv)
    out = torch.empty(70, 1, 128, dtype=torch.bfloat16, device="cuda")
    K.dequantise_kv(out, None, pos, torch.zeros_like(pos), kv)
    assert torch.equal(out.cpu().double(), plain.values(*plain.quantise(x)))
    with pytest.raises(K.KernelError):
        K.quantise_kv(x.cuda(), x.cuda(), pos, torch.zeros_like(pos), kv)


def test_offsets_beyond_32_bits():
    """An entry that starts more than 2^32 numbers into its pools."""
    K = kernels()
    entries, n_pages, kv_heads, hd = 3, 8192, 32, 128
    cache = tuple(torch.empty((entries, n_pages, kv_heads, 64, hd) if i < 2 else (entries, n_pages, kv_heads, 64), dtype=torch.uint8, device="cuda")
                  for i in range(4))
    x = special_rows(3, kv_heads, hd, torch.bfloat16, 5)
    pos = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    kv = view(cache, 2, torch.tensor([[n_pages - 1]], dtype=torch.int32, device="cuda"))
    assert kv.entry_offset >= 2 ** 32
    K.quantise_kv(x.cuda(), x.cuda(), pos, torch.zeros_like(pos), kv)
    assert torch.equal(cache[1][2, n_pages - 1, :, :3].cpu().transpose(0, 1), plain.quantise(x)[0])
    out = torch.empty(3, kv_heads, hd, dtype=torch.bfloat16, device="cuda")
    K.dequantise_kv(out, torch.empty_like(out), pos, torch.zeros_like(pos), kv)
    assert torch.equal(out.cpu().double(), plain.values(*plain.quantise(x)))


def test_captured_and_on_another_stream():
    K = kernels()
    k, v = special_rows(100, 2, 64, torch.bfloat16, 6).cuda(), special_rows(100, 2, 64, torch.bfloat16, 7).cuda()
    cache = make_cache(2, 64, 3)
    kv = view(cache, 0, torch.tensor([[1, 2]], dtype=torch.int32, device="cuda"))
    pos = torch.arange(100, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    out = [torch.empty_like(k), torch.empty_like(v)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        K.quantise_kv(k, v, pos, seq, kv)
        K.dequantise_kv(out[0], out[1], pos, seq, kv)
    stream.synchronize()
    assert torch.equal(out[0].cpu().double(), plain.values(*plain.quantise(k.cpu())))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        K.quantise_kv(k, v, pos, seq, kv)
        K.dequantise_kv(out[0], out[1], pos, seq, kv)
    for seed in (8, 9):
        k.copy_(special_rows(100, 2, 64, torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0].cpu().double(), plain.values(*plain.quantise(k.cpu())))


def test_no_tokens():
    K = kernels()
    cache = make_cache(1, 64, 1)
    kv = view(cache, 0, torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    none = torch.empty(0, 1, 64, device="cuda")
    nobody = torch.empty(0, dtype=torch.int32, device="cuda")
    K.quantise_kv(none, none, nobody, nobody, kv)
    K.dequantise_kv(none, none, nobody, nobody, kv)


def test_refusals():
    K = kernels()
    cache = make_cache(2, 64, 2)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    kv = view(cache, 0, table)
    rows = torch.zeros(3, 2, 64, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    import dataclasses
    bad_views = [
        dataclasses.replace(kv, k_pool=cache[0]),                                        # bytes, not e4m3
        dataclasses.replace(kv, k_scale=cache[2].float()),
        dataclasses.replace(kv, v_scale=cache[3][:, :1]),
        dataclasses.replace(kv, head_dim=32),
        dataclasses.replace(kv, entry_offset=64),
        dataclasses.replace(kv, entry_offset=cache[0].numel()),
        dataclasses.replace(kv, page_table=table.long()),
        dataclasses.replace(kv, page_table=table.cpu()),
        dataclasses.replace(kv, k_pool=kv.k_pool.cpu()),
    ]
    for b in bad_views:
        with pytest.raises(K.KernelError):
            K.quantise_kv(rows, rows, i, i, b)
        with pytest.raises(K.KernelError):
            K.dequantise_kv(rows, rows, i, i, b)
    for k, v, p, s in ((rows.half(), rows.half(), i, i), (rows, rows.bfloat16(), i, i), (rows[:, :1], rows[:, :1], i, i), (rows, None, i, i),
                       (rows, rows, i[:2], i), (rows, rows, i, i.long()), (rows.transpose(1, 2).contiguous().transpose(1, 2), rows, i, i),
                       (rows.cpu(), rows, i, i)):
        with pytest.raises(K.KernelError):
            K.quantise_kv(k, v, p, s, kv)
    small = make_cache(1, 24, 2)
    r24 = torch.zeros(3, 1, 24, device="cuda")
    with pytest.raises(K.KernelError):                                                   # heads are multiples of 16
        K.quantise_kv(r24, r24, i, i, view(small, 0, table))
