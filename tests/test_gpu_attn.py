"""GPU: the paged key-value cache's write and the attention over it (decode and prompt) against a
plain 64-bit implementation, element by element within bounds derived in attn_util."""
import math

import pytest

from attn_util import Setup, TYPES, check
from gpu_util import log

pytestmark = pytest.mark.gpu

MODEL = (16, 2, 256)


def run_decode(gpu, s, ref=True, **kw):
    import torch
    ctx = s.context(gpu)
    k, v = s.pools()
    q = s.q.cuda()
    lse = torch.full((s.n_rows, s.hq), 77.0, device="cuda")
    call = ctx.attn_decode if s.rows is None else ctx.attn_prompt
    o = torch.full((s.n_rows, s.hq, s.d), 55.0, dtype=s.type, device="cuda")
    call(gpu.KVCache(k, v), s.seqs(gpu), q, o=o, lse=lse, **kw)
    flags = ctx.device_flags()
    if not ref:
        return o, lse, flags
    want, bound, wl, lb = s.reference(kw.get("scale"))
    rows = [r for r, _, _ in s.row_seen()]
    rest = [r for r in range(s.n_rows) if r not in set(rows)]
    check("o", o[rows], want[rows], bound[rows])
    seen = [r for r, _, n in s.row_seen() if n]
    check("lse", lse[seen], wl[seen], lb[seen])
    for r in set(rows) - set(seen):
        assert (lse[r] == -math.inf).all()
    assert (o[rest] == 55.0).all() and (lse[rest] == 77.0).all()
    assert flags == 0
    return o, lse, flags


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("heads", [MODEL, (32, 8, 128), (12, 12, 64), (8, 1, 128), (24, 1, 64), (40, 2, 128), (3, 1, 256),
                                   (17, 1, 64)])
def test_decode_heads_and_lengths(gpu, heads, type):
    log(f"decode heads {heads} {type}")
    run_decode(gpu, Setup(*heads, 16, type, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 1000],
                          seed=1))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 512, 1024])
@pytest.mark.parametrize("order", ["hnd", "nhd", "mixed"])
def test_decode_pages_and_orders(gpu, page, order):
    log(f"decode page {page} {order}")
    run_decode(gpu, Setup(*MODEL, page, "bf16", [257, 0, 1025, 90], order=order, seed=2))


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_decode_long_single_sequences(gpu, type):
    """Split over the length: one or two sequences of many pages."""
    log(f"decode long {type}")
    run_decode(gpu, Setup(4, 2, 64, 16, type, [20011], seed=3))
    run_decode(gpu, Setup(4, 1, 128, 64, type, [9001, 5], seed=4))


def test_decode_many_sequences(gpu):
    log("decode 1500 sequences")
    kv = [(37 * b) % 53 for b in range(1500)]
    run_decode(gpu, Setup(2, 1, 64, 16, "f16", kv, seed=5))


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("heads", [MODEL, (32, 8, 128), (12, 12, 64), (24, 1, 64), (40, 2, 128), (3, 1, 256), (200, 1, 64)])
def test_prompt_heads_and_rows(gpu, heads, type):
    """Packed sequences of 0, 1 and odd numbers of rows, with and without cached tokens before them,
    and rows in front of the cache."""
    log(f"prompt heads {heads} {type}")
    rows = [1, 0, 5, 17, 64, 33, 3, 2, 70]
    before = [0, 40, 0, 100, 0, 1, -2, -2, 300]
    run_decode(gpu, Setup(*heads, 16, type, [r + c for r, c in zip(rows, before)], rows, seed=6, extra_rows=3))


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("order", ["hnd", "nhd", "mixed"])
def test_prompt_pages_and_orders(gpu, page, order):
    log(f"prompt page {page} {order}")
    run_decode(gpu, Setup(8, 2, 128, page, "f16", [150, 65, 0, 31], [150, 7, 0, 30], order=order, seed=7))


@pytest.mark.parametrize("heads", [(2, 1, 256), (4, 4, 64), (4, 1, 128)])
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_prompt_longer(gpu, heads, type):
    log(f"prompt 700 rows {heads} {type}")
    run_decode(gpu, Setup(*heads, 32, type, [700, 129], [700, 128], seed=8))


@pytest.mark.parametrize("rows", [1, 3, 20])
def test_prompt_few_rows_over_a_long_cache(gpu, rows):
    log(f"prompt {rows} rows over 12000")
    run_decode(gpu, Setup(4, 2, 128, 64, "bf16", [12000 + rows, rows], [rows, rows], seed=9))


def test_prompt_of_one_row_each_equals_decode_in_bound(gpu):
    import torch
    log("prompt as decode")
    kv = [5, 100, 33]
    run_decode(gpu, Setup(*MODEL, 16, "f16", kv, [1, 1, 1], seed=10))


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
@pytest.mark.parametrize("rows", [None, [40, 9]])
def test_scales(gpu, scale, rows):
    """scale 0 (all weights equal), negative, and large enough that one key takes nearly all."""
    log(f"scale {scale} rows {rows}")
    run_decode(gpu, Setup(8, 2, 64, 16, "f16", [150, 70], rows, seed=11), scale=scale)


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_small_weights_keep_their_bits(gpu, type):
    """One key far above 3000 equal others that together outweigh it: e^-8.4 each."""
    import torch
    log(f"small weights {type}")
    s = Setup(4, 1, 64, 16, type, [3001], seed=12)
    s.q[:] = 1.0
    s.K[0][:] = 0.0
    s.K[0][1500] = 8.4 * 8 / 64
    s.V[0][:] = torch.randn(3001, 1, 64, generator=torch.Generator().manual_seed(3)).abs().to(s.type)
    run_decode(gpu, s)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_later_tokens_do_not_reach_earlier_rows(gpu, bad):
    """A token whose key and value are not finite is seen by the rows from its own on only."""
    import torch
    log(f"prompt with {bad} at token 45 of 80")
    s = Setup(8, 2, 128, 16, "bf16", [80], [80], seed=13)
    want, bound, _, _ = s.reference()
    s.V[0][45] = bad
    s.K[0][45] = bad
    o, _, flags = run_decode(gpu, s, ref=False)
    check("o before", o[:45], want[:45], bound[:45])
    assert torch.isnan(o[45:].float()).all() and flags == 0


@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 4, 64), (2, 1, 256)])
def test_infinite_value_of_a_seen_token(gpu, heads):
    """V_j = inf in some elements: those of the rows that see it are inf, all else stays in bound."""
    import torch
    log(f"inf value {heads}")
    s = Setup(*heads, 16, "f16", [70], [70], seed=14)
    want, bound, _, _ = s.reference()
    s.V[0][30, :, 5] = float("inf")
    o, _, _ = run_decode(gpu, s, ref=False)
    assert (o[30:, :, 5] == math.inf).all()
    o[30:, :, 5] = 0
    want[30:, :, 5] = 0
    check("o", o, want, bound)


def test_minus_infinite_scores(gpu):
    """A key of -inf has weight 0; a row whose every score is -inf gets 0, as one that sees nothing."""
    import torch
    log("-inf keys")
    s = Setup(4, 2, 64, 16, "f16", [40], [40], seed=15)
    s.q = s.q.abs() + 0.1
    s.K[0][0] = float("-inf")
    s.V[0][0] = 3.0
    o, lse, _ = run_decode(gpu, s, ref=False)
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all()
    t = Setup(4, 2, 64, 16, "f16", [40], [40], seed=15)
    t.q = s.q
    ref = Setup(4, 2, 64, 16, "f16", [39], [39], seed=15)
    ref.q, ref.K, ref.V = s.q[1:], [s.K[0][1:]], [s.V[0][1:]]
    want, bound, _, _ = ref.reference()
    check("o", o[1:], want, bound)


@pytest.mark.parametrize("rows", [None, [20, 9, 4]])
def test_bad_pages_and_lengths_are_left_out_and_flagged(gpu, rows):
    import torch
    log(f"bad pages, rows {rows}")
    s = Setup(8, 2, 64, 16, "f16", [100, 50, 30], rows, seed=16, pad_pages=0)
    k, v = s.pools()
    ctx = s.context(gpu)
    call = ctx.attn_decode if rows is None else ctx.attn_prompt
    cache, q = gpu.KVCache(k, v), s.q.cuda()
    batch = s.seqs(gpu)
    good = call(cache, batch, q).clone()
    assert ctx.device_flags() == 0
    # sequence 0 loses its page 2 (tokens 32..47)
    for bad in (-1, s.n_pages, 2 ** 31 - 1, -2 ** 31):
        batch.pages[0, 2] = bad
        o = call(cache, batch, q)
        assert ctx.device_flags() == gpu.DEVFLAG_BAD_PAGE
        n0 = 1 if rows is None else rows[0]
        assert torch.equal(o[n0:], good[n0:])
        ref = Setup(8, 2, 64, 16, "f16", [84, 50, 30], rows, seed=16)
        keep = list(range(32)) + list(range(48, 100))
        ref.q, ref.K, ref.V = s.q, [s.K[0][keep]] + s.K[1:], [s.V[0][keep]] + s.V[1:]
        want, bound, _, _ = ref.reference()
        check("o", o[:n0], want[:n0], bound[:n0])
    batch.pages[0, 2] = s.pages[0, 2].item()
    # lengths out of range: below 0 is 0, behind the page list is the list's end
    batch.kv_len[2] = -5
    o = call(cache, batch, q)
    assert ctx.device_flags() == gpu.DEVFLAG_BAD_SEQ
    assert torch.equal(o[:-1 if rows is None else -4], good[:-1 if rows is None else -4])
    assert (o[-1 if rows is None else -4:] == 0).all()
    assert ctx.device_flags() == 0


def test_length_behind_the_page_list(gpu):
    import torch
    log("length behind the list")
    s = Setup(8, 2, 64, 16, "f16", [96, 50], seed=17, pad_pages=0)
    k, v = s.pools()
    ctx = s.context(gpu)
    cache, batch, q = gpu.KVCache(k, v), s.seqs(gpu), s.q.cuda()
    good = ctx.attn_decode(cache, batch, q)
    batch.kv_len[0] = 2 ** 31 - 1
    o = ctx.attn_decode(cache, batch, q)
    assert ctx.device_flags() == gpu.DEVFLAG_BAD_SEQ
    assert torch.equal(o, good)


def test_row_start_that_does_not_ascend_touches_nothing_else(gpu):
    """Every row written is one of the packed rows; nothing out of range is read or written."""
    import torch
    log("row_start not ascending")
    s = Setup(4, 2, 64, 16, "bf16", [40, 40, 40, 40], [10, 10, 10, 10], seed=18)
    k, v = s.pools()
    ctx = s.context(gpu)
    q = s.q.cuda()
    for start in ([0, 30, 10, 50, 20], [-5, 10, 20, 30, 40], [0, 10, 20, 30, 2 ** 31 - 1], [40, 30, 20, 10, 0],
                  [-2 ** 31, 0, 0, 0, 0]):
        batch = s.seqs(gpu)
        batch.row_start.copy_(torch.tensor(start, dtype=torch.int32))
        buf = torch.full((s.n_rows + 20, 4, 64), 9.0, dtype=s.type, device="cuda")
        ctx.attn_prompt(gpu.KVCache(k, v), batch, q, o=buf[10:-10])
        ctx.device_flags()
        assert (buf[:10] == 9.0).all() and (buf[-10:] == 9.0).all()


@pytest.mark.parametrize("rows", [None, [30, 12]])
def test_slices_of_wider_rows_and_output_in_place(gpu, rows):
    """q and o as slices of wider rows (what lies beside them stays), and o in q's place."""
    import torch
    log(f"slices, rows {rows}")
    s = Setup(8, 2, 128, 16, "f16", [90, 50], rows, seed=19)
    want, bound, _, _ = s.reference()
    k, v = s.pools()
    ctx = s.context(gpu)
    call = ctx.attn_decode if rows is None else ctx.attn_prompt
    wide = torch.full((s.n_rows, 14, 128), 4.0, dtype=s.type, device="cuda")
    wide[:, 2:10] = s.q.cuda()
    out = torch.full((s.n_rows, 11, 128), 6.0, dtype=s.type, device="cuda")
    call(gpu.KVCache(k, v), s.seqs(gpu), wide[:, 2:10], o=out[:, 1:9])
    check("o", out[:, 1:9], want, bound)
    assert (out[:, 0] == 6).all() and (out[:, 9:] == 6).all()
    alone = out[:, 1:9].clone()
    call(gpu.KVCache(k, v), s.seqs(gpu), wide[:, 2:10], o=wide[:, 2:10])
    assert torch.equal(wide[:, 2:10], alone)
    assert (wide[:, :2] == 4).all() and (wide[:, 10:] == 4).all()


@pytest.mark.parametrize("rows", [None, [9, 130]])
def test_same_bits_again(gpu, rows):
    import torch
    log(f"same bits, rows {rows}")
    s = Setup(*MODEL, 16, "bf16", [4000, 1000], rows, seed=20)
    k, v = s.pools()
    ctx = s.context(gpu)
    call = ctx.attn_decode if rows is None else ctx.attn_prompt
    cache, batch, q = gpu.KVCache(k, v), s.seqs(gpu), s.q.cuda()
    first = call(cache, batch, q)
    for _ in range(10):
        assert torch.equal(call(cache, batch, q), first)


def test_offsets_past_32_bits(gpu):
    """Pages that lie more than 2^32 bytes (and 2^31 elements) into the pools."""
    import torch
    log("pools of 5 GiB")
    s = Setup(2, 1, 64, 1024, "f16", [1500, 40], [300, 40], seed=21)
    small_k, small_v = s.pools()
    n = 5 * 2 ** 30 // (1024 * 64 * 2)
    k = torch.empty((n, 1, 1024, 64), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    far = [n - 1 - i * 3 for i in range(s.n_pages)]
    for i, f in enumerate(far):
        k[f], v[f] = small_k[i], small_v[i]
    assert far[-1] * 1024 * 64 > 2 ** 31
    want, bound, _, _ = s.reference()
    batch = s.seqs(gpu)
    for b, m in enumerate(s.kv):
        for t in range(-(-m // 1024)):
            batch.pages[b, t] = far[int(s.pages[b, t])]
    ctx = s.context(gpu)
    o = ctx.attn_prompt(gpu.KVCache(k, v), batch, s.q.cuda())
    check("prompt", o, want, bound)
    new = torch.randn((340, 1, 64), device="cuda")
    ctx.kv_append(gpu.KVCache(k, v), batch, new, new + 1)
    for t in (0, 299):
        pos = 1200 + t
        assert torch.equal(k[far[int(s.pages[0, pos // 1024])], 0, pos % 1024], new[t, 0].half())
    dec = Setup(2, 1, 64, 1024, "f16", [1500, 40], seed=21)
    ctx.kv_append(gpu.KVCache(k, v), batch, torch.cat([s.K[0][1200:], s.K[1]]).cuda(),
                  torch.cat([s.V[0][1200:], s.V[1]]).cuda())
    want, bound, _, _ = dec.reference()
    o = ctx.attn_decode(gpu.KVCache(k, v), gpu.SeqBatch(batch.pages, batch.kv_len), dec.q.cuda())
    check("decode", o, want, bound)
    assert ctx.device_flags() == 0


@pytest.mark.parametrize("src", ["same", "f32"])
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("order", ["hnd", "nhd", "mixed"])
@pytest.mark.parametrize("heads", [MODEL, (12, 12, 64), (5, 5, 128)])
def test_append(gpu, heads, order, type, src):
    """Every new row lands in its place, rounded to nearest even; every other place stays."""
    import torch
    log(f"append {heads} {order} {type} {src}")
    rows, before = [1, 0, 40, 3, 17], [0, 9, 5, 100, 15]
    s = Setup(*heads, 16, type, [r + c for r, c in zip(rows, before)], rows, order=order, junk=7.0, seed=22,
              extra_rows=2)
    k, v = s.pools(filled=False)
    hk = s.hkv
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn((s.n_rows, s.hq + 2 * hk, s.d), generator=g)
    # ties, values over the type's range, infinities and NaN
    qkv[0, s.hq, :6] = torch.tensor([1 + 2.0 ** -11, 1 + 3 * 2.0 ** -9, 7e4, -3.4e38, float("inf"), float("nan")])
    qkv = qkv if src == "f32" else qkv.to(s.type)
    dev = qkv.cuda()
    ctx = s.context(gpu)
    ctx.kv_append(gpu.KVCache(k, v), s.seqs(gpu), dev[:, s.hq:s.hq + hk], dev[:, s.hq + hk:])
    assert ctx.device_flags() == 0
    wk, wv = torch.full((s.n_pages, hk, 16, s.d), 7.0, dtype=s.type), torch.full((s.n_pages, hk, 16, s.d), 7.0, dtype=s.type)
    row = 0
    for b, (r, c) in enumerate(zip(rows, before)):
        for i in range(r):
            pg, t = int(s.pages[b, (c + i) // 16]), (c + i) % 16
            wk[pg, :, t] = qkv[row, s.hq:s.hq + hk].to(s.type)
            wv[pg, :, t] = qkv[row, s.hq + hk:].to(s.type)
            row += 1
    for got, want in ((k, wk), (v, wv)):
        got = got.cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(nan=1.0), want.nan_to_num(nan=1.0))


def test_append_decode_step(gpu):
    """Without row_start every sequence's one row goes to its last place."""
    import torch
    log("append decode step")
    s = Setup(8, 2, 64, 16, "f16", [1, 16, 17, 40], junk=0.0, seed=23)
    k, v = s.pools(filled=False)
    ctx = s.context(gpu)
    nk, nv = torch.randn((4, 2, 64), device="cuda"), torch.randn((4, 2, 64), device="cuda")
    ctx.kv_append(gpu.KVCache(k, v), s.seqs(gpu), nk, nv)
    for b, n in enumerate(s.kv):
        pg, t = int(s.pages[b, (n - 1) // 16]), (n - 1) % 16
        assert torch.equal(k[pg, :, t], nk[b].half()) and torch.equal(v[pg, :, t], nv[b].half())
        k[pg, :, t] = 0
        v[pg, :, t] = 0
    assert (k == 0).all() and (v == 0).all() and ctx.device_flags() == 0


def test_append_out_of_range_is_left_out_and_flagged(gpu):
    import torch
    log("append out of range")
    s = Setup(4, 2, 64, 16, "f16", [20, 20, 20], [4, 4, 4], junk=0.0, seed=24, pad_pages=0)
    ctx = s.context(gpu)
    nk = torch.ones((12, 2, 64), device="cuda")
    for what, flag in (("page", gpu.DEVFLAG_BAD_PAGE), ("short", gpu.DEVFLAG_BAD_SEQ), ("long", gpu.DEVFLAG_BAD_SEQ)):
        k, v = s.pools(filled=False)
        batch = s.seqs(gpu)
        if what == "page":
            batch.pages[1, 1] = s.n_pages
        elif what == "short":
            batch.kv_len[1] = 0
        else:
            batch.kv_len[1] = 2 ** 31 - 1
        ctx.kv_append(gpu.KVCache(k, v), batch, nk, nk)
        assert ctx.device_flags() == flag, what
        assert int((k != 0).sum()) == int((v != 0).sum()) == 8 * 2 * 64


def test_captured_and_replayed(gpu):
    """Append and both attentions in one graph, replayed as the sequences grow (the lengths and the
    new rows are read from device memory), every replay against the eager calls."""
    import torch
    log("graph of append, prompt and decode")
    hq, hkv, d, page = MODEL[0], MODEL[1], MODEL[2], 16
    s = Setup(hq, hkv, d, page, "f16", [300, 40], junk=0.0, seed=25)
    k, v = s.pools()
    cache, batch = gpu.KVCache(k, v), s.seqs(gpu)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    as_prompt = gpu.SeqBatch(batch.pages, batch.kv_len, start, n_rows=2)
    ctx, other = s.context(gpu), s.context(gpu)
    nk, nv = torch.randn((2, hkv, d), device="cuda"), torch.randn((2, hkv, d), device="cuda")
    q = s.q.cuda()
    o, p = torch.empty_like(q), torch.empty_like(q)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        with torch.cuda.graph(g, stream=st):
            ctx.kv_append(cache, batch, nk, nv)
            ctx.attn_decode(cache, batch, q, o=o)
            ctx.attn_prompt(cache, as_prompt, q, o=p)
    torch.cuda.synchronize()
    for step in range(5):
        batch.kv_len.copy_(torch.tensor([max(1, 250 + 11 * step), 1 + 9 * step], dtype=torch.int32))
        nk.normal_()
        nv.normal_()
        q.normal_()
        o.fill_(float("nan"))
        p.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, other.attn_decode(cache, batch, q)), step
        assert torch.equal(p, other.attn_prompt(cache, as_prompt, q)), step
        torch.cuda.synchronize()
    assert ctx.device_flags() == 0


def test_two_contexts_on_two_streams(gpu):
    """Two contexts at work at once do not share anything."""
    import torch
    log("two streams")
    s = Setup(*MODEL, 16, "bf16", [9000, 800], seed=26)
    t = Setup(*MODEL, 16, "bf16", [500, 7000], seed=27)
    got = []
    for x in (s, t):
        ctx = x.context(gpu)
        cache, batch, q = gpu.KVCache(*x.pools()), x.seqs(gpu), x.q.cuda()
        got.append((ctx, cache, batch, q, ctx.attn_decode(cache, batch, q)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i, (ctx, cache, batch, q, _) in enumerate(got):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ctx.attn_decode(cache, batch, q))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert torch.equal(o, got[i][4])


def test_no_sequences_and_no_rows(gpu):
    import torch
    log("empty calls")
    ctx = gpu.AttnContext(4, 2, 64, 16, 8)
    k = torch.zeros((2, 2, 16, 64), dtype=torch.float16, device="cuda")
    pages = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    q = torch.zeros((0, 4, 64), dtype=torch.float16, device="cuda")
    empty = gpu.SeqBatch(pages, none)
    assert ctx.attn_decode(gpu.KVCache(k, k.clone()), empty, q).shape == (0, 4, 64)
    ctx.kv_append(gpu.KVCache(k, k.clone()), empty, q[:, :2], q[:, :2])
    # a sequence without rows, and packed rows of no sequence
    two = gpu.SeqBatch(torch.zeros((1, 3), dtype=torch.int32, device="cuda"),
                       torch.ones(1, dtype=torch.int32, device="cuda"),
                       torch.zeros(2, dtype=torch.int32, device="cuda"), n_rows=5)
    o = torch.full((5, 4, 64), 3.0, dtype=torch.float16, device="cuda")
    ctx.attn_prompt(gpu.KVCache(k, k.clone()), two, o.clone(), o=o)
    assert (o == 3).all() and ctx.device_flags() == 0


def test_a_layer_of_decode_steps_with_the_experts(gpu):
    """A layer as it is used: a prompt in two pieces, then decode steps, each one append and attention,
    and the layer's MoE FFN on the result -- against the attention of the whole text at once."""
    import torch
    log("prompt, decode steps and the FFN")
    hq, hkv, d, page = 8, 2, 64, 16
    H = hq * d
    total, pieces, steps = 61, [30, 25], 6
    s = Setup(hq, hkv, d, page, "f16", [total], [total], seed=28, junk=float("nan"))
    want, bound, _, _ = s.reference()
    k, v = s.pools(filled=False)
    cache = gpu.KVCache(k, v)
    ctx = s.context(gpu)
    moe = gpu.Context(H, 256, 16, 1, 64, gpu.W_RENORM)
    moe.bind_packed(0, gpu.gen_layer(H, 256, 16, 99))
    K, V, Q = s.K[0].cuda(), s.V[0].cuda(), s.q.cuda()
    pages = s.pages.cuda()
    done, outs = 0, []
    for n in pieces:
        batch = gpu.SeqBatch(pages, torch.tensor([done + n], dtype=torch.int32, device="cuda"),
                             torch.tensor([0, n], dtype=torch.int32, device="cuda"), n_rows=n)
        ctx.kv_append(cache, batch, K[done:done + n], V[done:done + n])
        outs.append(ctx.attn_prompt(cache, batch, Q[done:done + n]))
        done += n
    length = torch.tensor([done], dtype=torch.int32, device="cuda")
    batch = gpu.SeqBatch(pages, length)
    for _ in range(steps):
        length += 1
        ctx.kv_append(cache, batch, K[done:done + 1].float(), V[done:done + 1].float())
        outs.append(ctx.attn_decode(cache, batch, Q[done:done + 1]))
        done += 1
    o = torch.cat(outs)
    check("o", o, want, bound)
    assert ctx.device_flags() == 0
    # the FFN of every row of the attention's output equals that of the whole output at once
    x = o.float().view(total, H)
    logits = gpu.gen_logits(total, 16, 7)
    whole, _, _ = moe.ffn_route(0, x, logits, rmsnorm=True)
    last, _, _ = moe.ffn_route(0, x[-1:].contiguous(), logits[-1:].contiguous(), rmsnorm=True)
    torch.cuda.synchronize()
    err = (whole[-1] - last[0]).abs().max() / whole[-1].abs().max()
    assert err <= 1e-3 + 5e-3  # the two paths' own bounds against the FFN's definition
    moe.close()


def test_refusals(gpu):
    """What a call refuses on the host, with a live handle: the C entry's statuses, then the binding's."""
    import ctypes
    import torch
    L = gpu.lib()
    ctx = gpu.AttnContext(4, 2, 64, 16, 4)
    k = torch.zeros((3, 2, 16, 64), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    pages = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda")
    o = torch.zeros_like(q)
    cache, batch, packed = gpu.KVCache(k, v), gpu.SeqBatch(pages, lens), gpu.SeqBatch(pages, lens, start, n_rows=2)
    st = torch.cuda.current_stream().cuda_stream

    def decode(kv=None, s=None, q_=q.data_ptr(), qs=256, scale=0.1, o_=o.data_ptr(), os=256, lse=None, fn=None):
        kv, s = cache._c if kv is None else kv, batch._c if s is None else s
        return (fn or L.moe_attn_decode)(ctx.handle, ctypes.addressof(kv), ctypes.addressof(s), q_, qs, scale, o_, os,
                                         lse, st)

    def changed(struct, **kw):
        c = type(struct)()
        ctypes.pointer(c)[0] = struct
        for n, val in kw.items():
            setattr(c, n, val)
        return c

    EINVAL = gpu.MOE_EINVAL
    assert decode() == gpu.MOE_OK
    assert decode(s=packed._c) == EINVAL  # row_start in a decode call
    assert decode(s=packed._c, fn=L.moe_attn_prompt) == gpu.MOE_OK
    for kw in (dict(q_=None), dict(o_=None), dict(qs=248), dict(os=255), dict(qs=260), dict(scale=float("nan")),
               dict(scale=float("inf")), dict(q_=q.data_ptr() + 8), dict(o_=o.data_ptr() + 2), dict(lse=o.data_ptr() + 2),
               dict(o_=q.data_ptr(), os=264)):
        assert decode(**kw) == EINVAL, kw
        assert L.moe_last_error()
    for kw in (dict(k=None), dict(v=None), dict(k=k.data_ptr() + 8), dict(n_pages=0), dict(page_stride=0),
               dict(head_stride=-64), dict(token_stride=32), dict(token_stride=68), dict(page_stride=1 << 50)):
        assert decode(kv=changed(cache._c, **kw)) == EINVAL, kw
    for kw in (dict(n_seqs=-1), dict(n_seqs=5), dict(n_rows=3), dict(n_rows=-1), dict(pages=None), dict(kv_len=None),
               dict(pages=pages.data_ptr() + 2), dict(max_pages=0), dict(pages_stride=2), dict(max_pages=1 << 30)):
        assert decode(s=changed(batch._c, **kw)) == EINVAL, kw
    assert decode(s=changed(packed._c, n_rows=(1 << 24) + 1), fn=L.moe_attn_prompt) == EINVAL
    new = torch.zeros((2, 2, 64), device="cuda")

    def append(t=gpu.T_F32, ks=128, vs=128, kp=new.data_ptr(), vp=new.data_ptr()):
        return L.moe_kv_append(ctx.handle, cache._ref, batch._ref, kp, vp, t, ks, vs, st)

    assert append() == gpu.MOE_OK
    assert append(t=gpu.T_BF16) == gpu.MOE_EUNSUPPORTED and append(t=5) == gpu.MOE_EUNSUPPORTED
    for kw in (dict(ks=124), dict(vs=130), dict(kp=None), dict(vp=None), dict(kp=new.data_ptr() + 4)):
        assert append(**kw) == EINVAL, kw
    assert L.moe_attn_flags(ctx.handle, st, None) == EINVAL
    assert L.moe_attn_flags_async(ctx.handle, lens.data_ptr() + 1, st) == EINVAL
    out = ctypes.c_void_p()
    assert L.moe_attn_create(99, ctypes.byref(gpu._AttnConfig(4, 2, 64, 16, 1, 4)), ctypes.byref(out)) == EINVAL
    # the binding
    cpu = torch.zeros((2, 4, 64), dtype=torch.float16)
    other = torch.zeros((3, 2, 32, 64), dtype=torch.float16, device="cuda")
    for bad in (lambda: ctx.attn_decode(cache, batch, cpu), lambda: ctx.attn_decode(cache, batch, q.bfloat16()),
                lambda: ctx.attn_decode(cache, batch, q[:1]), lambda: ctx.attn_decode(cache, batch, q[:, :3]),
                lambda: ctx.attn_decode(cache, batch, q, o=o.float()), lambda: ctx.attn_decode(cache, batch, q, o=o[:, :, :32]),
                lambda: ctx.attn_decode(cache, batch, q.transpose(1, 2).contiguous().transpose(1, 2)),
                lambda: ctx.attn_decode(cache, batch, q, lse=torch.zeros(2, 4)),
                lambda: ctx.attn_decode(cache, batch, q, lse=torch.zeros((2, 4), dtype=torch.float64, device="cuda")),
                lambda: ctx.attn_decode(gpu.KVCache(other, other), batch, q),
                lambda: ctx.attn_decode(gpu.KVCache(k.bfloat16(), v.bfloat16()), batch, q),
                lambda: ctx.attn_decode(gpu.KVCache(k.cpu(), v.cpu()), batch, q),
                lambda: ctx.attn_decode(cache, gpu.SeqBatch(pages.cpu(), lens.cpu()), q),
                lambda: ctx.kv_append(cache, batch, new, new.half()), lambda: ctx.kv_append(cache, batch, new.bfloat16(), new.bfloat16()),
                lambda: ctx.kv_append(cache, batch, new.cpu(), new.cpu()), lambda: ctx.kv_append(cache, batch, new[:1], new)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(gpu.MoeError):
        ctx.attn_decode(cache, packed, q)
    dst = torch.zeros(1, dtype=torch.int32, device="cuda")
    lens[0] = -1
    ctx.attn_decode(cache, batch, q)
    ctx.device_flags_async(dst)
    assert dst.item() == gpu.DEVFLAG_BAD_SEQ and ctx.device_flags() == 0
    ctx.close()
    with pytest.raises(ValueError):
        ctx.attn_decode(cache, batch, q)


@pytest.mark.parametrize("heads", [(200, 1, 64), (256, 1, 128), (36, 2, 256), (256, 256, 64)])
def test_decode_many_heads(gpu, heads):
    """Head blocks of 16, the last one short, and as many key-value heads as there may be."""
    log(f"decode heads {heads}")
    run_decode(gpu, Setup(*heads, 16, "f16", [200, 0, 33], seed=30))


def test_prompt_and_append_of_many_sequences(gpu):
    """More sequences than lanes, many without rows: rows, places and pages are found."""
    import torch
    log("prompt of 700 sequences")
    rows = [(7 * b) % 4 for b in range(700)]
    before = [(5 * b) % 23 for b in range(700)]
    s = Setup(2, 1, 64, 16, "bf16", [r + c for r, c in zip(rows, before)], rows, seed=31, extra_rows=2)
    run_decode(gpu, s)
    k, v = s.pools(filled=False)
    new_k = torch.cat([K[c:] for K, c in zip(s.K, before)] + [torch.full((2, 1, 64), 5.0, dtype=s.type)])
    new_v = torch.cat([V[c:] for V, c in zip(s.V, before)] + [torch.full((2, 1, 64), 5.0, dtype=s.type)])
    ctx = s.context(gpu)
    ctx.kv_append(gpu.KVCache(k, v), s.seqs(gpu), new_k.cuda(), new_v.cuda())
    k, v = k.cpu(), v.cpu()
    places = 0
    for b, (r, c) in enumerate(zip(rows, before)):
        for t in range(c, c + r):
            pg = int(s.pages[b, t // 16])
            assert torch.equal(k[pg, :, t % 16], s.K[b][t]) and torch.equal(v[pg, :, t % 16], s.V[b][t])
            places += 1
    assert int((~torch.isnan(k)).sum()) == int((~torch.isnan(v)).sum()) == places * 64
    assert ctx.device_flags() == 0


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_scores_that_keep_growing(gpu, type):
    """Each key's score is above the one before by 0.5: the running maximum is raised again and again."""
    import torch
    log(f"growing scores {type}")
    for rows in (None, [300]):
        s = Setup(4, 2, 64, 16, type, [300], rows, seed=32)
        s.q[:] = 1.0
        s.K[0][:] = (torch.arange(300).view(-1, 1, 1) * (0.5 * 8 / 64)).to(s.type)
        run_decode(gpu, s)


@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
def test_unseen_values_over_a_long_cache(gpu, bad):
    """Few rows over a cache that is cut into pieces: the last token's value reaches the last row only."""
    import torch
    log(f"{bad} at the end of a long cache")
    s = Setup(4, 2, 128, 16, "f16", [9003], [3], seed=33)
    want, bound, _, _ = s.reference()
    s.V[0][9002, :, 7] = bad
    o, _, flags = run_decode(gpu, s, ref=False)
    check("o", o[:2], want[:2], bound[:2])
    assert flags == 0
    assert torch.isnan(o[2, :, 7]).all() if math.isnan(bad) else (o[2, :, 7] == bad).all()
    o[2, :, 7] = 0
    want[2, :, 7] = 0
    check("o", o, want, bound)


def test_bad_page_beside_an_infinite_value(gpu):
    """A tile that all rows see whole, with a page outside the cache and an infinity in another page."""
    log("bad page and an infinity")
    s = Setup(4, 2, 64, 16, "f16", [200], [10], seed=34)
    s.V[0][5, :, 3] = float("inf")
    k, v = s.pools()
    ctx = s.context(gpu)
    batch = s.seqs(gpu)
    batch.pages[0, 2] = -7  # tokens 32..47 of the first tile
    o = ctx.attn_prompt(gpu.KVCache(k, v), batch, s.q.cuda())
    assert ctx.device_flags() == gpu.DEVFLAG_BAD_PAGE
    assert (o[:, :, 3] == math.inf).all()
    keep = list(range(32)) + list(range(48, 200))
    ref = Setup(4, 2, 64, 16, "f16", [184], [10], seed=34)
    ref.q, ref.K, ref.V = s.q, [s.K[0][keep]], [s.V[0][keep].clone()]
    ref.V[0][5, :, 3] = 0.0
    want, bound, _, _ = ref.reference()
    o[:, :, 3] = 0
    want[:, :, 3] = 0
    check("o", o, want, bound)


@pytest.mark.parametrize("rows", [None, [5, 60]])
def test_on_another_stream(gpu, rows):
    """stream= names another stream than the current one, as an object or a handle; the current stream
    is busy meanwhile."""
    import torch
    log(f"another stream, rows {rows}")
    s = Setup(*MODEL, 16, "bf16", [5000, 300], rows, seed=35)
    k, v = s.pools()
    ctx = s.context(gpu)
    call = ctx.attn_decode if rows is None else ctx.attn_prompt
    cache, batch, q = gpu.KVCache(k, v), s.seqs(gpu), s.q.cuda()
    good = call(cache, batch, q)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    busy = torch.randn(2048, 2048, device="cuda")
    for _ in range(5):
        for st in (other, other.cuda_stream):
            busy = busy @ busy * 1e-3
            o = call(cache, batch, q, stream=st)
            other.synchronize()
            assert torch.equal(o, good)
    torch.cuda.synchronize()


def test_scales_and_pools_out_of_range(gpu):
    import ctypes
    import torch
    log("scale and pool limits")
    ctx = gpu.AttnContext(4, 2, 64, 16, 4)
    k = torch.zeros((3, 2, 16, 64), dtype=torch.float16, device="cuda")
    batch = gpu.SeqBatch(torch.zeros((1, 1), dtype=torch.int32, device="cuda"),
                         torch.ones(1, dtype=torch.int32, device="cuda"))
    q = torch.zeros((1, 4, 64), dtype=torch.float16, device="cuda")
    cache = gpu.KVCache(k, k.clone())
    for scale in (3e38, -3e38, float("-inf")):
        with pytest.raises(gpu.MoeError):
            ctx.attn_decode(cache, batch, q, scale=scale)
    ctx.attn_decode(cache, batch, q, scale=1e37)
    cache._c.page_stride = 1 << 40
    cache._c.n_pages = 1 << 20
    with pytest.raises(gpu.MoeError):
        ctx.attn_decode(cache, batch, q)
    torch.cuda.synchronize()


@pytest.mark.parametrize("cut", [False, True])
def test_prompt_lengths_out_of_range(gpu, cut):
    """A length behind the page list is the list's end, also for the places of the rows; one below 0 is 0."""
    import torch
    log(f"prompt lengths out of range, {'a long cache' if cut else 'short'}")
    s = Setup(4, 2, 64, 16, "bf16", [9008 if cut else 96, 50], [33, 20], seed=36, pad_pages=0)
    k, v = s.pools()
    ctx = s.context(gpu)
    cache, batch, q = gpu.KVCache(k, v), s.seqs(gpu), s.q.cuda()
    good = ctx.attn_prompt(cache, batch, q)
    for n in (s.kv[0] + 1, s.kv[0] + 40, 2 ** 31 - 1):
        batch.kv_len[0] = n
        o = ctx.attn_prompt(cache, batch, q)
        assert ctx.device_flags() == gpu.DEVFLAG_BAD_SEQ
        assert torch.equal(o, good)
    batch.kv_len[0] = -2 ** 31
    o = ctx.attn_prompt(cache, batch, q)
    assert ctx.device_flags() == gpu.DEVFLAG_BAD_SEQ
    assert (o[:33] == 0).all()
    check("o", o[33:], *[x[33:] for x in s.reference()[:2]])


@pytest.mark.parametrize("heads", [(4, 2, 64), (4, 1, 128), (6, 2, 256)])
def test_decode_pieces_of_many_units(gpu, heads):
    """More units than workgroups, one sequence far longer than the rest: cut among many of them, and the
    ones in the middle cut in few."""
    log(f"decode pieces {heads}")
    kv = [1 + (11 * b) % 40 for b in range(600)]
    kv[311] = 30000
    kv[100] = 2500
    run_decode(gpu, Setup(*heads, 64, "f16", kv, seed=37))


def test_decode_pieces_of_some_units(gpu):
    """Fewer units than workgroups, with 512 to 2048 rows to join."""
    log("decode pieces of 64 units")
    run_decode(gpu, Setup(16, 1, 64, 32, "bf16", [700 + 3 * b for b in range(64)], seed=38))


@pytest.mark.parametrize("rows", [None, [4, 1, 2]])
def test_nothing_cached(gpu, rows):
    log(f"lengths of zero, rows {rows}")
    o, _, _ = run_decode(gpu, Setup(8, 2, 128, 16, "f16", [0, 0, 0], rows, seed=39))
    assert (o == 0).all()


@pytest.mark.parametrize("rows", [None, [7, 60], [1, 2]])
def test_a_query_that_is_not_finite(gpu, rows):
    """NaN and infinities in one row's query reach no other row."""
    import torch
    log(f"NaN queries, rows {rows}")
    s = Setup(8, 2, 64, 16, "f16", [5000, 80], rows, seed=40)
    want, bound, _, _ = s.reference()
    keep = [(r, h) for r in range(s.n_rows) for h in range(8) if (r, h) not in ((0, 3), (1, 0))]
    s.q[0, 3] = float("nan")
    s.q[1, 0, 5] = float("inf")
    o, _, _ = run_decode(gpu, s, ref=False)
    r, h = torch.tensor(keep).T
    check("o", o[r.cuda(), h.cuda()], want[r, h], bound[r, h])
    assert torch.isnan(o[0, 3]).all()


@pytest.mark.parametrize("rows", [None, [21, 30, 18]])
def test_shared_pages(gpu, rows):
    """Sequences that begin with the same pages, and one page twice in a list."""
    import torch
    log(f"shared pages, rows {rows}")
    s = Setup(8, 2, 64, 16, "bf16", [100, 90, 60], rows, seed=41)
    for b in (1, 2):  # the first 48 tokens
        s.pages[b, :3] = s.pages[0, :3]
        s.K[b][:48], s.V[b][:48] = s.K[0][:48], s.V[0][:48]
    s.pages[0, 4] = s.pages[0, 3]
    s.K[0][64:80], s.V[0][64:80] = s.K[0][48:64], s.V[0][48:64]
    run_decode(gpu, s)


def test_calls_in_a_row_share_the_workspace(gpu):
    """One context, no wait between calls of different shapes: each result is that of a call alone."""
    import torch
    log("calls in a row")
    sets = [Setup(4, 2, 128, 16, "f16", kv, rows, seed=42 + i) for i, (kv, rows) in enumerate([
        ([9000], None), ([9000], [5]), ([40] * 300, None), ([8000, 3], [2, 1]), ([2000, 60, 0, 7000], None)])]
    ctx = sets[0].context(gpu, max_seqs=300)
    calls = []
    for s in sets:
        call = ctx.attn_decode if s.rows is None else ctx.attn_prompt
        args = (gpu.KVCache(*s.pools()), s.seqs(gpu), s.q.cuda())
        calls.append((call, args, call(*args)))
        torch.cuda.synchronize()
    got = [(call(*args), good) for _ in range(4) for call, args, good in calls]
    for o, good in got:
        assert torch.equal(o, good)


def test_padded_batch_in_a_graph(gpu):
    """A captured step of a fixed number of sequences, some of them not in use (length 0, no page)."""
    import torch
    log("padded batch")
    full = Setup(*MODEL, 16, "f16", [700, 80, 33, 1, 500, 16], seed=43, junk=0.0)
    k, v = full.pools()
    cache, batch, q = gpu.KVCache(k, v), full.seqs(gpu), full.q.cuda()
    ctx, other = full.context(gpu), full.context(gpu)
    nk, nv = (torch.randn((6, 2, 256), device="cuda") for _ in range(2))
    o = torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st), torch.cuda.graph(g, stream=st):
        ctx.attn_decode(cache, batch, q, o=o)
    for used in (6, 3, 0, 5):
        kv = torch.tensor(full.kv, dtype=torch.int32)
        kv[used:] = 0
        batch.kv_len.copy_(kv)
        o.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        some = gpu.SeqBatch(batch.pages[:used], batch.kv_len[:used])
        assert (o[used:] == 0).all()
        if used:
            want, bound, _, _ = full.reference()
            check("o", o[:used], want[:used], bound[:used])
            check("alone", other.attn_decode(cache, some, q[:used]), want[:used], bound[:used])
        assert ctx.device_flags() == 0
    # the write leaves an unused sequence's row out and says so
    before = k.clone()
    batch.kv_len.zero_()
    ctx.kv_append(cache, batch, nk, nv)
    assert torch.equal(k, before) and ctx.device_flags() == gpu.DEVFLAG_BAD_SEQ


def test_most_sequences(gpu):
    """65535 sequences of a token or none; as prompts of as many rows and heads as cannot be launched."""
    import torch
    log("65535 sequences")
    n = 65535
    ctx = gpu.AttnContext(2, 1, 64, 16, n)
    v = torch.randn((50, 1, 16, 64), device="cuda").half()
    k = torch.randn_like(v)
    pages = (torch.arange(n, device="cuda", dtype=torch.int32) % 50).view(n, 1)
    kv_len = (torch.arange(n, device="cuda", dtype=torch.int32) % 3 > 0).int()
    q = torch.randn((n, 2, 64), device="cuda").half()
    want = (v[pages[:, 0].long(), :, 0] * kv_len.view(n, 1, 1)).expand(n, 2, 64)
    start = torch.arange(n + 1, device="cuda", dtype=torch.int32)
    cache = gpu.KVCache(k, v)
    assert torch.equal(ctx.attn_decode(cache, gpu.SeqBatch(pages, kv_len), q), want)
    assert torch.equal(ctx.attn_prompt(cache, gpu.SeqBatch(pages, kv_len, start, n), q), want)
    assert ctx.device_flags() == 0
    ctx = gpu.AttnContext(256, 256, 64, 16, n)
    k = torch.zeros((50, 256, 16, 64), dtype=torch.float16, device="cuda")
    q = torch.zeros((n, 256, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(gpu.MoeError):
        ctx.attn_prompt(gpu.KVCache(k, k.clone()), gpu.SeqBatch(pages, kv_len, start, n), q)
    torch.cuda.synchronize()


@pytest.mark.parametrize("heads", [(6, 3, 64), (10, 5, 128), (4, 1, 256)])
def test_cut_prompts_of_odd_heads_in_a_padded_batch(gpu, heads):
    """Few rows over long caches, among many sequences without rows; pieces that do not divide by 8."""
    import torch
    log(f"cut prompts {heads}")
    kv, rows = [0] * 40, [0] * 40
    for b, n, r in ((3, 7001, 37), (17, 30, 30), (18, 2600, 5), (39, 577, 1)):
        kv[b], rows[b] = n, r
    kv[20] = 4000  # cached tokens, no new row
    run_decode(gpu, Setup(*heads, 32, "f16", kv, rows, seed=50, extra_rows=4))


@pytest.mark.parametrize("n", [511, 512, 513, 576, 577])
def test_prompt_around_the_length_that_is_cut(gpu, n):
    log(f"prompt of 3 rows, {n} cached")
    run_decode(gpu, Setup(8, 2, 64, 16, "bf16", [n, 100], [3, 60], seed=51))


@pytest.mark.parametrize("heads", [(32, 8, 64), (16, 2, 256), (64, 16, 128)])
def test_prompts_of_many_weights(gpu, heads):
    """More tiles than are at work at once, of sequences of all lengths in no order, some with rows in front of
    the cache: each tile is worked on, once."""
    log(f"prompts of many weights {heads}")
    rows = [(193 * b + 71) % 260 for b in range(24)]
    before = [(389 * b) % 700 - 60 if b % 3 else 0 for b in range(24)]
    kv = [max(0, r + c) for r, c in zip(rows, before)]
    run_decode(gpu, Setup(*heads, 32, "bf16", kv, rows, seed=52, extra_rows=1))


@pytest.mark.parametrize("heads", [(4, 2, 64), (6, 1, 128), (16, 1, 256), (20, 1, 256)])
@pytest.mark.parametrize("kv", [[8192], [8193, 0], [8300, 17, 4000]])
def test_decode_around_64_steps(gpu, heads, kv):
    log(f"decode {heads} over {kv}")
    run_decode(gpu, Setup(*heads, 16, "bf16", kv, seed=53, pad_pages=0))


@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0])
@pytest.mark.parametrize("heads, rows", [((8, 2, 64), [3, 50]), ((16, 2, 256), [20, 1]), ((8, 2, 128), None)])
def test_scales_of_pieces(gpu, scale, heads, rows):
    log(f"scale {scale} of pieces, {heads} rows {rows}")
    run_decode(gpu, Setup(*heads, 16, "f16", [3500, 900], rows, seed=54), scale=scale)


@pytest.mark.parametrize("rows", [None, [30, 5]])
def test_tokens_far_apart(gpu, rows):
    """The largest token stride: a page's tokens 8 MiB apart (and 256 MiB from its first to its last)."""
    import torch
    log(f"token stride 2^22, rows {rows}")
    s = Setup(2, 1, 64, 32, "f16", [35, 5], rows, seed=55)
    small = s.pools()
    stride = 1 << 22
    buf = torch.empty(2, 32 * stride, dtype=torch.float16, device="cuda")
    far = [torch.as_strided(buf[i], (s.n_pages, 1, 32, 64), (64, 64 * s.n_pages, stride, 1)) for i in range(2)]
    for f, x in zip(far, small):
        f.copy_(x)
    far = [torch.as_strided(f, f.shape, (64, 64, stride, 1), f.storage_offset()) for f in far]
    want, bound, _, _ = s.reference()
    ctx = s.context(gpu)
    call = ctx.attn_decode if rows is None else ctx.attn_prompt
    check("o", call(gpu.KVCache(*far), s.seqs(gpu), s.q.cuda()), want, bound)
    assert ctx.device_flags() == 0


@pytest.mark.parametrize("n", [64, 65, 700, 4096, 4097, 9000])
def test_counts_of_many_sequences(gpu, n):
    """Of a token or none each, and as many rows: every sequence's rows are found (one token: o is its value)."""
    import torch
    log(f"{n} sequences")
    ctx = gpu.AttnContext(4, 2, 64, 16, n)
    v = torch.randn((50, 2, 16, 64), device="cuda").half()
    b = torch.arange(n, device="cuda", dtype=torch.int32)
    pages = (b * 7 % 50).view(n, 1)
    kv_len = ((b * 5 + b // 64) % 3 > 0).int()
    cache = gpu.KVCache(torch.randn_like(v), v)
    want = (v[pages[:, 0].long(), :, 0] * kv_len.view(n, 1, 1)).repeat_interleave(2, 1)
    q = torch.randn((n, 4, 64), device="cuda").half()
    assert torch.equal(ctx.attn_decode(cache, gpu.SeqBatch(pages, kv_len), q), want)
    start = torch.zeros(n + 1, device="cuda", dtype=torch.int32)
    start[1:] = kv_len.cumsum(0)
    rows = int(start[-1])
    o = ctx.attn_prompt(cache, gpu.SeqBatch(pages, kv_len, start, rows), q[:rows])
    assert torch.equal(o, want[kv_len.bool()])
    assert ctx.device_flags() == 0
