"""Measured cases of the attention operators: writing new keys and values into a paged cache
(`kv_append`), one new token of every sequence over its cache (`attn_decode`), and packed causal
prompts over the cache (`attn_prompt`), through `AttnContext` (moe-680m_amd/__init__.py).

A case is a dict of plain values:
  kind    "append", "decode" or "prompt"
  type    element type of the cache, of q and of o: "f16" or "bf16"
  src     append: element type of the new rows ("" otherwise)
  hq, hkv query and key-value heads;  d  head size;  page  tokens of a page
  seqs    sequences of the call
  kv_lo, kv_hi      tokens already cached (decode: with the new one) of a sequence
  rows_lo, rows_hi  new rows of a sequence (decode: 1)
  mix     picks the sequences' lengths in those ranges (the first has the largest of both)

The lengths follow from the case alone; the values and the pages' places come from the seed.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _package():
    """The package directory moe-680m_amd/ (not an importable name) as moe680m_amd."""
    if "moe680m_amd" in sys.modules:
        return sys.modules["moe680m_amd"]
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe-680m_amd")
    spec = importlib.util.spec_from_file_location("moe680m_amd", os.path.join(here, "__init__.py"),
                                                  submodule_search_locations=[here])
    mod = importlib.util.module_from_spec(spec)
    sys.modules["moe680m_amd"] = mod
    spec.loader.exec_module(mod)
    return mod


# ---------------------------------------------------------------- the cases
def _case(name, kind, type, heads, page, seqs, kv, rows=(1, 1), src="", mix=1):
    c = {"kind": kind, "type": type, "src": src, "hq": heads[0], "hkv": heads[1], "d": heads[2], "page": page,
         "seqs": seqs, "kv_lo": kv[0], "kv_hi": kv[1], "rows_lo": rows[0], "rows_hi": rows[1], "mix": mix}
    return dict(name=name, **c) if name else c


MODEL = (16, 2, 256)  # the attention layers of the model whose MoE layers the library runs


def listed():
    return [
        # a decode step of a serving batch: 64 sequences' new keys and values, f32 from the projections
        _case("append_step64_f32", "append", "f16", MODEL, 16, 64, (0, 4000), (1, 1), src="f32"),
        # the keys and values of eight packed prompts of very different lengths
        _case("append_prompts_bf16", "append", "bf16", MODEL, 64, 8, (0, 0), (37, 4096), src="bf16"),
        # one sequence with a short context: the smallest decode call, all latency
        _case("decode_1x512", "decode", "f16", MODEL, 16, 1, (512, 512)),
        # one sequence over a long cache: only the split over its length fills the card
        _case("decode_1x131072", "decode", "bf16", MODEL, 64, 1, (131072, 131072)),
        # a serving batch of ragged contexts
        _case("decode_64_ragged", "decode", "f16", MODEL, 16, 64, (200, 16384)),
        # a large batch of short contexts, more key-value heads
        _case("decode_256_gqa4", "decode", "bf16", (32, 8, 128), 16, 256, (1, 2048)),
        # an odd batch of small contexts, one key-value head to a query head
        _case("decode_17_mha64", "decode", "f16", (12, 12, 64), 32, 17, (1, 777)),
        # short prompts of several requests, packed (odd lengths)
        _case("prompt_16_short", "prompt", "f16", MODEL, 16, 16, (0, 0), (9, 101)),
        # the prompts of a batch, of very different lengths
        _case("prompt_8_ragged", "prompt", "f16", (32, 8, 128), 16, 8, (0, 0), (100, 2001)),
        # one prompt of the model's heads
        _case("prompt_4096", "prompt", "bf16", MODEL, 64, 1, (0, 0), (4096, 4096)),
        # a piece of a long prompt over what is cached already: few rows, a long cache
        _case("prompt_64_over_32k", "prompt", "bf16", MODEL, 64, 1, (32704, 32704), (64, 64)),
        # one long prompt: the largest call
        _case("prompt_8192_gqa4", "prompt", "bf16", (32, 8, 128), 64, 1, (0, 0), (8192, 8192)),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1))))))))


def draw(rng):
    heads = rng.choice([MODEL, MODEL, (32, 8, 128), (12, 12, 64), (8, 1, 128), (24, 2, 64), (20, 4, 128), (6, 2, 256)])
    type, page, mix = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128]), rng.randrange(1 << 20)
    hq, hkv, d = heads
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    if kind == "append":
        seqs = _log(rng, 1, 128)
        rows = _log(rng, 1, min(4096, 3_400_000 // (hkv * d * seqs)))
        return _case("", kind, type, heads, page, seqs, (0, _log(rng, 1, 2000)), (_log(rng, 1, rows), rows),
                     src=rng.choice([type, "f32"]), mix=mix)
    if kind == "decode":
        seqs = _log(rng, 1, 256)
        kv = _log(rng, 1, min(131072, 120_000_000 // (hkv * d * seqs)))
        return _case("", kind, type, heads, page, seqs, (_log(rng, 1, kv), kv), mix=mix)
    seqs = _log(rng, 1, 16)
    most = 1.2e11 / (hq * d * seqs)
    rows = _log(rng, 1, int(math.sqrt(most)))
    before = rng.choice([0, 0, _log(rng, 1, int(min(32768, most / (2 * rows))))])
    return _case("", kind, type, heads, page, seqs, (0, before), (_log(rng, 1, rows), rows), mix=mix)


def _lengths(case):
    """(new rows, cached tokens with the new ones) of every sequence."""
    rng = random.Random(case["mix"])
    rows, kv = [case["rows_hi"]], [case["kv_hi"]]
    for _ in range(case["seqs"] - 1):
        rows.append(_log(rng, case["rows_lo"], case["rows_hi"]))
        kv.append(_log(rng, case["kv_lo"], case["kv_hi"]))
    return rows, kv if case["kind"] == "decode" else [r + c for r, c in zip(rows, kv)]


def work(case):
    rows, kv = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    index = 4 * sum(-(-n // case["page"]) + 2 for n in kv)
    if case["kind"] == "append":
        return {"bytes": sum(rows) * hkv * d * 2 * (2 + (4 if case["src"] == "f32" else 2)) + index, "flops": 0}
    seen = sum(r * (n - r) + r * (r + 1) // 2 for r, n in zip(rows, kv))
    return {"bytes": sum(kv) * hkv * d * 2 * 2 + sum(rows) * hq * d * 2 * 2 + index, "flops": 4 * hq * d * seen}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    rows, kv = _lengths(case)
    type, page, seqs = TYPES[case["type"]], case["page"], case["seqs"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    need = [-(-n // page) for n in kv]
    wide, pool = max(need), sum(need) + 3
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    start = torch.tensor([sum(need[:b]) for b in range(seqs)], device=dev).view(-1, 1)
    col = torch.arange(wide, device=dev).view(1, -1)
    pages = order[(start + col).clamp(max=pool - 1)]  # behind a sequence's last page: any page, not read
    n = sum(rows)
    state = {"case": case, "pages": pages.contiguous(), "kv_len": torch.tensor(kv, dtype=torch.int32, device=dev),
             "rows": n, "wide": max(kv), "tall": max(rows), "start": None}
    state["k"] = torch.randn((pool, hkv, page, d), generator=g, device=dev).to(type)
    state["v"] = torch.randn((pool, hkv, page, d), generator=g, device=dev).to(type)
    if case["kind"] != "decode":
        cum = [sum(rows[:b]) for b in range(seqs + 1)]
        state["start"] = torch.tensor(cum, dtype=torch.int32, device=dev)
    if case["kind"] == "append":
        # one fused projection's rows: q | k | v
        qkv = torch.randn((n, hq + 2 * hkv, d), generator=g, device=dev).to(TYPES[case["src"]])
        state["k_new"], state["v_new"] = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    else:
        # scores of standard deviation 1.5: some keys stand out
        state["q"] = (1.5 * torch.randn((n, hq, d), generator=g, device=dev)).to(type)
    if own:
        P = _package()
        state["attn"] = P.AttnContext(hq, hkv, d, page, max_seqs=seqs, dtype=type)
        state["cache"] = P.KVCache(state["k"], state["v"])
        state["batch"] = P.SeqBatch(state["pages"], state["kv_len"], state["start"], n_rows=n)
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        a, cache, batch = state["attn"], state["cache"], state["batch"]
        if kind == "append":
            a.kv_append(cache, batch, state["k_new"], state["v_new"])
            return {"k": state["k"], "v": state["v"]}
        if kind == "decode":
            return {"o": a.attn_decode(cache, batch, state["q"])}
        return {"o": a.attn_prompt(cache, batch, state["q"])}
    if kind == "append":
        return _plain_append(state)
    return {"o": _plain_decode(state) if kind == "decode" else _plain_prompt(state)}


def _row_sequence(state):
    """(sequence, index in it) of every packed row."""
    start = state["start"].long()
    row = torch.arange(state["rows"], device=start.device)
    seq = (row.view(-1, 1) >= start[1:].view(1, -1)).sum(1)
    return seq, row - start[seq]


def _plain_append(state):
    page = state["case"]["page"]
    seq, i = _row_sequence(state)
    start, length = state["start"].long(), state["kv_len"].long()
    pos = length[seq] - (start[seq + 1] - start[seq]) + i
    at = state["pages"][seq, pos // page].long()
    state["k"][at, :, pos % page] = state["k_new"].to(state["k"].dtype)
    state["v"][at, :, pos % page] = state["v_new"].to(state["v"].dtype)
    return {"k": state["k"], "v": state["v"]}


def _gather(state, pool):
    """The cached rows of every sequence, [seqs][heads][tokens][d] in 32 bits."""
    t = pool[state["pages"].long()].float().transpose(1, 2)
    return t.reshape(t.shape[0], t.shape[1], -1, t.shape[-1])[:, :, :state["wide"]].contiguous()


def _softmax_product(s, seen, v):
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (s - m).exp()
    o = torch.matmul(p, v)
    return o / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _plain_decode(state):
    c = state["case"]
    b, hq, hkv, d = c["seqs"], c["hq"], c["hkv"], c["d"]
    k, v = _gather(state, state["k"]), _gather(state, state["v"])
    q = state["q"].float().view(b, hkv, hq // hkv, d)
    s = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d)
    seen = torch.arange(state["wide"], device=s.device).view(1, 1, 1, -1) < state["kv_len"].view(-1, 1, 1, 1)
    return _softmax_product(s, seen, v).reshape(b, hq, d).to(state["q"].dtype)


def _plain_prompt(state):
    c = state["case"]
    b, hq, hkv, d, tall = c["seqs"], c["hq"], c["hkv"], c["d"], state["tall"]
    k, v = _gather(state, state["k"]), _gather(state, state["v"])
    seq, i = _row_sequence(state)
    q = torch.zeros((b, tall, hq, d), device=k.device)
    q[seq, i] = state["q"].float()
    q = q.view(b, tall, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    s = (torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d)).view(b, hkv, hq // hkv, tall, -1)
    start, length = state["start"].long(), state["kv_len"].long()
    pos = (length - (start[1:] - start[:-1])).view(-1, 1) + torch.arange(tall, device=k.device).view(1, -1)
    pos = torch.minimum(pos, length.view(-1, 1) - 1)
    seen = torch.arange(state["wide"], device=k.device).view(1, 1, -1) <= pos.unsqueeze(-1)
    o = _softmax_product(s, seen.view(b, 1, 1, tall, -1), v.unsqueeze(2))
    o = o.permute(0, 3, 1, 2, 4).reshape(b, tall, hq, d)
    return o[seq, i].to(state["q"].dtype)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """Sequence by sequence and head by head, in 64 bits."""
    s = prepare(dict(case), seed)
    page, d, group = case["page"], case["d"], case["hq"] // case["hkv"]
    rows, kv = _lengths(case)
    first = 0
    if case["kind"] == "append":
        k, v = s["k"].double(), s["v"].double()
        for b, (r, n) in enumerate(zip(rows, kv)):
            for name, pool in (("k_new", k), ("v_new", v)):
                new = s[name][first:first + r].to(pool.device).to(s["k"].dtype).double()
                where = torch.arange(n - r, n, device=pool.device)
                pool[s["pages"][b].long()[where // page], :, where % page] = new
            first += r
        return {"k": k, "v": v}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (r, n) in enumerate(zip(rows, kv)):
        used = s["pages"][b, :-(-n // page)].long()
        for h in range(case["hkv"]):
            k = s["k"][used, h].reshape(-1, d)[:n].double()
            v = s["v"][used, h].reshape(-1, d)[:n].double()
            q = s["q"][first:first + r, h * group:(h + 1) * group].double()
            z = (q.reshape(-1, d) @ k.t().contiguous()).view(r, group, n) * d ** -0.5
            ahead = torch.arange(n, device="cuda").view(1, 1, -1) > torch.arange(n - r, n, device="cuda").view(-1, 1, 1)
            w = torch.softmax(z.masked_fill(ahead, -math.inf), -1)
            out[first:first + r, h * group:(h + 1) * group] = (w.view(-1, n) @ v).view(r, group, d)
        first += r
    return {"o": out}
