"""Serving over a paged KV cache: the operators next to paged decode, measured.

Three operators that run one after the other in a serving step:

* append: the new tokens' queries and keys are rotated by their positions and
  the keys and values are written into their pages of the cache;
* paged:  attention of several new tokens per sequence (a prompt, a chunk of
  one, or single tokens) over the sequence's pages;
* prefix: attention of one new token per sequence of a batch whose sequences
  share a long prefix, which is read once for all of them.

`run` computes them in elementary torch operations in 32 bits (`own` false) or
through this repository's library (`own` true).
"""

import math
import random
import sys

import numpy as np
import torch

own = False
_lib = None

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _library():
    global _lib
    if _lib is None:
        sys.path.insert(0, "cuflash-attn_b200")
        import cuflash_attn

        _lib = cuflash_attn.CuFlashAttn()
    return _lib


# ------------------------------------------------------------------- cases
def _append(name, dtype, batch, tokens, history, hq, hkv, d, page, rotary, interleaved, lens):
    return {"name": name, "op": "append", "dtype": dtype, "batch": batch, "tokens": tokens,
            "history": history, "hq": hq, "hkv": hkv, "d": d, "page": page, "rotary": rotary,
            "interleaved": interleaved, "lens": lens}


def _prefix(name, dtype, batch, prefix, suffix, hq, hkv, d, page, lens):
    return {"name": name, "op": "prefix", "dtype": dtype, "batch": batch, "prefix": prefix,
            "suffix": suffix, "hq": hq, "hkv": hkv, "d": d, "page": page, "lens": lens}


def _paged(name, dtype, batch, tokens, history, hq, hkv, d, page, causal, lens):
    return {"name": name, "op": "paged", "dtype": dtype, "batch": batch, "tokens": tokens,
            "history": history, "hq": hq, "hkv": hkv, "d": d, "page": page, "causal": causal,
            "lens": lens}


def listed():
    return [
        # one decode step of a small batch: a handful of rows, latency only
        _append("append_decode_b8", "bf16", 8, 1, 1500, 32, 8, 128, 16, 128, False, 1),
        # one decode step of a large batch, 16-bit floats, larger pages
        _append("append_decode_b256", "f16", 256, 1, 2500, 32, 4, 128, 64, 128, False, 2),
        # prompts of a prefill batch enter the cache (ragged, up to 8192 tokens)
        _append("append_prompts", "bf16", 5, 8192, 0, 32, 8, 128, 16, 128, False, 3),
        # odd chunk lengths, a narrow head, half of it rotated in neighbouring pairs
        _append("append_chunks_odd", "f16", 9, 131, 777, 14, 2, 64, 32, 32, True, 4),
        # a few requests behind a short system prompt: latency
        _prefix("prefix_b4_p512", "bf16", 4, 512, 60, 32, 8, 128, 16, 5),
        # the usual decode step of a served batch behind a common prompt
        _prefix("prefix_b32_p4096", "bf16", 32, 4096, 700, 32, 8, 128, 16, 6),
        # a large batch behind a long document
        _prefix("prefix_b128_p32768", "bf16", 128, 32768, 2000, 32, 8, 128, 64, 7),
        # odd batch, odd prefix, seven query heads on each key head, 16-bit floats
        _prefix("prefix_b19_p5003", "f16", 19, 5003, 301, 28, 4, 64, 32, 8),
        # the tail chunk of one prompt: few rows
        _paged("paged_tail_chunk", "bf16", 1, 33, 700, 32, 8, 128, 16, True, 9),
        # a mixed step: single tokens and prompt chunks of up to 256 tokens together
        _paged("paged_mixed_b16", "bf16", 16, 256, 3500, 32, 8, 128, 16, True, 10),
        # chunks of long prompts over long histories: the tensor cores' case
        _paged("paged_chunks_4096", "bf16", 2, 4096, 12288, 32, 8, 128, 64, True, 11),
        # equal head counts, narrow head, no causal mask (scoring of given passages)
        _paged("paged_full_mask", "f16", 7, 400, 900, 16, 16, 64, 32, False, 12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "prefix", "paged"])
    dtype = rng.choice(["bf16", "f16"])
    d = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    while hq > 32:
        hq = hkv * rng.choice([1, 2, 3, 4])
    lens = rng.randrange(1 << 30)
    if op == "append":
        if rng.random() < 0.5:
            return _append("", dtype, _log_int(rng, 1, 256), 1, _log_int(rng, 1, 2500), hq, hkv,
                           d, page, d, False, lens)
        rotary = rng.choice([d, d // 2, d // 4])
        return _append("", dtype, rng.randint(1, 9), _log_int(rng, 2, 4000),
                       _log_int(rng, 1, 2000), hq, hkv, d, page, rotary, rng.random() < 0.5, lens)
    if op == "prefix":
        return _prefix("", dtype, _log_int(rng, 2, 128), _log_int(rng, 64, 32768),
                       _log_int(rng, 1, 1500), hq, hkv, d, page, lens)
    if rng.random() < 0.5:
        return _paged("", dtype, _log_int(rng, 1, 24), _log_int(rng, 1, 400),
                      _log_int(rng, 1, 4000), hq, hkv, d, page, rng.random() < 0.7, lens)
    return _paged("", dtype, rng.randint(1, 2), _log_int(rng, 256, 4096), _log_int(rng, 1, 12288),
                  hq, hkv, d, page, True, lens)


def _lengths(case):
    """(new tokens, cache length behind them) of each sequence; lengths belong to
    the case, not to the seed. The first sequence has the full sizes; the others
    are spread from a single token (or none, behind a prefix) upwards."""
    r = random.Random(case["lens"])
    out = []
    for b in range(case["batch"]):
        if case["op"] == "prefix":
            n = case["suffix"] if b == 0 else r.randint(0, case["suffix"])
            out.append((1, n))
            continue
        new = case["tokens"] if b == 0 else r.randint(1, case["tokens"])
        if case["op"] == "paged" and case["batch"] >= 8 and b % 2:
            new = 1  # every other sequence of a mixed step decodes
        old = case["history"] if b == 0 else r.randint(0, case["history"])
        out.append((new, old + new))
    return out


# ----------------------------------------------------------------- inputs
def _table(gen, lens, page, first_pages=0):
    """Block table over shuffled pages, with pages left over in the pool; the
    entries behind a sequence's last page name no page."""
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + first_pages + 3
    order = torch.randperm(total, generator=gen).tolist()
    width = max(1, max(need))
    table = np.full((len(lens), width), -1, np.int32)
    at = first_pages
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, np.array(order[:first_pages], np.int32), total


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hkv, d, page, batch = (case[k] for k in ("hq", "hkv", "d", "page", "batch"))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    lens = _lengths(case)
    seq = [n for _, n in lens]
    first = (case["prefix"] + page - 1) // page if case["op"] == "prefix" else 0
    table, first_table, pages = _table(host, seq, page, first)
    st = {"case": case, "scale": 1.0 / math.sqrt(d), "new": [n for n, _ in lens], "seq": seq,
          "k_cache": normal(pages, page, hkv, d), "v_cache": normal(pages, page, hkv, d),
          "table": torch.from_numpy(table).cuda(),
          "seq_lens": torch.tensor(seq, dtype=torch.int32, device="cuda")}
    starts = np.concatenate([[0], np.cumsum(st["new"])]).astype(np.int32)
    st["cu"] = torch.from_numpy(starts).cuda()
    tokens = int(starts[-1])
    if case["op"] == "append":
        # one projection's output: queries, keys and values side by side
        qkv = normal(tokens, (hq + 2 * hkv) * d)
        st["q"] = qkv[:, :hq * d].view(tokens, hq, d)
        st["k"] = qkv[:, hq * d:(hq + hkv) * d].view(tokens, hkv, d)
        st["v"] = qkv[:, (hq + hkv) * d:].view(tokens, hkv, d)
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        angle = torch.arange(max(seq), dtype=torch.float64)[:, None] * freq
        st["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        st["q_out"] = torch.empty(tokens, hq, d, dtype=dt, device="cuda")
    elif case["op"] == "prefix":
        st["q"] = normal(batch, hq, 1, d)
        st["first_table"] = torch.from_numpy(first_table).cuda()
        st["first_len"] = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda")
    else:
        st["q"] = normal(tokens, hq, d)
    return st


# ------------------------------------------------------------- plain forms
def _rows(table, n, page):
    """Cache row of each of a sequence's n tokens."""
    t = torch.arange(n, device=table.device)
    return table[t // page].long() * page + t % page


def _rotate(x, rope, pos, interleaved):
    half = rope.shape[1] // 2
    cos, sin = rope[pos, :half][:, None], rope[pos, half:][:, None]
    x = x.float()
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2] = a * cos - b * sin
        y[..., 1:2 * half:2] = b * cos + a * sin
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half] = a * cos - b * sin
        y[..., half:2 * half] = b * cos + a * sin
    return y


def _plain_append(st):
    page, il = st["case"]["page"], st["case"]["interleaved"]
    kc = st["k_cache"].view(-1, *st["k_cache"].shape[2:])
    vc = st["v_cache"].view(-1, *st["v_cache"].shape[2:])
    token = torch.arange(st["q"].shape[0], device="cuda")
    seq = torch.searchsorted(st["cu"].long(), token, right=True) - 1
    pos = token - st["cu"][seq + 1] + st["seq_lens"][seq]
    rows = st["table"][seq, pos // page].long() * page + pos % page
    st["q_out"].copy_(_rotate(st["q"], st["rope"], pos, il).to(st["q_out"].dtype))
    kc[rows] = _rotate(st["k"], st["rope"], pos, il).to(kc.dtype)
    vc[rows] = st["v"]
    return st["q_out"], st["k_cache"], st["v_cache"]


def _plain_attention(q, k, v, scale, hidden):
    """q [hkv, rows, d], k and v [hkv, n, d] in 32 bits; hidden [rows, n] or None.
    The unnormalised output, the row maximum and the row sum."""
    s = torch.matmul(q, k.transpose(1, 2)) * scale
    if hidden is not None:
        s.masked_fill_(hidden, -math.inf)
    m = s.amax(2, keepdim=True)
    p = torch.exp(s - m)
    return torch.matmul(p, v), m, p.sum(2, keepdim=True)


def _plain_paged(st):
    case, page = st["case"], st["case"]["page"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g = hq // hkv
    kc = st["k_cache"].view(-1, hkv, d)
    vc = st["v_cache"].view(-1, hkv, d)
    out = torch.empty_like(st["q"])
    lse = torch.empty(st["q"].shape[:2], device="cuda")
    at = 0
    for b, (new, n) in enumerate(zip(st["new"], st["seq"])):
        rows = _rows(st["table"][b], n, page)
        k, v = kc[rows].float().transpose(0, 1), vc[rows].float().transpose(0, 1)
        for lo in range(0, new, 512):  # a block of queries at a time
            hi = min(new, lo + 512)
            q = st["q"][at + lo:at + hi].float().view(hi - lo, hkv, g, d)
            q = q.transpose(0, 1).reshape(hkv, (hi - lo) * g, d)
            hidden = None
            if case["causal"]:
                last = torch.arange(n - new + lo, n - new + hi, device="cuda")
                hidden = torch.arange(n, device="cuda") > last.repeat_interleave(g)[:, None]
            o, m, l = _plain_attention(q, k, v, st["scale"], hidden)
            o = (o / l).view(hkv, hi - lo, g, d).transpose(0, 1).reshape(hi - lo, hq, d)
            out[at + lo:at + hi] = o.to(out.dtype)
            ls = (m + l.log()).view(hkv, hi - lo, g).transpose(0, 1).reshape(hi - lo, hq)
            lse[at + lo:at + hi] = ls
        at += new
    return out, lse


def _plain_prefix(st):
    case, page = st["case"], st["case"]["page"]
    hq, hkv, d, batch = case["hq"], case["hkv"], case["d"], case["batch"]
    g = hq // hkv
    kc = st["k_cache"].view(-1, hkv, d)
    vc = st["v_cache"].view(-1, hkv, d)
    q = st["q"].float().view(batch, hkv, g, d)
    # the shared prefix, for all sequences' queries at once
    rows = _rows(st["first_table"], case["prefix"], page)
    k, v = kc[rows].float().transpose(0, 1), vc[rows].float().transpose(0, 1)
    o0, m0, l0 = _plain_attention(q.transpose(0, 1).reshape(hkv, batch * g, d), k, v,
                                  st["scale"], None)
    o0 = o0.view(hkv, batch, g, d).transpose(0, 1)
    m0 = m0.view(hkv, batch, g, 1).transpose(0, 1)
    l0 = l0.view(hkv, batch, g, 1).transpose(0, 1)
    # each sequence's own tokens, padded to the longest
    n = max(max(st["seq"]), 1)
    t = torch.arange(n, device="cuda")
    rows = (st["table"][:, t // page].clamp(min=0).long() * page + t % page)
    k, v = kc[rows].float().permute(0, 2, 1, 3), vc[rows].float().permute(0, 2, 1, 3)
    s = torch.matmul(q, k.transpose(2, 3)) * st["scale"]
    s.masked_fill_((t >= st["seq_lens"][:, None])[:, None, None], -math.inf)
    m = torch.maximum(s.amax(3, keepdim=True), m0)
    p = torch.exp(s - m)
    w = torch.exp(m0 - m)
    l = p.sum(3, keepdim=True) + w * l0
    o = (torch.matmul(p, v) + w * o0) / l
    return (o.reshape(batch, hq, 1, d).to(st["q"].dtype), (m + l.log()).reshape(batch, hq))


def run(state):
    st, case = state, state["case"]
    if not own:
        return {"append": _plain_append, "prefix": _plain_prefix,
                "paged": _plain_paged}[case["op"]](st)
    lib = _library()
    if case["op"] == "append":
        lib.kv_append_paged(st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"],
                            st["seq_lens"], cu_seqlens=None if case["tokens"] == 1 else st["cu"],
                            Q=st["q"], rope_table=st["rope"], interleaved=case["interleaved"],
                            Q_out=st["q_out"])
        return st["q_out"], st["k_cache"], st["v_cache"]
    if case["op"] == "prefix":
        return lib.decode_shared_prefix(st["q"], st["k_cache"], st["v_cache"], st["first_table"],
                                        st["first_len"], st["table"], st["seq_lens"],
                                        scale=st["scale"])
    return lib.forward_paged(st["q"], st["k_cache"], st["v_cache"], st["table"], st["seq_lens"],
                             st["cu"], causal=case["causal"], scale=st["scale"])


# ------------------------------------------------------------ definitions
def exact(case, seed):
    """The definition, one sequence and one key head at a time, in 64 bits: the
    whole row of scores is formed (prefix and own tokens together) and its
    exponentials are divided by their sum."""
    st = prepare(case, seed)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    g = hq // hkv
    lens = _lengths(case)
    if case["op"] == "append":
        half = case["rotary"] // 2
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        q, k = st["q"].double(), st["k"].double()
        rope = st["rope"].double()
        turn = torch.complex(rope[:, :half], rope[:, half:])
        at = 0
        for b, (new, n) in enumerate(lens):
            w = turn[n - new:n][:, None]
            for x in (q, k):
                part = x[at:at + new, :, :2 * half]
                if case["interleaved"]:
                    z = torch.view_as_complex(part.reshape(new, -1, half, 2).contiguous()) * w
                    x[at:at + new, :, :2 * half] = torch.view_as_real(z).flatten(2)
                else:
                    z = torch.complex(part[..., :half].contiguous(),
                                      part[..., half:].contiguous()) * w
                    x[at:at + new, :, :2 * half] = torch.cat([z.real, z.imag], 2)
            pos = torch.arange(n - new, n, device="cuda")
            pages = st["table"][b].long()[torch.div(pos, page, rounding_mode="floor")]
            kc[pages, pos % page] = k[at:at + new]
            vc[pages, pos % page] = st["v"][at:at + new].double()
            at += new
        return q, kc, vc
    prefix = case["op"] == "prefix"
    q = st["q"].double().view(-1, hq, d)
    out = torch.zeros_like(q)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for b, (new, n) in enumerate(lens):
        own_pages = st["table"][b].long()[:(n + page - 1) // page]
        for h in range(hkv):
            k = st["k_cache"][own_pages, :, h].reshape(-1, d)[:n].double()
            v = st["v_cache"][own_pages, :, h].reshape(-1, d)[:n].double()
            if prefix:
                fp = st["first_table"].long()
                k = torch.cat([st["k_cache"][fp, :, h].reshape(-1, d)[:case["prefix"]].double(), k])
                v = torch.cat([st["v_cache"][fp, :, h].reshape(-1, d)[:case["prefix"]].double(), v])
            for lo in range(0, new, 256):
                hi = min(new, lo + 256)
                qq = q[at + lo:at + hi, h * g:(h + 1) * g].reshape(-1, d)
                s = (qq @ k.T) / math.sqrt(d)
                if not prefix and case["causal"]:
                    sees = torch.arange(lo, hi, device="cuda") + (n - new)
                    key = torch.arange(n, device="cuda")
                    s = torch.where(key[None] <= sees.repeat_interleave(g)[:, None], s, -math.inf)
                ls = torch.logsumexp(s, 1)
                o = torch.exp(s - ls[:, None]) @ v
                out[at + lo:at + hi, h * g:(h + 1) * g] = o.view(hi - lo, g, d)
                lse[at + lo:at + hi, h * g:(h + 1) * g] = ls.view(hi - lo, g)
        at += new
    return out.view(st["q"].shape), lse


def work(case):
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    lens = _lengths(case)
    tokens = sum(n for n, _ in lens)
    row = hkv * d * 2 * 2  # keys and values of one token, 16 bits
    if case["op"] == "append":
        # each token's q, k, v in; its rotated q and its cache rows out; angles, page, length
        each = 2 * (hq * d * 2 + row) + case["rotary"] * 4 + 4
        return {"bytes": tokens * each + 8 * case["batch"],
                "flops": tokens * (hq + hkv) * case["rotary"] * 3}
    io = tokens * hq * (2 * d * 2 + 4)
    if case["op"] == "prefix":
        keys = case["prefix"] + sum(n for _, n in lens)
        pairs = case["batch"] * case["prefix"] + sum(n for _, n in lens)
    else:
        keys = sum(n for _, n in lens)
        pairs = 0
        for new, n in lens:
            pairs += new * n - (new * (new - 1) // 2 if case["causal"] else 0)
    return {"bytes": io + keys * row + 4 * (keys // page + 2 * case["batch"]),
            "flops": 4 * pairs * hq * d}
