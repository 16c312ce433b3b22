"""Workloads of the paged 8-bit key/value cache and of draft verification.

Each case is one pass through an operator: ``run`` computes it with elementary
torch operations where ``own`` is false and through the public entry points of
this repository's package where it is true.

The cache (one layer, or several for the page copies) holds

  k        int8    [layers, pages, heads, P, hd]
  v        int8    [layers, pages, heads, P / 16, hd, 16]   (16 tokens innermost)
  k_scale  float32 [layers, pages, heads]                   (v_scale likewise)

and a value is code * scale.  ``table[b, j]`` is the page of tokens j*P .. j*P +
P - 1 of sequence b, ``kv_len[b]`` its length with this call's tokens, and row
(b, i) of a call is token kv_len[b] - n_new[b] + i, for i < n_new[b].  Page 0
is in no table.
"""
import importlib
import math

import torch

own = False

PACKAGE = "glassboxai-transformer_b200"
VOCAB = 50257


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of each of 32 conversations, GPT-2 small heads: write the token, read its block back
        dict(name="append decode", op="append", B=32, S=1, heads=12, hd=64, P=16, kv=700, ragged=True),
        # drafted tokens of a serving batch, 0 to 5 of them a sequence
        dict(name="append drafts", op="append", B=96, S=5, heads=25, hd=64, P=32, kv=900, ragged=True),
        # whole prompts of 1024 tokens, GPT-2 XL heads
        dict(name="append prompts", op="append", B=8, S=1024, heads=25, hd=64, P=64, kv=1024, ragged=False),
        # one conversation, one new token, GPT-2 small: latency
        dict(name="decode one", op="attn", B=1, S=1, H=12, heads=12, hd=64, P=16, kv=1023, ragged=False),
        # the decode workload of the benchmark: GPT-2 XL, 256 sequences at position 2047
        dict(name="decode XL batch", op="attn", B=256, S=1, H=25, heads=25, hd=64, P=64, kv=2048, ragged=False),
        # scoring up to 5 drafted tokens of sequences of mixed lengths, GPT-2 medium
        dict(name="drafts mixed", op="attn", B=32, S=5, H=16, heads=16, hd=64, P=16, kv=1021, ragged=True),
        # one new token over long documents, 4 query heads to a key head
        dict(name="decode long", op="attn", B=2, S=1, H=32, heads=8, hd=128, P=128, kv=120001, ragged=False),
        # the next 512 tokens of a prompt over what is cached
        dict(name="prompt chunk", op="attn", B=2, S=512, H=16, heads=16, hd=64, P=64, kv=2048, ragged=False),
        # the last, partly filled pages of 16 forked sequences
        dict(name="copy fork", op="copy", n=16, layers=12, heads=12, hd=64, P=16),
        # a compaction that moves 600 pages of GPT-2 medium
        dict(name="copy compact", op="copy", n=600, layers=24, heads=16, hd=64, P=32),
        # one sequence's 4 drafted tokens: latency
        dict(name="verify one", op="verify", B=1, n=4, vocab=VOCAB, T=0.8, drafts=True, ragged=False),
        # a serving batch with up to 7 drafted tokens
        dict(name="verify batch", op="verify", B=64, n=7, vocab=VOCAB, T=1.0, drafts=True, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("append", "append", "attn", "attn", "attn", "copy", "verify", "verify"))
    P = rng.choice((16, 32, 64, 128))
    hd = rng.choice((64, 64, 64, 32, 80, 96, 128))
    if op == "append":
        heads = rng.randint(1, 32)
        S = _log(rng, 1, 1024)
        B = _log(rng, 1, max(1, min(256, 8_000_000 // (S * heads * hd))))
        return dict(op=op, B=B, S=S, heads=heads, hd=hd, P=P, kv=S + _log(rng, 1, 1500), ragged=rng.random() < 0.6)
    if op == "attn":
        heads = rng.randint(1, 25)
        G = rng.choice((1, 1, 1, 2, 4, 5, 8))
        S = rng.choice((1, 1, 1, rng.randint(2, 9), _log(rng, 10, 300)))
        kv = S + _log(rng, 1, 60000 if S < 10 else 4000)
        B = _log(rng, 1, max(1, min(256, 300_000_000 // (kv * heads * hd), 1_000_000_000 // (kv * heads * G * S))))
        return dict(op=op, B=B, S=S, H=heads * G, heads=heads, hd=hd, P=P, kv=kv, ragged=rng.random() < 0.6)
    if op == "copy":
        layers, heads = rng.randint(1, 24), rng.randint(1, 25)
        return dict(op=op, n=_log(rng, 1, max(1, min(1000, 200_000_000 // (layers * heads * P * hd)))), layers=layers, heads=heads,
                    hd=hd, P=P)
    n = rng.randint(1, 8)
    vocab = rng.choice((VOCAB, _log(rng, 1000, 60000)))
    return dict(op=op, B=_log(rng, 1, 64), n=n, vocab=vocab, T=rng.choice((0.0, 0.6, 0.8, 1.0, 1.3)), drafts=rng.random() < 0.7,
                ragged=rng.random() < 0.5)


# ------------------------------------------------------------------- inputs
def _pages_of(kv, P):
    return -(-kv // P)


def _lengths(case, g):
    """kv_len and n_new of each sequence (int32): all full, or mixed."""
    B, S, kv = case["B"], case["S"], case["kv"]
    if not case["ragged"]:
        full = torch.full((B,), kv, dtype=torch.int32, device="cuda")
        return full, torch.full((B,), S, dtype=torch.int32, device="cuda")
    n_new = torch.randint(0, S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n_new[0] = S
    before = torch.randint(0, kv - S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    before[0] = kv - S
    return before + n_new, n_new


def _codes(shape, g):
    return (torch.randn(shape, generator=g, device="cuda") * 40.0).round().clamp(-127, 127).to(torch.int8)


def _pool(layers, pages, heads, P, hd, g):
    s = {"k": torch.empty((layers, pages, heads, P, hd), dtype=torch.int8, device="cuda"),
         "v": torch.empty((layers, pages, heads, P // 16, hd, 16), dtype=torch.int8, device="cuda")}
    for t in s.values():
        flat = t.view(-1)
        for a in range(0, flat.numel(), 1 << 28):
            part = flat[a:a + (1 << 28)]
            part.copy_(_codes(part.shape, g))
    # a token's keys and values are about N(0, 1): the largest of a page over 40 is about 1 / 40
    for name in ("k_scale", "v_scale"):
        s[name] = (0.6 + 0.8 * torch.rand((layers, pages, heads), generator=g, device="cuda")) / 40.0
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = dict(case)
    if op in ("append", "attn"):
        B, S, heads, hd, P = (case[k] for k in ("B", "S", "heads", "hd", "P"))
        m = _pages_of(case["kv"], P)
        pages = 1 + B * m
        state.update(_pool(1, pages, heads, P, hd, g))
        state["table"] = (1 + torch.randperm(pages - 1, generator=g, device="cuda")).to(torch.int32).view(B, m)
        state["kv_len"], state["n_new"] = _lengths(case, g)
        if op == "append":
            d = heads * hd
            state["qkv"] = torch.randn((B * S, 3 * d), generator=g, device="cuda")   # as the QKV product leaves it
            R = min(S + P - 1, m * P)
            state["R"] = R
            state["n_read"] = torch.where(state["n_new"] > 0, torch.minimum(state["n_new"] + (P - 1), state["kv_len"]),
                                          torch.zeros_like(state["n_new"])).to(torch.int32)
            state["k_out"] = torch.zeros((B * R, d), device="cuda")
            state["v_out"] = torch.zeros((B * R, d), device="cuda")
        else:
            d = case["H"] * hd
            state["q"] = torch.randn((B * S, d), generator=g, device="cuda") * 1.5
            state["out"] = torch.zeros((B * S, d), device="cuda")
            state["scale"] = math.sqrt(hd)
    elif op == "copy":
        n = case["n"]
        pages = 1 + 2 * n + n // 4
        state.update(_pool(case["layers"], pages, case["heads"], case["P"], case["hd"], g))
        ids = (1 + torch.randperm(pages - 1, generator=g, device="cuda")).to(torch.int32)
        state["src"], state["dst"] = ids[:n].contiguous(), ids[n:2 * n].contiguous()
    else:
        B, n, V = case["B"], case["n"], case["vocab"]
        # a draft model that knows the target's distribution roughly, and its own samples as the drafts
        base = torch.randn((B, n + 1, V), generator=g, device="cuda") * 2.5
        state["logits"] = base + 0.4 * torch.randn((B, n + 1, V), generator=g, device="cuda")
        draft = base[:, :n] + 0.4 * torch.randn((B, n, V), generator=g, device="cuda")
        noise = -torch.log(-torch.log(torch.rand((B, n, V), generator=g, device="cuda").clamp(1e-30, 1 - 1e-7)))
        T = case["T"]
        state["draft_ids"] = (draft / T + noise if T > 0.01 else draft).argmax(-1).to(torch.int32)
        state["draft_logits"] = draft.contiguous() if case["drafts"] else None
        state["uniforms"] = torch.rand((B, n + 1), generator=g, device="cuda", dtype=torch.float64)
        state["draft_len"] = torch.full((B,), n, dtype=torch.int32, device="cuda")
        if case["ragged"]:
            state["draft_len"] = torch.randint(0, n + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            state["draft_len"][0] = n
        state["out_ids"] = torch.empty((B, n + 1), dtype=torch.int32, device="cuda")
        state["accepted"] = torch.empty((B,), dtype=torch.int32, device="cuda")
    if own:
        gbx = importlib.import_module(PACKAGE)
        state["gbx"] = gbx
        if op != "verify":
            state["cache"] = gbx.KVCache(k=state["k"], v=state["v"], k_scale=state["k_scale"], v_scale=state["v_scale"])
        if op == "attn":
            state["workspace"] = torch.empty(gbx.attn_cached_workspace(state["cache"], B=case["B"], S=case["S"], H=case["H"],
                                                                       max_pages=state["table"].shape[1]), device="cuda")
    return state


# ------------------------------------------------------------------- run
def run(state):
    op = state["op"]
    if op == "append":
        return _append_own(state) if own else _append_plain(state)
    if op == "attn":
        return _attn_own(state) if own else _attn_plain(state)
    if op == "copy":
        return _copy_own(state) if own else _copy_plain(state)
    return _verify_own(state) if own else _verify_plain(state)


def _append_own(s):
    gbx, d = s["gbx"], s["heads"] * s["hd"]
    gbx.kv_append(s["cache"], 0, s["qkv"][:, d:], s["qkv"][:, 2 * d:], s["table"], s["kv_len"], B=s["B"], S=s["S"], ld=3 * d,
                  n_new=s["n_new"])
    gbx.kv_read(s["cache"], 0, s["table"], s["kv_len"], s["k_out"], s["v_out"], B=s["B"], S=s["R"], ld=d, n=s["n_read"])
    return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _attn_own(s):
    d = s["H"] * s["hd"]
    s["gbx"].attn_cached(s["cache"], 0, s["q"], s["out"], s["table"], s["kv_len"], B=s["B"], S=s["S"], H=s["H"], ld=d, ld_out=d,
                         scale=s["scale"], n_new=s["n_new"], workspace=s["workspace"])
    return s["out"]


def _copy_own(s):
    s["gbx"].kv_copy_pages(s["cache"], s["src"], s["dst"], n=s["n"])
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _verify_own(s):
    s["gbx"].verify_tokens(s["logits"], s["draft_ids"], s["out_ids"], s["accepted"], B=s["B"], n_draft=s["n"], vocab=s["vocab"],
                           temperature=s["T"], uniforms=s["uniforms"], draft_logits=s["draft_logits"], draft_len=s["draft_len"])
    return {"ids": s["out_ids"], "accepted": s["accepted"]}


# ------------------------------------------------------------------- plain forms
def _slots(s, rows, count):
    """Page, slot and validity of row (b, i), i < rows, of the last count[b] tokens; page 0 where there is none."""
    i = torch.arange(rows, device="cuda")
    t = (s["kv_len"] - count)[:, None].long() + i
    ok = i < count[:, None]
    t = torch.where(ok, t, torch.zeros_like(t))
    page = torch.where(ok, s["table"].long().gather(1, t // s["P"]), torch.zeros_like(t))
    return page, t % s["P"], ok


def _append_one(s, x, codes, scale, transposed):
    """codes[page, head, slot, :] and scale[page, head] with the rows x [B, S, heads, hd] added."""
    B, S, P = s["B"], s["S"], s["P"]
    page, slot, ok = _slots(s, S, s["n_new"])
    a = torch.where(ok[..., None], x.abs().amax(-1), torch.zeros((), device="cuda"))
    top = torch.zeros_like(scale).scatter_reduce_(0, page.reshape(-1, 1).expand(-1, scale.shape[1]), a.reshape(B * S, -1), "amax")
    fresh = (top.double() / 127.0).float()          # the float nearest to the quotient
    fresh = torch.where(top >= 2.0 ** -100, fresh, torch.zeros_like(fresh))
    # only the first page of a sequence's new tokens can hold earlier ones
    p0, slot0 = page[:, 0], slot[:, 0]
    old = scale[p0]
    grown = torch.where((slot0 > 0)[:, None], torch.maximum(old, fresh[p0]), fresh[p0])
    was = codes[p0].double()
    keep = torch.arange(P, device="cuda") < slot0[:, None]
    if transposed:
        keep, shape = keep.view(B, 1, P // 16, 1, 16), (B, -1, 1, 1, 1)
    else:
        keep, shape = keep.view(B, 1, P, 1), (B, -1, 1, 1)
    div = torch.where(grown > 0, grown, torch.ones_like(grown)).double().view(shape)
    now = torch.where(keep, torch.round(was * old.double().view(shape) / div), was)
    live = (s["n_new"] > 0)
    codes[p0] = torch.where(live.view((B,) + (1,) * (now.dim() - 1)), now, was).to(torch.int8)
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, page.reshape(-1), True)
    touched[0] = False
    fresh = torch.where(touched[:, None], fresh, scale)
    fresh[p0] = torch.where(live[:, None], grown, scale[p0])
    scale.copy_(fresh)
    by = scale[page]                                 # [B, S, heads]
    by = torch.where(by > 0, by, torch.full_like(by, math.inf))
    c = torch.round(x.double() / by.double()[..., None]).to(torch.int8)
    if transposed:
        codes[page, :, slot // 16, :, slot % 16] = c
    else:
        codes[page, :, slot] = c


def _append_plain(s):
    B, S, R, heads, hd = s["B"], s["S"], s["R"], s["heads"], s["hd"]
    d = heads * hd
    page, slot, ok = _slots(s, R, s["n_read"])
    for name, at, transposed in (("k", 1, False), ("v", 2, True)):
        codes, scale, out = s[name][0], s[name + "_scale"][0], s[name + "_out"]
        _append_one(s, s["qkv"][:, at * d:(at + 1) * d].view(B, S, heads, hd), codes, scale, transposed)
        got = codes[page, :, slot // 16, :, slot % 16] if transposed else codes[page, :, slot]
        vals = (got.float() * scale[page][..., None]).reshape(B, R, d)
        out.copy_(torch.where(ok[..., None], vals, out.view(B, R, d)).view(B * R, d))
    return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _attn_plain(s):
    B, S, H, heads, hd, P = (s[k] for k in ("B", "S", "H", "heads", "hd", "P"))
    table = s["table"].long()
    L = table.shape[1] * P
    k = s["k"][0][table].float() * s["k_scale"][0][table][..., None, None]              # [B, m, heads, P, hd]
    k = k.permute(0, 2, 1, 3, 4).reshape(B, heads, L, hd)
    v = s["v"][0][table].float() * s["v_scale"][0][table][..., None, None, None]        # [B, m, heads, P/16, hd, 16]
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(B, heads, L, hd)
    q = s["q"].view(B, S, heads, H // heads, hd).permute(0, 2, 3, 1, 4).reshape(B, heads, -1, hd)
    x = (q @ k.transpose(-1, -2)) / s["scale"]
    i = torch.arange(S, device="cuda")
    limit = (s["kv_len"] - s["n_new"])[:, None] + i + 1                                  # keys that row i sees
    limit = limit.repeat(1, H // heads)[:, None, :, None]
    x = x.masked_fill(torch.arange(L, device="cuda") >= limit, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    o = (e @ v) / e.sum(-1, keepdim=True)
    o = o.view(B, heads, H // heads, S, hd).permute(0, 3, 1, 2, 4).reshape(B, S, H * hd)
    live = (i < s["n_new"][:, None])[..., None]
    s["out"].copy_(torch.where(live, o, s["out"].view(B, S, H * hd)).view(B * S, H * hd))
    return s["out"]


def _copy_plain(s):
    src, dst = s["src"].long(), s["dst"].long()
    for name in ("k", "v", "k_scale", "v_scale"):
        s[name][:, dst] = s[name][:, src]
    return {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _verify_plain(s):
    B, n, V, T = s["B"], s["n"], s["vocab"], s["T"]
    logits, ids, length = s["logits"], s["draft_ids"].long(), s["draft_len"].long()
    i = torch.arange(n, device="cuda")
    if T <= 0.01:
        best = logits.argmax(-1)
        ok = best[:, :n] == ids
    else:
        # in 64 bits: a draw next to a border of the cumulative sum decides which token comes out
        x = logits.double() / T
        e = torch.exp(x - x.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        if s["draft_logits"] is None:
            q = torch.zeros((B, n, V), dtype=torch.float64, device="cuda").scatter_(2, ids[..., None], 1.0)
        else:
            x = s["draft_logits"].double() / T
            e = torch.exp(x - x.amax(-1, keepdim=True))
            q = e / e.sum(-1, keepdim=True)
        pd = p[:, :n].gather(2, ids[..., None])[..., 0]
        qd = q.gather(2, ids[..., None])[..., 0]
        ok = s["uniforms"][:, :n] * qd < pd
    ok = ok & (i < length[:, None])
    acc = ok.long().cumprod(1).sum(1)
    if T <= 0.01:
        nxt = best.gather(1, acc[:, None])[:, 0]
    else:
        row = p.gather(1, acc[:, None, None].expand(-1, 1, V))[:, 0]
        rej = acc < length
        at = torch.where(rej, acc, torch.zeros_like(acc))
        less = torch.where(rej[:, None], q.gather(1, at[:, None, None].expand(-1, 1, V))[:, 0], torch.zeros_like(row))
        r = (row - less).clamp_min(0)
        c = r.cumsum(1)
        nxt = (c > (s["uniforms"][:, n] * c[:, -1])[:, None]).long().argmax(1)
    j = torch.arange(n + 1, device="cuda")
    out = torch.where(j < acc[:, None], torch.nn.functional.pad(ids, (0, 1)), torch.full_like(ids[:, :1], -1))
    out = torch.where(j == acc[:, None], nxt[:, None], out)
    s["out_ids"].copy_(out)
    s["accepted"].copy_(acc)
    return {"ids": s["out_ids"], "accepted": s["accepted"]}


# ------------------------------------------------------------------- work
def _mean_len(case):
    """Expected cached tokens and new rows of a sequence."""
    if not case["ragged"]:
        return case["kv"], case["S"]
    return (case["kv"] - case["S"]) / 2 + case["S"] / 2, case["S"] / 2


def work(case):
    op = case["op"]
    if op == "append":
        d = case["heads"] * case["hd"]
        _, rows = _mean_len(case)
        read = min(rows + case["P"] - 1, case["kv"])
        # K and V rows in as fp32, codes out, and the values of the touched pages out as fp32
        return {"bytes": case["B"] * d * (8 * rows + 2 * read + 8 * read), "flops": 8.0 * case["B"] * d * rows}
    if op == "attn":
        kv, rows = _mean_len(case)
        cache = case["B"] * case["heads"] * kv * (2 * case["hd"] + 8 / case["P"])
        keys = kv - (rows - 1) / 2 if case["S"] > 1 else kv
        return {"bytes": cache + 8 * case["B"] * rows * case["H"] * case["hd"],
                "flops": 4.0 * case["B"] * rows * case["H"] * case["hd"] * keys}
    if op == "copy":
        return {"bytes": 2 * case["n"] * case["layers"] * case["heads"] * (2 * case["P"] * case["hd"] + 8), "flops": 0}
    n = case["n"] / 2 if case["ragged"] else case["n"]
    rows = case["B"] * (n + 1 + (n if case["drafts"] and case["T"] > 0.01 else 0))
    return {"bytes": 4 * rows * case["vocab"], "flops": 4.0 * rows * case["vocab"]}


# ------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definition in 64 bits, sequence by sequence."""
    op = case["op"]
    if op in ("copy", "verify"):
        return None                                   # whole numbers and copies
    s = prepare(case, seed)
    return _exact_attn(s) if op == "attn" else _exact_append(s)


def _exact_attn(s):
    B, S, H, heads, hd, P = (s[k] for k in ("B", "S", "H", "heads", "hd", "P"))
    out = torch.zeros((B, S, H, hd), dtype=torch.float64, device="cuda")
    lens, news = s["kv_len"].tolist(), s["n_new"].tolist()
    q = s["q"].double().view(B, S, H, hd)
    for b in range(B):
        L, n = lens[b], news[b]
        if not L or not n:
            continue
        pages = s["table"][b, :-(-L // P)].long()
        k = torch.einsum("mhpd,mh->hmpd", s["k"][0, pages].double(), s["k_scale"][0, pages].double()).reshape(heads, -1, hd)[:, :L]
        v = torch.einsum("mhgdt,mh->hmgtd", s["v"][0, pages].double(), s["v_scale"][0, pages].double()).reshape(heads, -1, hd)[:, :L]
        for h0 in range(0, heads, 4):                 # a few heads at a time
            qq = q[b, :n].view(n, heads, H // heads, hd)[:, h0:h0 + 4]
            x = torch.einsum("shgd,htd->shgt", qq, k[h0:h0 + 4]) / s["scale"]
            seen = torch.arange(L, device="cuda")[None] <= (L - n + torch.arange(n, device="cuda"))[:, None]
            w = torch.softmax(x.masked_fill(~seen[:, None, None], -math.inf), -1)
            o = torch.einsum("shgt,htd->shgd", w, v[h0:h0 + 4])
            out[b, :n].view(n, heads, H // heads, hd)[:, h0:h0 + 4] = o
    return out.view(B * S, H * hd)


def _exact_append(s):
    B, S, R, heads, hd, P = (s[k] for k in ("B", "S", "R", "heads", "hd", "P"))
    d = heads * hd
    lens, news, reads = s["kv_len"].tolist(), s["n_new"].tolist(), s["n_read"].tolist()
    x = s["qkv"].view(B, S, 3, heads, hd)
    table = s["table"].tolist()
    got = {}
    for name, at in (("k", 1), ("v", 2)):
        scale = s[name + "_scale"][0].double()
        out = torch.zeros((B, R, heads, hd), dtype=torch.float64, device="cuda")
        for b in range(B):
            first, i = lens[b] - news[b], 0
            vals = []
            while i < news[b]:                        # page by page
                page, slot = table[b][(first + i) // P], (first + i) % P
                n = min(P - slot, news[b] - i)
                new = x[b, i:i + n, at].double()                                        # [n, heads, hd]
                grown = (new.abs().amax((0, 2)) / 127).float().double()
                if slot:
                    was = s[name][0, page].double()
                    was = was if name == "k" else was.permute(0, 1, 3, 2).reshape(heads, P, hd)
                    was = was[:, :slot].permute(1, 0, 2)
                    before = scale[page]
                    grown = torch.maximum(before, grown)
                    vals.append((was * before[:, None] / grown[:, None]).round() * grown[:, None])
                vals.append((new / grown[:, None]).round() * grown[:, None])
                scale[page] = grown
                i += n
            if not vals:
                continue
            have = torch.cat(vals)
            n = reads[b]
            lack = n - have.shape[0]
            if lack > 0:                              # tokens of the page before, as they were
                t = range(lens[b] - n, lens[b] - n + lack)
                pages = torch.tensor([table[b][u // P] for u in t], device="cuda")
                slots = torch.tensor([u % P for u in t], device="cuda")
                old = (s[name][0][pages, :, slots] if name == "k" else s[name][0][pages, :, slots // 16, :, slots % 16]).double()
                have = torch.cat([old * scale[pages][..., None], have])
            out[b, :n] = have[-n:]
        got[name] = out.view(B * R, d)
        got[name + "_scale"] = scale[None]
    return got
