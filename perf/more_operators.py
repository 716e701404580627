"""The operators of a step that takes many tokens at once, as they are measured:
prompts that enter, and trees of drafted tokens that are checked.

    product  `build("qgemm")`: many tokens times an INT8 weight with a scale for
             each output channel.  The tokens are quantized to INT8 with a scale
             each (`quantize_tokens`), the sums are whole numbers (`forward`).
    place    `build("attention").place`: from the requests' lengths the pages
             that they need, their block tables, and for every token of the
             packed batch its position and its slot in the cache.
    rows     `append_rows`: packed keys and values quantized into the cache at
             those slots.  What the cache then holds is read back.
    prompt   `prompt`: attention of packed sequences over their own tokens,
             causal, grouped heads.
    tree     `forward(tree=...)`: drafted tokens that form a tree attend to the
             quantized cache and to their ancestors.

With `own` false `run` computes the same in elementary torch operations; with
`own` true it makes the framework's calls.  Inputs come from the case and the
seed alone.  Lengths come from the case: all `most`, or spread over [0, most],
the first the longest and one of them empty.

A page of the cache holds `page` tokens of every key/value head:
    K       int8 [pages, heads, page, D], or uint8 [.., D/2] for 4 bits
            (dim 2j in the low nibble of byte j, 2j + 1 in the high one)
    V       int8 [pages, heads, page / 16, D, 16], or uint8 [.., D/2, 16]
    scales  fp32 [pages, heads, 2, page]: K's, then V's
and a value is its code times its token's scale.
"""
import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _product(name, tokens, n, k, dtype):
    return {"name": name, "kind": "product", "tokens": tokens, "n": n, "k": k, "dtype": dtype}


def _place(name, batch, most, ragged, behind, page, spare):
    return {"name": name, "kind": "place", "batch": batch, "most": most, "ragged": ragged,
            "behind": behind, "page": page, "spare": spare}


def _rows(name, batch, most, ragged, behind, kept, hkv, d, bits, page, dtype):
    return {"name": name, "kind": "rows", "batch": batch, "most": most, "ragged": ragged,
            "behind": behind, "kept": kept, "hkv": hkv, "d": d, "bits": bits, "page": page,
            "dtype": dtype}


def _prompt(name, batch, most, ragged, ahead, causal, hq, hkv, d, dtype, fused):
    return {"name": name, "kind": "prompt", "batch": batch, "most": most, "ragged": ragged,
            "ahead": ahead, "causal": causal, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype,
            "fused": fused}


def _tree(name, batch, new, most, ragged, hq, hkv, d, bits, page, dtype):
    return {"name": name, "kind": "tree", "batch": batch, "new": new, "most": most,
            "ragged": ragged, "hq": hq, "hkv": hkv, "d": d, "bits": bits, "page": page,
            "dtype": dtype}


def listed():
    return [
        # seven sequences check five drafted tokens each through one of
        # Llama-70B's square projections: few rows, the weights are what is read
        _product("product_draft", 35, 8192, 8192, "fp16"),
        # a small batch of prompts, sizes that divide by nothing
        _product("product_ragged", 777, 5003, 4100, "bf16"),
        # a long prompt through Llama-70B's gate projection: the largest arithmetic
        _product("product_prompt", 4096, 28672, 8192, "fp16"),
        # a decode step of a batch: one token each, now and then a new page
        _place("place_step", 256, 1, False, 1000, 64, 0),
        # prompts of unequal length enter, rows to spare behind the last
        _place("place_prompts", 64, 4096, True, 0, 16, 77),
        # checked drafts: of five tokens each those that were accepted go to
        # the places behind one another, the others nowhere
        _rows("rows_accepted", 64, 5, False, 1000, 0.6, 8, 128, 8, 64, "fp16"),
        # packed prompts of Llama-70B's key/value heads enter in 4 bits
        _rows("rows_prompts", 16, 2048, True, 0, 1.0, 8, 128, 4, 64, "bf16"),
        # a few short prompts of odd heads: latency counts
        _prompt("prompt_short", 5, 100, True, 0, True, 28, 4, 64, "bf16", False),
        # a batch of prompts of Llama-7B's heads (no grouping), q, k and v as
        # views of one tensor
        _prompt("prompt_packed", 16, 2048, True, 0, True, 32, 32, 128, "fp16", True),
        # one long prompt of Llama-70B's heads
        _prompt("prompt_long", 1, 8192, False, 0, True, 64, 8, 128, "bf16", True),
        # small trees, odd counts, some sequences shorter than the draft
        _tree("tree_small", 7, 13, 1501, True, 28, 4, 64, 8, 32, "bf16"),
        # a batch of large trees over long contexts
        _tree("tree_batch", 16, 48, 8000, True, 64, 8, 128, 8, 64, "fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["product", "product", "place", "rows", "prompt", "prompt", "tree"])
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "product":
        k = _log(rng, 64, 28672)
        n = _log(rng, 64, 28672)
        if rng.random() < 0.7:
            k = (k + 127) // 128 * 128
        if rng.random() < 0.5:
            n = (n + 63) // 64 * 64
        room = 4096 * 28672 * 8192 // (n * k)
        c = _product("", _log(rng, 1, max(1, min(room, 8192))), n, k, dtype)
    elif kind == "place":
        batch = _log(rng, 1, 1024)
        most = 1 if rng.random() < 0.3 else _log(rng, 1, max(1, 131072 // batch))
        c = _place("", batch, most, rng.random() < 0.7 and most > 1,
                   rng.choice([0, 0, 1, 15, 16, 1000]), page, rng.choice([0, 0, 1, 300]))
    elif kind == "rows":
        d, hkv = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 5, 8, 16])
        batch = _log(rng, 1, 64)
        room = 16 * 2048 * 8 * 128 // (batch * hkv * d)
        most = _log(rng, 1, max(1, room))
        c = _rows("", batch, most, rng.random() < 0.7 and most > 1,
                  rng.choice([0, 0, 1, 37, 1000]), rng.choice([1.0, 1.0, 0.6]), hkv, d,
                  rng.choice([4, 8]), page, dtype)
    elif kind == "prompt":
        d = rng.choice([64, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8, 16])
        hq = hkv * rng.choice([1, 2, 4, 7, 8])
        batch, most = _log(rng, 1, 64), _log(rng, 1, 8192)
        ahead = rng.choice([0, 0, 0, 1, 129, 2000])
        while batch * hq * most * (most + ahead) * d > 64 * 8192 * 8192 * 128:
            batch, most, ahead = (batch + 1) // 2, (most * 3 + 3) // 4, ahead // 2
        c = _prompt("", batch, most, rng.random() < 0.8 and batch > 1, ahead,
                    rng.random() < 0.85, hq, hkv, d, dtype, rng.random() < 0.5)
    else:
        d = rng.choice([64, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4, 7, 8])
        batch, new, most = _log(rng, 1, 32), rng.choice([2, 5, 9, 16, 33, 64, 70]), _log(rng, 1, 8000)
        while batch * new * hq * most * d > 16 * 48 * 64 * 8000 * 128:
            batch, most = (batch + 1) // 2, (most + 1) // 2
        c = _tree("", batch, new, most, rng.random() < 0.8, hq, hkv, d, rng.choice([4, 8]),
                  page, dtype)
    del c["name"]
    return c


def _lengths(case):
    """Tokens of each sequence: all `most`, or spread over [0, most] with the
    first the longest and, of three or more, the third empty."""
    most, n = case["most"], case["batch"]
    if not case["ragged"]:
        return [most] * n
    spread = [most] + [1 + int((most - 1) * ((b * 0.6180339887498949) % 1.0))
                       for b in range(1, n)]
    if n > 2 and case["kind"] != "tree":
        spread[2] = 0
    return spread


def _pages(tokens, page):
    return (tokens + page - 1) // page


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _tables(totals, page, g):
    """A block table over shuffled pages for sequences of `totals` tokens, and
    the number of pages."""
    need = [_pages(t, page) for t in totals]
    count = sum(need) + 1
    order = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(totals), max(max(need), 1), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, count


def _pool(case, pages, g):
    """A cache with valid codes everywhere: values of about unit size."""
    h, d, page, bits = case["hkv"], case["d"], case["page"], case["bits"]
    top = 127 if bits == 8 else 7

    def codes(*shape):
        if bits == 8:
            return torch.randint(-top, top + 1, shape, generator=g, device="cuda",
                                 dtype=torch.int8)
        lo, hi = (torch.randint(-top, top + 1, shape, generator=g, device="cuda",
                                dtype=torch.int8).view(torch.uint8) & 15
                  for _ in range(2))
        return lo | (hi << 4)

    row = d if bits == 8 else d // 2
    k = codes(pages, h, page, row)
    v = codes(pages, h, page // 16, row, 16)
    s = (0.75 + 0.5 * torch.rand(pages, h, 2, page, generator=g, device="cuda")) * (1.7 / top)
    return {"k": k, "v": v, "scales": s}


def _trees(batch, new, g):
    """Which of the drafted tokens each one sees, itself and its ancestors, as
    bits (batch, new, words): token t hangs on one of those before it or, now
    and then, on none."""
    parents = torch.rand(batch, new, generator=g, device="cuda").cpu()
    words = (new + 63) // 64
    rows = []
    for b in range(batch):
        seen = []
        for t in range(new):
            up = int(parents[b, t] * (t + 1)) - 1
            seen.append((seen[up] if up >= 0 else 0) | (1 << t))
        rows.append([[((m >> (64 * w)) & (2 ** 64 - 1)) for w in range(words)] for m in seen])
    signed = [[[x - 2 ** 64 if x >= 2 ** 63 else x for x in m] for m in r] for r in rows]
    return torch.tensor(signed, dtype=torch.int64).cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    st = {"case": case}

    def normal(*shape, by=1.0):
        x = torch.randn(*shape, generator=g, device="cuda")
        return (x * by).to(TYPES[case["dtype"]])

    if own:
        from cudalab_amd.build import build
        st["att" if kind != "product" else "gemm"] = build(
            "attention" if kind != "product" else "qgemm")
    if kind == "product":
        n, k = case["n"], case["k"]
        st["x"] = normal(case["tokens"], k)
        st["w"] = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
        # a weight of unit variance over its row keeps y of about unit size
        st["scale"] = ((0.5 + torch.rand(n, generator=g, device="cuda"))
                       / (73.3 * math.sqrt(k)))
        return st
    lens = _lengths(case)
    st["lens"] = lens
    if kind == "place":
        page, before = case["page"], case["behind"]
        held = _pages(before, page)
        cols = max(_pages(before + case["most"], page), 1)
        need = sum(_pages(before + n, page) - held for n in lens if n)
        order = torch.randperm(held * len(lens) + need + 9, generator=g, device="cuda")
        order = order.to(torch.int32)
        st["table"] = torch.full((len(lens), cols), -1, dtype=torch.int32, device="cuda")
        st["table"][:, :held] = order[:held * len(lens)].view(len(lens), held)
        st["free"] = order[held * len(lens):].contiguous()
        st["starts"], st["counts"] = _ints([before] * len(lens)), _ints(lens)
        st["tokens"] = sum(lens) + case["spare"]
        return st
    if kind == "prompt":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        seen = [n + case["ahead"] for n in lens]
        rows, keys = sum(lens), sum(seen)
        st["q"] = normal(rows, hq, d)
        st["k"], st["v"] = normal(keys, hkv, d), normal(keys, hkv, d)
        if case["fused"] and rows == keys:
            wide = normal(rows, (hq + 2 * hkv) * d)
            st["q"] = wide[:, :hq * d].view(rows, hq, d)
            st["k"] = wide[:, hq * d:(hq + hkv) * d].view(rows, hkv, d)
            st["v"] = wide[:, (hq + hkv) * d:].view(rows, hkv, d)
        st["offsets"] = _ints(_offsets(lens))
        st["k_offsets"] = _ints(_offsets(seen)) if case["ahead"] else None
        return st
    if kind == "rows":
        before, page = case["behind"], case["page"]
        st["table"], pages = _tables([before + n for n in lens], page, g)
        st["starts"], st["counts"] = _ints([before] * len(lens)), _ints(lens)
        total = sum(lens)
        st["new_k"], st["new_v"] = (normal(total, case["hkv"], case["d"]) for _ in range(2))
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"),
                                      torch.tensor(lens, device="cuda"))
        first = torch.tensor(_offsets(lens)[:-1], device="cuda")[seq]
        keep = torch.rand(total, generator=g, device="cuda") < case["kept"]
        rank = torch.cumsum(keep, 0) - keep.long()
        start = torch.cat((rank, rank.new_zeros(1)))[first]
        pos = before + rank - start
        slot = st["table"].long()[seq, pos // page] * page + pos % page
        st["slots"] = torch.where(keep, slot, -1)
    else:
        st["table"], pages = _tables(lens, case["page"], g)
        st["lengths"] = _ints(lens)
        st["q"] = normal(case["batch"], case["new"], case["hq"], case["d"], by=1.5)
        st["tree"] = _trees(case["batch"], case["new"], g)
    st["pool"] = _pool(case, pages, g)
    if own:
        from cudalab_amd.kvcache import KVCache
        p = st["pool"]
        st["cache"] = KVCache(p["k"], p["v"], p["scales"])
    return st


# ------------------------------------------------------------- plain forms
def _plain_product(st):
    x = st["x"].float()
    recip = torch.tensor(1.0, device="cuda") / 127.0
    scale = x.abs().amax(dim=-1) * recip
    code = torch.round(x * (1.0 / scale)[:, None]).clamp(-127.0, 127.0)
    y = torch.matmul(code, st["w"].float().t())
    return (y * scale[:, None] * st["scale"]).to(st["x"].dtype)


def _plain_place(st):
    page, tokens, table, free = st["case"]["page"], st["tokens"], st["table"], st["free"]
    starts, counts = st["starts"].long(), st["counts"].long()
    ends = torch.cumsum(counts, 0)
    offsets = torch.cat((ends.new_zeros(1), ends))
    lengths = starts + counts
    have, want = (starts + page - 1) // page, (lengths + page - 1) // page
    need = torch.where(counts > 0, want - have, 0)
    upto = torch.cumsum(need, 0)
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    new = (col >= have[:, None]) & (col < (have + need)[:, None])
    index = (upto - need)[:, None] + col - have[:, None]
    table.copy_(torch.where(new, free.long()[index.clamp(0, free.shape[0] - 1)], table.long()))
    t = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(ends, t, right=True)
    live = seq < counts.shape[0]
    seq = seq.clamp(max=counts.shape[0] - 1)
    pos = torch.where(live, starts[seq] + t - offsets[seq], 0)
    entry = table.long()[seq, (pos // page).clamp(max=table.shape[1] - 1)]
    slots = torch.where(live & (entry >= 0), entry * page + pos % page, -1)
    i32 = torch.int32
    return [slots, pos.to(i32), offsets.to(i32), lengths.to(i32), upto[-1:].to(i32), table]


def _unpack(codes, bits, dim):
    """Codes as numbers; for 4 bits axis `dim` doubles."""
    if bits == 8:
        return codes.to(torch.float32)
    b = codes.to(torch.int32)
    two = torch.stack((b & 15, b >> 4), dim=dim + 1)
    two = two - ((two & 8) << 1)
    return two.flatten(dim, dim + 1).to(torch.float32)


def _plain_rows(st):
    c = st["case"]
    bits, page = c["bits"], c["page"]
    top = 127.0 if bits == 8 else 7.0
    some = st["slots"] >= 0
    slots = st["slots"][some]
    at, off = slots // page, slots % page
    pool = st["pool"]
    for which, x in ((0, st["new_k"]), (1, st["new_v"])):
        f = x[some].float()                                  # n, h, D
        recip = torch.tensor(1.0, device="cuda") / top
        scale = f.abs().amax(dim=-1) * recip
        code = torch.round(f * (1.0 / scale)[..., None]).clamp(-top, top).to(torch.int32)
        if bits == 4:
            code = (code[..., 0::2] & 15) | ((code[..., 1::2] & 15) << 4)
        if which == 0:
            pool["k"][at, :, off] = code.to(pool["k"].dtype)
        else:
            pool["v"][at, :, off // 16, :, off % 16] = code.to(pool["v"].dtype)
        pool["scales"][at, :, which, off] = scale
    # what the sequences' places hold now
    t = torch.arange(c["most"], device="cuda")[None, :]
    pos = st["starts"].long()[:, None] + t
    valid = t < st["counts"][:, None]
    col = (pos // page).clamp(max=st["table"].shape[1] - 1)
    at, off = st["table"].long().gather(1, col), pos % page
    outs = []
    for which in (0, 1):
        code = pool["k"][at, :, off] if which == 0 else pool["v"][at, :, off // 16, :, off % 16]
        val = _unpack(code, bits, 3) * pool["scales"][at, :, which, off][..., None]
        outs.append(torch.where(valid[:, :, None, None], val, 0.0).to(TYPES[c["dtype"]]))
    return outs


def _softmax_rows(s):
    """The softmax of scores with -Inf where nothing is seen; rows of zeros
    where that is all."""
    m = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(dim=-1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0)


def _plain_prompt(st):
    c = st["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    g = hq // hkv
    out = torch.zeros(st["q"].shape, dtype=st["q"].dtype, device="cuda")
    at = kat = 0
    for n in st["lens"]:
        m = n + c["ahead"]
        if n:
            q = st["q"][at:at + n].float().view(n, hkv, g, d).permute(1, 2, 0, 3)
            k = st["k"][kat:kat + m].float().permute(1, 2, 0).contiguous()    # hkv, d, m
            v = st["v"][kat:kat + m].float().transpose(0, 1).contiguous()     # hkv, m, d
            step = max(1, min(hkv, 2 ** 29 // (g * n * m)))
            hidden = (torch.arange(m, device="cuda")[None, :]
                      > torch.arange(m - n, m, device="cuda")[:, None])
            for h in range(0, hkv, step):
                hs = slice(h, min(h + step, hkv))
                s = torch.matmul(q[hs].reshape(-1, g * n, d), k[hs]) * d ** -0.5
                s = s.view(-1, g, n, m)
                if c["causal"]:
                    s = torch.where(hidden, -math.inf, s)
                o = torch.matmul(_softmax_rows(s).view(-1, g * n, m), v[hs])
                o = o.view(-1, g, n, d).permute(2, 0, 1, 3).reshape(n, -1, d)
                out[at:at + n, hs.start * g:hs.stop * g] = o.to(out.dtype)
        at, kat = at + n, kat + m
    return out


def _seen_bits(words, new):
    """Bits (.., words) as truth values (.., new)."""
    j = torch.arange(new, device="cuda")
    return ((words[..., j // 64] >> (j % 64)) & 1).bool()


def _plain_tree(st):
    c = st["case"]
    b, t, hq, hkv, d = c["batch"], c["new"], c["hq"], c["hkv"], c["d"]
    g = hq // hkv
    table = st["table"].long()
    k = _unpack(st["pool"]["k"][table], c["bits"], 4)        # b, w, h, page, D
    v = _unpack(st["pool"]["v"][table], c["bits"], 4)        # b, w, h, page/16, D, 16
    v = v.transpose(4, 5).flatten(3, 4)
    s = st["pool"]["scales"][table]                          # b, w, h, 2, page
    k, v = (x.permute(0, 2, 1, 3, 4).flatten(2, 3)
            for x in (k * s[:, :, :, 0, :, None], v * s[:, :, :, 1, :, None]))
    q = st["q"].float().view(b, t, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * g, d)
    s = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    bits = _seen_bits(st["tree"], t)                         # b, t, t
    first = st["lengths"].long() - t                         # where the drafts start
    j = torch.arange(k.shape[2], device="cuda")[None, :] - first[:, None]     # b, keys
    among = bits.gather(2, j.clamp(0, t - 1)[:, None, :].expand(b, t, j.shape[1]))
    seen = torch.where((j < 0)[:, None], True, among & (j < t)[:, None])
    seen = seen.repeat_interleave(g, dim=1)[:, None]
    o = torch.matmul(_softmax_rows(torch.where(seen, s, -math.inf)), v)
    o = o.view(b, hkv, t, g, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d)
    return o.to(st["q"].dtype)


def run(state):
    c = state["case"]
    kind = c["kind"]
    if not own:
        return {"product": _plain_product, "place": _plain_place, "rows": _plain_rows,
                "prompt": _plain_prompt, "tree": _plain_tree}[kind](state)
    if kind == "product":
        gemm = state["gemm"]
        codes, scales = gemm.quantize_tokens(state["x"])
        return gemm.forward(codes, scales, state["w"], state["scale"], state["x"].dtype)
    att = state["att"]
    if kind == "place":
        p = att.place(state["table"], state["starts"], state["counts"], state["tokens"],
                      c["page"], state["free"])
        return [p.slots, p.positions, p.offsets, p.lengths, p.taken, state["table"]]
    if kind == "rows":
        att.append_rows(state["cache"], state["new_k"], state["new_v"], state["slots"])
        return att.read(state["cache"], state["table"], state["starts"], state["counts"],
                        c["most"], TYPES[c["dtype"]])
    if kind == "prompt":
        return att.prompt(state["q"], state["k"], state["v"], state["offsets"],
                          k_offsets=state["k_offsets"], causal=c["causal"])
    return att.forward(state["q"], state["cache"], state["table"], state["lengths"],
                       tree=state["tree"])


def work(case):
    kind = case["kind"]
    if kind == "product":
        m, n, k = case["tokens"], case["n"], case["k"]
        return {"bytes": n * k + 4 * n + 2 * m * (n + k), "flops": 2 * m * n * k + 4 * m * k}
    lens = _lengths(case)
    total, batch = sum(lens), case["batch"]
    if kind == "place":
        pages = sum(_pages(case["behind"] + n, case["page"])
                    - _pages(case["behind"], case["page"]) for n in lens if n)
        # slots, positions; starts, counts, offsets, lengths; pages from the
        # free list to the table; entries of pages that are already held
        held = sum(1 for n in lens if n and case["behind"] % case["page"])
        return {"bytes": 12 * (total + case["spare"]) + 16 * batch + 8 * pages + 4 * held,
                "flops": 6 * total}
    d, hkv = case["d"], case["hkv"]
    if kind == "prompt":
        es, rows = 2, case["hq"]
        ahead = case["ahead"]
        if case["causal"]:
            pairs = sum(n * ahead + n * (n + 1) // 2 for n in lens)
        else:
            pairs = sum(n * (n + ahead) for n in lens)
        keys = sum(n + ahead for n in lens if n)
        return {"bytes": 2 * total * rows * d * es + 2 * keys * hkv * d * es,
                "flops": 4 * d * rows * pairs}
    token = hkv * 2 * (d * case["bits"] // 8 + 4)            # codes and scales of one
    if kind == "rows":
        kept = int(total * case["kept"])
        whole = batch * case["most"] * hkv * d * 2 * 2
        return {"bytes": kept * hkv * d * 2 * 2 + kept * token + total * (token + 8) + whole,
                "flops": 6 * kept * hkv * d * 2}
    t, rows = case["new"], case["hq"]
    # a drafted token sees a few of the others; counted as half of them
    seen = sum(max(0, n - t) * t + min(n, t) * (min(n, t) + 1) // 2 for n in lens)
    return {"bytes": 2 * batch * t * rows * d * 2 + sum(lens) * token,
            "flops": 4 * d * rows * seen}


# ------------------------------------------------- from the definition, FP64
def _exact_product(st):
    """Codes from the definition: the scale is amax times the FP32 number
    nearest 1 / 127, rounded to FP32, as is its reciprocal; a code is the integer
    nearest (ties to even) the FP32 product of value and reciprocal."""
    x = st["x"].double()
    step = (x.abs().amax(1, keepdim=True) * torch.tensor(1 / 127).double().item())
    step = step.float().double()
    back = (1 / step).float().double()
    code = (x * back).float().double().round()
    out = torch.empty(x.shape[0], st["w"].shape[0], dtype=torch.float64, device="cuda")
    for n in range(0, out.shape[1], 8192):
        part = slice(n, n + 8192)
        out[:, part] = code @ st["w"][part].double().T * st["scale"][part].double()
    return out * step


def _exact_place(st):
    """Sequence by sequence, on the host."""
    page = st["case"]["page"]
    table, free = st["table"].cpu().tolist(), st["free"].cpu().tolist()
    slots, positions, offsets, lengths, taken = [], [], [0], [], 0
    for b, n in enumerate(st["lens"]):
        before = st["case"]["behind"]
        held = -(-before // page)
        for t in range(before, before + n):
            if t // page >= held:
                table[b][held] = free[taken]
                taken += 1
                held += 1
            slots.append(table[b][t // page] * page + t % page)
            positions.append(t)
        offsets.append(offsets[-1] + n)
        lengths.append(before + n)
    spare = st["tokens"] - len(slots)
    return [torch.tensor(x, dtype=torch.int64, device="cuda")
            for x in (slots + [-1] * spare, positions + [0] * spare, offsets, lengths, [taken],
                      table)]


def _exact_values(st, table, n, which):
    """Values [heads, n, D] of a sequence's first n tokens in FP64."""
    c = st["case"]
    d, bits, page = c["d"], c["bits"], c["page"]
    ids = table[:_pages(n, page)].long()
    raw = st["pool"]["k" if which == 0 else "v"][ids]
    if which == 1:                                           # w, h, page/16, row, 16
        raw = raw.movedim(3, 4).reshape(raw.shape[0], raw.shape[1], page, raw.shape[3])
    if bits == 4:
        wide = torch.empty(*raw.shape[:-1], d, dtype=torch.float64, device="cuda")
        for side in (0, 1):
            nib = (raw >> (4 * side)) & 15
            wide[..., side::2] = nib.double() - 16.0 * (nib > 7)
        raw = wide
    val = raw.double() * st["pool"]["scales"][ids][:, :, which, :, None].double()
    return val.transpose(0, 1).reshape(c["hkv"], -1, d)[:, :n]


def _exact_rows(st):
    """What the places hold: the calls' tokens quantized by the definition (as
    the product's), and what was there where none came."""
    c = st["case"]
    top = 127 if c["bits"] == 8 else 7
    before, res = c["behind"], []
    for which, name in ((0, "new_k"), (1, "new_v")):
        x = st[name].double()
        step = x.abs().amax(-1, keepdim=True) * torch.tensor(1 / top).double().item()
        step = step.float().double()
        back = (1 / step).float().double()
        new = (x * back).float().double().round() * step
        val = torch.zeros(c["batch"], c["most"], c["hkv"], c["d"], dtype=torch.float64,
                          device="cuda")
        at = 0
        for b, n in enumerate(st["lens"]):
            if n:
                old = _exact_values(st, st["table"][b], before + n, which)
                val[b, :n] = old[:, before:].transpose(0, 1)
                came = new[at:at + n][st["slots"][at:at + n] >= 0]
                val[b, :came.shape[0]] = came
            at += n
        res.append(val)
    return res


def _exact_prompt(st):
    c = st["case"]
    g, d = c["hq"] // c["hkv"], c["d"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    at = kat = 0
    for n in st["lens"]:
        m = n + c["ahead"]
        last = torch.arange(n, device="cuda")[:, None] + c["ahead"]
        above = torch.arange(m, device="cuda")[None, :] > last
        for h in range(c["hq"] if n else 0):
            k, v = (st[x][kat:kat + m, h // g].double() for x in ("k", "v"))
            z = st["q"][at:at + n, h].double() @ k.T / math.sqrt(d)
            if c["causal"]:
                z.masked_fill_(above, -math.inf)
            out[at:at + n, h] = torch.softmax(z, dim=1) @ v
        at, kat = at + n, kat + m
    return out


def _exact_tree(st):
    c = st["case"]
    t, hkv, d = c["new"], c["hkv"], c["d"]
    g = c["hq"] // hkv
    out = torch.zeros(c["batch"], t, c["hq"], d, dtype=torch.float64, device="cuda")
    words = st["tree"].cpu().tolist()
    for b, n in enumerate(st["lens"]):
        k, v = (_exact_values(st, st["table"][b], n, w) for w in (0, 1))
        hidden = torch.zeros(t, n, dtype=torch.bool)
        for i in range(t):
            for j in range(t):
                if n - t + j >= 0 and not (words[b][i][j // 64] >> (j % 64)) & 1:
                    hidden[i, n - t + j] = True
        some = (~hidden).any(dim=1).cuda().repeat_interleave(g)
        hidden = hidden.cuda().repeat_interleave(g, dim=0)
        for h in range(hkv):
            q = st["q"][b, :, h * g:(h + 1) * g].double().reshape(t * g, d)
            z = (q @ k[h].T / math.sqrt(d)).masked_fill_(hidden, -math.inf)
            o = torch.zeros(t * g, d, dtype=torch.float64, device="cuda")
            o[some] = torch.softmax(z[some], dim=1) @ v[h]
            out[b, :, h * g:(h + 1) * g] = o.view(t, g, d)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"product": _exact_product, "place": _exact_place, "rows": _exact_rows,
            "prompt": _exact_prompt, "tree": _exact_tree}[case["kind"]](st)
