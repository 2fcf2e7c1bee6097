"""The 8-bit paged KV cache's operators as cases that can be timed and checked.

Three operators, in their plain form (elementary torch operations) and as the
calls a user makes of this package:

  append   rotate the new keys and write keys and values into 8-bit pages,
           then read back the rows of every block that was written
  attend   attention of each sequence's new tokens over its pages: one token
           (decode), a few (verification of drafted tokens) or a whole prompt
  window   the same with a sliding window and first tokens that stay visible

A page holds 64 positions of every KV head, keys and values, as bytes
code + 128; a block of 16 positions of one head shares one f32 scale.  Inside
a block the bytes are in the order described in include/furnace.h; `tokens_of`
and `bytes_of` below turn them into [16, head_dim] and back.
"""

import math

import torch

own = False

PAGE, BLOCK = 64, 16
DTYPES = {"f32": torch.float32, "f16": torch.float16}


# ---------------------------------------------------------------------------
# Cases.  heads: query heads, kv: KV heads, hd: head dimension; n: sequences;
# new: the most new tokens of a sequence; hist: the most positions it held
# before; ragged: whether both vary from sequence to sequence.
# ---------------------------------------------------------------------------
def _case(op, heads, kv, hd, dtype, n, new, hist, ragged, window=0, sinks=0):
    return {"op": op, "heads": heads, "kv": kv, "hd": hd, "dtype": dtype, "n": n, "new": new, "hist": hist,
            "ragged": ragged, "window": window, "sinks": sinks}


def listed():
    cases = {
        # one token of one sequence, the 0.5B shape: nothing but latency
        "append one token": _case("append", 14, 2, 64, "f32", 1, 1, 700, False),
        # a decode step of a serving batch, 7B shape
        "append 64 sequences": _case("append", 28, 4, 128, "f16", 64, 1, 4000, True),
        # prompts of different lengths arriving together, 1.5B shape
        "append ragged prompts": _case("append", 12, 2, 128, "f16", 7, 1500, 90, True),
        # the 72B shape's prompt, starting in the middle of a block
        "append prompt 8192": _case("append", 64, 8, 128, "f32", 1, 8192, 103, False),
        # the first steps of an answer, 0.5B shape: latency
        "decode short": _case("attend", 14, 2, 64, "f32", 1, 1, 32, False),
        # the single-user decode loop of the 7B shape after its 2048-token prompt
        "decode one 7B": _case("attend", 28, 4, 128, "f32", 1, 1, 2560, False),
        # a serving batch of mixed lengths, 7B shape
        "decode 48 ragged": _case("attend", 28, 4, 128, "f16", 48, 1, 8191, True),
        # long contexts, 72B shape: 1 GB of cache
        "decode 16 long": _case("attend", 64, 8, 128, "f32", 16, 1, 32767, False),
        # drafted tokens verified together, 32B shape
        "verify 6 drafted": _case("attend", 40, 8, 128, "f16", 12, 6, 3000, True),
        # the 7B shape's 2048-token prompt behind a short cached prefix
        "prompt 2048": _case("attend", 28, 4, 128, "f32", 1, 2048, 100, False),
        # a windowed serving batch, 32B shape: few of the cached positions count
        "window decode 32": _case("window", 40, 8, 128, "f16", 32, 1, 20000, True, 4096, 4),
        # prompt pieces of long dialogues under a window, 1.5B shape
        "window prompts": _case("window", 12, 2, 128, "f32", 3, 700, 5000, True, 1024, 4),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "window"])
    hd, kv = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 6, 7, 8, 12])
    dtype, ragged = rng.choice(["f32", "f16"]), rng.random() < 0.7
    if op == "append":
        n = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, max(3, 8192 // n))
        hist = rng.randint(0, 4000)
    else:
        kind = rng.choice(["one", "one", "few", "prompt"])
        n = _log(rng, 1, 64) if kind != "prompt" else _log(rng, 1, 8)
        new = {"one": 1, "few": rng.randint(2, 12), "prompt": _log(rng, 20, max(40, 2048 // n))}[kind]
        # at most half of the largest listed case's cached positions x heads
        most = min(32767, (1 << 21) // (n * kv))
        hist = _log(rng, 1, most) if kind != "prompt" else _log(rng, 1, min(most, 4000))
    window = _log(rng, 16, 8000) if op == "window" else 0
    sinks = rng.choice([0, 1, 4, 5, 20, 100]) if op == "window" else 0
    return _case(op, group * kv, kv, hd, dtype, n, new, hist, ragged, window, sinks)


def _lengths(case):
    """(new tokens, positions held before) of each sequence: a function of the
    case alone, so that work() knows them too."""
    n, new, hist = case["n"], case["new"], case["hist"]
    if not case["ragged"]:
        return [new] * n, [hist] * n
    # a fixed spread over the ranges: the first sequence has the most of both
    spread = [((i * 7919 + 13) % 1009) / 1009 for i in range(n)]
    news = [new if i == 0 else max(1, int(new * (0.1 + 0.9 * spread[i]))) for i in range(n)]
    hists = [hist if i == 0 else int(hist * spread[(3 * i + 1) % n]) for i in range(n)]
    return news, hists


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kv, hd, heads, dtype = case["kv"], case["hd"], case["heads"], DTYPES[case["dtype"]]
    news, hists = _lengths(case)
    lens = [a + b for a, b in zip(news, hists)]
    need = [(x + PAGE - 1) // PAGE for x in lens]
    n_pages, max_pages = sum(need) + 3, max(need) + 1
    # pages in the order a free list hands them out after a while: any
    perm = torch.randperm(n_pages, device=dev, generator=gen).to(torch.int32)
    pages = torch.zeros(case["n"], max_pages, dtype=torch.int32, device=dev)
    at = 0
    for i, k in enumerate(need):
        pages[i, :k] = perm[at : at + k]
        at += k
    shape = (n_pages, kv, 2, PAGE * hd)
    codes = torch.randint(0, 128, shape, dtype=torch.uint8, device=dev, generator=gen)
    codes += torch.randint(1, 129, shape, dtype=torch.uint8, device=dev, generator=gen)
    # values near 1: the codes spread by 52 around 128
    scales = (torch.rand(n_pages, kv, 2, PAGE // BLOCK, device=dev, generator=gen) + 0.5) / 52
    rows = sum(news)
    q = torch.randn(rows, heads, hd, device=dev, generator=gen)
    k = torch.randn(rows, kv, hd, device=dev, generator=gen)
    v = torch.randn(rows, kv, hd, device=dev, generator=gen)
    # rotation factors of every position, as the cache of this package keeps them
    angle = torch.arange(max(lens), device=dev, dtype=torch.float64)[:, None] * (
        1e6 ** (-2.0 * torch.arange(hd // 2, device=dev, dtype=torch.float64) / hd))[None]
    rope = torch.stack([angle.cos(), angle.sin()], -1).to(torch.float32).contiguous()
    # rows read back after an append: from the start of the first block written
    back = [min(x, x - h // BLOCK * BLOCK) for x, h in zip(lens, hists)]

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    def starts(x):
        return ints([sum(x[:i]) for i in range(len(x) + 1)])

    state = {
        "case": case, "pages": pages, "codes": codes, "scales": scales, "rope": rope, "lens": ints(lens),
        "starts": starts(news), "back": starts(back), "max_new": max(news), "max_back": max(back), "rows": rows,
        "back_rows": sum(back), "n_pages": n_pages, "max_pages": max_pages, "max_len": max(lens),
        "q": q.to(dtype), "k": k.to(dtype), "v": v.to(dtype), "status": torch.zeros(1, dtype=torch.int32, device=dev),
    }
    if case["op"] == "append":
        state["k_out"] = torch.zeros(sum(back), kv, hd, dtype=torch.float16, device=dev)
        state["v_out"] = torch.zeros_like(state["k_out"])
    else:
        state["out"] = torch.zeros(rows, heads, hd, dtype=dtype, device=dev)
    if own:
        _handles(state)
    return state


def _handles(s):
    """The descriptors and the workspace a program makes once."""
    import furnace_b200 as fz

    c = s["case"]
    s["cache"] = fz.KvQ8(s["codes"].data_ptr(), s["scales"].data_ptr(), s["status"].data_ptr(), s["n_pages"],
                         c["heads"], c["kv"], c["hd"], rope=s["rope"].data_ptr(), n_rope=s["rope"].shape[0])
    one = s["max_new"] == 1
    s["seqs"] = fz.KvQ8Seqs(s["pages"].data_ptr(), s["lens"].data_ptr(), c["n"], s["max_pages"], s["rows"],
                            starts=None if one else s["starts"].data_ptr(), max_new=s["max_new"])
    s["dt"] = {"f32": fz.F32, "f16": fz.F16}[c["dtype"]]
    if c["op"] == "append":
        s["seqs_back"] = fz.KvQ8Seqs(s["pages"].data_ptr(), s["lens"].data_ptr(), c["n"], s["max_pages"],
                                     s["back_rows"], starts=s["back"].data_ptr(), max_new=s["max_back"])
        s["dt_out"] = fz.F16
    else:
        s["work"] = torch.empty(s["cache"].attend_work(s["seqs"]), dtype=torch.uint8, device=s["codes"].device)


def run(state):
    if own:
        return _run_own(state)
    return _append(state) if state["case"]["op"] == "append" else _attend(state)


def _run_own(s):
    c, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        ld = c["kv"] * c["hd"]
        s["cache"].append(s["seqs"], s["k"].data_ptr(), s["v"].data_ptr(), ld, dtype=s["dt"], stream=stream)
        s["cache"].read(s["seqs_back"], s["k_out"].data_ptr(), s["v_out"].data_ptr(), ld, dtype=s["dt_out"],
                        stream=stream)
        return {"k": s["k_out"], "v": s["v_out"], "scales": s["scales"]}
    ld = c["heads"] * c["hd"]
    s["cache"].attend(s["seqs"], s["q"].data_ptr(), s["out"].data_ptr(), ld, ld, s["work"].data_ptr(),
                      s["work"].numel(), dtype=s["dt"], window=c["window"], sinks=c["sinks"], stream=stream)
    return s["out"]


# ---------------------------------------------------------------------------
# Plain form
# ---------------------------------------------------------------------------
def tokens_of(block, hd, values):
    """[..., 16 * hd] bytes of a block as [..., 16, hd] (values: of V, else of K)."""
    lead = block.shape[:-1]
    d = len(lead)
    keep = list(range(d))
    if values:  # [32 dims][dim % 8][token pair][dim / 8][half][parity]
        x = block.reshape(*lead, hd // 32, 8, 4, 4, 2, 2)
        x = x.permute(*keep, d + 4, d + 2, d + 5, d, d + 3, d + 1)
    else:  # [8 tokens][64 dims][token][16 dims][dim]
        x = block.reshape(*lead, 2, hd // 64, 8, 4, 16)
        x = x.permute(*keep, d, d + 2, d + 1, d + 3, d + 4)
    return x.reshape(*lead, BLOCK, hd)


def bytes_of(tokens, hd, values):
    """The inverse of tokens_of."""
    lead = tokens.shape[:-2]
    d = len(lead)
    keep = list(range(d))
    if values:
        x = tokens.reshape(*lead, 2, 4, 2, hd // 32, 4, 8)
        x = x.permute(*keep, d + 3, d + 5, d + 1, d + 4, d, d + 2)
    else:
        x = tokens.reshape(*lead, 2, 8, hd // 64, 4, 16)
        x = x.permute(*keep, d, d + 2, d + 1, d + 3, d + 4)
    return x.reshape(*lead, BLOCK * hd)


def _rotate(x, rope):
    """x [rows, heads, hd] rotated by rope [rows, hd / 2, 2] (pairs half a head
    apart); each product rounded by itself."""
    a, b = x.float().chunk(2, -1)
    c, s = rope[:, None, :, 0], rope[:, None, :, 1]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _row_index(starts, lens, rows):
    """Sequence and position of every row."""
    row = torch.arange(rows, device=starts.device)
    seq = torch.searchsorted(starts[1:].long(), row, right=True)
    return seq, lens.long()[seq] - (starts.long()[seq + 1] - row)


def _append(s):
    c, dev = s["case"], s["codes"].device
    hd, kv, n = c["hd"], c["kv"], c["n"]
    seq, pos = _row_index(s["starts"], s["lens"], s["rows"])
    k = _rotate(s["k"], s["rope"][pos])
    new = torch.stack([k, s["v"].float()], 2)  # [rows, kv, 2, hd]
    # the blocks written, as [sequence, block] with each sequence's first block at 0
    count = s["starts"].long().diff()
    first = (s["lens"].long() - count) // BLOCK
    nb = (s["max_new"] + 2 * BLOCK - 2) // BLOCK
    blk = first[:, None] + torch.arange(nb, device=dev)
    live = (blk * BLOCK < s["lens"].long()[:, None]) & (count[:, None] > 0)
    at = torch.zeros(n, nb, BLOCK, kv, 2, hd, device=dev)
    slot = pos - first[seq] * BLOCK
    at[seq, slot // BLOCK, slot % BLOCK] = new
    amax = at.abs().amax(dim=(2, 5))  # [n, nb, kv, 2]; unwritten slots are zero
    page = s["pages"].long()[torch.arange(n, device=dev)[:, None], torch.where(live, blk * BLOCK // PAGE, 0)]
    sub = blk % (PAGE // BLOCK)
    codes = s["codes"].view(s["n_pages"], kv, 2, PAGE // BLOCK, BLOCK * hd)
    si, bi = live.nonzero(as_tuple=True)
    pg, sb = page[si, bi], sub[si, bi]
    old_scale = s["scales"][pg, :, :, sb]  # [live blocks, kv, 2]
    n_old = ((s["lens"].long() - count)[si] - blk[si, bi] * BLOCK).clamp(0, BLOCK)
    fresh = (n_old == 0)[:, None, None]
    scale = amax[si, bi] / 127
    scale = torch.where(fresh, scale, torch.maximum(scale, old_scale))
    ratio = torch.where(scale > 0, old_scale / scale, torch.zeros_like(scale))
    raw = codes[pg, :, :, sb]  # [live, kv, 2, 16 * hd]
    old = torch.stack([tokens_of(raw[:, :, 0], hd, False), tokens_of(raw[:, :, 1], hd, True)], 2)
    here = torch.arange(BLOCK, device=dev)[None, :] + (blk[si, bi] * BLOCK)[:, None]
    is_old = here < (s["lens"].long() - count)[si][:, None]
    is_new = ~is_old & (here < s["lens"].long()[si][:, None])
    oldq = old.float() - 128  # [live, kv, 2, 16, hd]
    grew = (scale > old_scale)[..., None, None]
    oldq = torch.where(grew, torch.round(oldq * ratio[..., None, None]), oldq)
    x = at[si, bi].permute(0, 2, 3, 1, 4)  # [live, kv, 2, 16, hd]
    sc = scale[..., None, None]
    newq = torch.where(sc > 0, torch.round(x / sc).clamp(-127, 127), torch.zeros_like(x))
    is_old, is_new = is_old[:, None, None, :, None], is_new[:, None, None, :, None]
    byte = torch.where(is_new, newq + 128, torch.where(is_old, oldq + 128, old.float())).to(torch.uint8)
    codes[pg, :, :, sb] = torch.stack([bytes_of(byte[:, :, 0], hd, False), bytes_of(byte[:, :, 1], hd, True)], 2)
    s["scales"][pg, :, :, sb] = scale
    # the rows of the written blocks as the cache holds them
    seq, pos = _row_index(s["back"], s["lens"], s["back_rows"])
    pg, sb = s["pages"].long()[seq, pos // PAGE], pos // BLOCK % (PAGE // BLOCK)
    block = (pos // BLOCK - first[seq])
    inverse = torch.zeros(n, nb, dtype=torch.long, device=dev)
    inverse[si, bi] = torch.arange(si.numel(), device=dev)
    held = (byte.float() - 128)[inverse[seq, block], :, :, pos % BLOCK]  # [back rows, kv, 2, hd]
    held = (held * s["scales"][pg, :, :, sb][..., None]).to(torch.float16)
    s["k_out"].copy_(held[:, :, 0])
    s["v_out"].copy_(held[:, :, 1])
    return {"k": s["k_out"], "v": s["v_out"], "scales": s["scales"]}


def _attend(s):
    c, dev = s["case"], s["codes"].device
    hd, kv, heads, n = c["hd"], c["kv"], c["heads"], c["n"]
    group, used = heads // kv, (s["max_len"] + PAGE - 1) // PAGE
    table = s["pages"].long()[:, :used]
    raw = s["codes"].view(s["n_pages"], kv, 2, PAGE // BLOCK, BLOCK * hd)[table]
    sc = s["scales"][table]  # [n, pages, kv, 2, 4]

    def side(which):
        x = tokens_of(raw[:, :, :, which], hd, which == 1).float() - 128  # [n, pages, kv, 4, 16, hd]
        x *= sc[:, :, :, which, :, None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(n, kv, used * PAGE, hd)

    keys, values = side(0), side(1)
    seq, pos = _row_index(s["starts"], s["lens"], s["rows"])
    q = _rotate(s["q"], s["rope"][pos])
    # rows padded to [n, max_new]
    slot = torch.arange(s["rows"], device=dev) - s["starts"].long()[seq]
    qp = torch.zeros(n, s["max_new"], heads, hd, device=dev)
    qp[seq, slot] = q
    limit = torch.full((n, s["max_new"]), -1, dtype=torch.long, device=dev)
    limit[seq, slot] = pos
    qp = qp.reshape(n, s["max_new"], kv, group, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, s["max_new"] * group, hd)
    score = (qp @ keys.transpose(-1, -2)) / math.sqrt(hd)
    t = torch.arange(used * PAGE, device=dev)[None, None, :]
    seen = t <= limit[:, :, None]
    if c["window"]:
        seen &= (t > limit[:, :, None] - c["window"]) | (t < c["sinks"])
    seen = seen.repeat_interleave(group, 1)[:, None]
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(score - top)
    out = (p @ values) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = out.reshape(n, kv, s["max_new"], group, hd).permute(0, 2, 1, 3, 4).reshape(n, s["max_new"], heads, hd)
    s["out"].copy_(out[seq, slot])
    return s["out"]


# ---------------------------------------------------------------------------
# The definition in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------
def _page_codes(s, i, upto):
    """Sequence i's codes as [2, kv, positions, hd] and scales as [2, kv, positions], in 64 bits."""
    c = s["case"]
    hd, kv = c["hd"], c["kv"]
    table = s["pages"][i, : (upto + PAGE - 1) // PAGE].long()
    raw = s["codes"][table].view(-1, kv, 2, PAGE // BLOCK, BLOCK * hd)
    tok, dim = torch.meshgrid(torch.arange(BLOCK), torch.arange(hd), indexing="ij")
    at_k = (tok // 8) * 8 * hd + (dim // 64) * 512 + (tok % 8) * 64 + dim % 64
    at_v = (dim // 32) * 512 + (dim % 8) * 64 + (tok % 8 // 2) * 16 + (dim % 32 // 8) * 4 + (tok // 8) * 2 + tok % 2
    out = []
    for which, at in ((0, at_k), (1, at_v)):
        x = raw[:, :, which][..., at.to(raw.device)].double() - 128  # [pages, kv, 4, 16, hd]
        out.append(x.permute(1, 0, 2, 3, 4).reshape(kv, -1, hd))
    sc = s["scales"][table].double().permute(2, 1, 0, 3).reshape(2, kv, -1)
    return torch.stack(out), sc.repeat_interleave(BLOCK, -1)


def _turn(x, rope):
    x, rope = x.double(), rope.double()
    h = x.shape[-1] // 2
    turned = torch.view_as_complex(torch.stack([x[..., :h], x[..., h:]], -1)) * torch.view_as_complex(
        rope.contiguous())[:, None]
    return torch.cat([turned.real, turned.imag], -1)


def exact(case, seed):
    s = prepare(case, seed)
    news, hists = _lengths(case)
    group = case["heads"] // case["kv"]
    if case["op"] == "append":
        scales, ks, vs = s["scales"].double(), [], []
        row = 0
        for i, (new, hist) in enumerate(zip(news, hists)):
            lo, end = hist // BLOCK * BLOCK, hist + new
            codes, sc = _page_codes(s, i, end)
            k = _turn(s["k"][row : row + new], s["rope"][hist:end])
            fresh = torch.stack([k, s["v"][row : row + new].double()]).transpose(1, 2)  # [2, kv, new, hd]
            row += new
            pad = -end % BLOCK
            x = torch.nn.functional.pad(fresh, (0, 0, hist - lo, pad))  # whole blocks
            x = x.reshape(2, case["kv"], -1, BLOCK, case["hd"])
            top = x.abs().amax((-1, -2)) / 127
            before = sc[:, :, lo : end + pad : BLOCK]
            if hist > lo:
                top[:, :, 0] = torch.maximum(top[:, :, 0], before[:, :, 0])
            q = torch.round(x / top[..., None, None]).clamp(-127, 127).reshape(2, case["kv"], -1, case["hd"])
            if hist > lo:  # positions that were there keep their codes, or take those of the larger scale
                held = codes[:, :, lo:hist]
                q[:, :, : hist - lo] = torch.round(held * (before[:, :, :1] / top[:, :, :1])[..., None])
            for b in range(top.shape[2]):
                p = lo + b * BLOCK
                scales[s["pages"][i, p // PAGE].long(), :, :, p // BLOCK % (PAGE // BLOCK)] = top[:, :, b].T
            held = (q * top.repeat_interleave(BLOCK, -1)[..., None])[:, :, : end - lo].transpose(1, 2)
            ks.append(held[0])
            vs.append(held[1])
        return {"k": torch.cat(ks), "v": torch.cat(vs), "scales": scales}
    out, row = [], 0
    for i, (new, hist) in enumerate(zip(news, hists)):
        end = hist + new
        codes, sc = _page_codes(s, i, end)
        held = codes[:, :, :end] * sc[:, :, :end, None]
        pos = torch.arange(hist, end, device=codes.device)
        q = _turn(s["q"][row : row + new], s["rope"][hist:end]).reshape(new, case["kv"], group, case["hd"])
        row += new
        t = torch.arange(end, device=codes.device)
        seen = t[None] <= pos[:, None]
        if case["window"]:
            seen &= (t[None] > pos[:, None] - case["window"]) | (t[None] < case["sinks"])
        heads = []
        for h in range(case["kv"]):
            score = torch.einsum("ngd,td->ngt", q[:, h], held[0, h]) * case["hd"] ** -0.5
            p = torch.softmax(score.masked_fill(~seen[:, None], float("-inf")), -1)
            heads.append(torch.einsum("ngt,td->ngd", p, held[1, h]))
        out.append(torch.stack(heads, 1).reshape(new, case["heads"], case["hd"]))
    return torch.cat(out)


def work(case):
    news, hists = _lengths(case)
    kv, hd, heads = case["kv"], case["hd"], case["heads"]
    size = 4 if case["dtype"] == "f32" else 2
    rows, scale_bytes = sum(news), 8 / BLOCK
    if case["op"] == "append":
        back = sum(h % BLOCK + n for n, h in zip(news, hists))
        held = sum(h % BLOCK for h in hists)
        # new keys and values and their rotation factors in, the blocks' older bytes in; codes, scales and the rows read back out
        per = kv * (2 * hd)
        return {"bytes": rows * (per * size + hd * 4) + held * per + back * (per * 1 + per * 2 + kv * scale_bytes),
                "flops": rows * kv * hd * 6}
    read = seen = 0
    for n, h in zip(news, hists):
        end, window, sinks = h + n, case["window"], case["sinks"]
        if window:
            lo = max(0, h + 1 - window)
            read += end - lo + min(sinks, lo)
            seen += sum(min(p + 1, window + min(sinks, max(0, p + 1 - window))) for p in range(h, end))
        else:
            read += end
            seen += n * h + n * (n + 1) // 2
    return {"bytes": read * kv * (2 * hd + scale_bytes) + rows * (heads * hd * 2 * size + hd * 4),
            "flops": 4 * hd * heads * seen}
