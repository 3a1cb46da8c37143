"""Cases of the paged latent cache, the attention over it and the token log probabilities.

Each case is one call (or the pair of calls) that a server makes between the framework's decode
steps: attention of new tokens over latents held in pages, page bookkeeping of admitted, forked and
finished sequences, and the scores of given tokens. `run` computes it in plain torch operations, or
with the framework's operators where `own` is true; `exact` computes it in 64 bits.

The latent row is the framework's: 448 E4M3 codes with one E8M0 scale per 64, and 64 BF16 RoPE
values; K and V are the same row, shared by all heads.
"""
import math
import os
import random
import sys

import torch

own = False

NOPE, ROPE, DIM = 448, 64, 512
ROW_BYTES = 584  # codes, 8 scale slots, RoPE values
VOCAB = 129280


def _binding():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "deepseek-v4-flash-0731-in-c_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import dsv4cuda
    return dsv4cuda


def listed():
    return [
        # one sequence's decode step at the benchmark's 2,048-token context: latency
        dict(name="attn_token", op="attn", heads=64, seqs=1, new=1, len=2048, ragged=False,
             window=0, page=64, freed=False),
        # a decode step of a batch of sequences of many lengths
        dict(name="attn_decode_batch", op="attn", heads=64, seqs=32, new=1, len=8192, ragged=True,
             window=0, page=64, freed=False),
        # speculative verify: the pending token and up to 5 drafts of each sequence, 128 heads,
        # pages that end inside a tile
        dict(name="attn_verify", op="attn", heads=128, seqs=8, new=6, len=4001, ragged=True,
             window=0, page=48, freed=False),
        # prompts through a sliding-window layer (window 128), pages before the window given back
        dict(name="attn_window_prefill", op="attn", heads=64, seqs=4, new=1000, len=3000,
             ragged=True, window=128, page=64, freed=True),
        # a prompt's last chunk of 2,048 tokens on top of what is already cached
        dict(name="attn_chunk", op="attn", heads=64, seqs=1, new=2048, len=11987, ragged=False,
             window=0, page=64, freed=False),
        # two samples forked off one prompt, two layers: latency
        dict(name="fork_few", op="fork", layers=2, page=64, pages=256, seqs=8, len=700, ops=2),
        # many samples per prompt through all 43 layers, finished ones replaced
        dict(name="fork_many", op="fork", layers=43, page=64, pages=768, seqs=96, len=900, ops=64),
        # a fragmented pool made dense before it is shrunk, all 43 layers
        dict(name="compact", op="compact", layers=43, page=64, pages=768, seqs=48, len=1400, ops=0),
        # finished sequences released and new prompts admitted in a large pool
        dict(name="admit", op="admit", layers=1, page=16, pages=16384, seqs=256, len=2000, ops=48),
        # the decode step's token with its 20 alternatives
        dict(name="logprob_token", op="logprob", rows=1, vocab=VOCAB, top=20, dtype="f32", pad=0,
             masked=0.0),
        # verify rows of a batch under a constraint that masks most of the vocabulary
        dict(name="logprob_masked", op="logprob", rows=48, vocab=VOCAB, top=5, dtype="bf16", pad=37,
             masked=0.9),
        # every token of a prompt scored
        dict(name="logprob_prompt", op="logprob", rows=2048, vocab=VOCAB, top=8, dtype="f32", pad=0,
             masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "pages", "pages", "logprob"])
    if op == "attn":
        limit = _attn_flops(listed()[4])
        while True:
            window = rng.choice([0, 0, 128, rng.randint(1, 700)])
            c = dict(op="attn", heads=rng.choice([64, 128, 64, 16, rng.randint(1, 128)]),
                     seqs=_log_int(rng, 1, 64), new=rng.choice([1, _log_int(rng, 2, 8),
                                                                _log_int(rng, 9, 2048)]),
                     len=_log_int(rng, 1, 16384), ragged=rng.random() < 0.7, window=window,
                     page=rng.choice([64, 16, 128, rng.randint(1, 200)]),
                     freed=window > 0 and rng.random() < 0.5)
            spans = [b - a for a, b in (_span(c, n, L) for n, L in _lens(c))]
            news = [n for n, _ in _lens(c)]
            if (_attn_flops(c) <= limit
                    and c["seqs"] * max(news) * c["heads"] * max(spans) <= 1 << 31):
                return c
    if op == "pages":
        kind = rng.choice(["fork", "compact", "admit"])
        page = rng.choice([16, 64, rng.randint(2, 100)])
        seqs = _log_int(rng, 4, 128)
        length = _log_int(rng, 20, 3000)
        layers = 1 if kind == "admit" else _log_int(rng, 1, 43)
        room = 43 * 768 * 64 // (layers * page)
        most = max(2, min(room // (-(-length // page) + 1), seqs))
        seqs = max(2, most // 2 * 2)
        return dict(op=kind, layers=layers, page=page,
                    pages=seqs * (-(-length // page) + 1) + rng.randint(1, 200) if kind == "admit"
                    else min(room + 8, seqs * (-(-length // page) + 1) + rng.randint(1, 40)),
                    seqs=seqs, len=length, ops=max(1, rng.randint(1, seqs // 2)))
    vocab = rng.choice([VOCAB, VOCAB, _log_int(rng, 40, 300000)])
    rows = _log_int(rng, 1, max(1, min(4096, 2048 * VOCAB // vocab)))
    return dict(op="logprob", rows=rows, vocab=vocab, top=rng.randint(0, 32),
                dtype=rng.choice(["f32", "bf16"]), pad=rng.choice([0, rng.randint(1, 64)]),
                masked=rng.choice([0.0, 0.0, 0.3, 0.95]))


# ------------------------------------------------------------------ sizes --


def _lens(c):
    """(new tokens, length with them) of each sequence of an attention case."""
    r = random.Random("%d %d %d %d" % (c["seqs"], c["new"], c["len"], c["heads"]))
    out = []
    for i in range(c["seqs"]):
        length = c["len"] if not c["ragged"] or i == 0 else max(1, int(c["len"] * r.uniform(0.04, 1)))
        new = c["new"] if not c["ragged"] or i == 0 else max(1, int(c["new"] * r.uniform(0.1, 1) + 0.5))
        out.append((min(new, length), length))
    return out


def _span(c, n, length):
    """Positions that any of the sequence's new tokens sees."""
    first = length - n
    return (max(0, first - c["window"] + 1) if c["window"] else 0), length


def _attn_flops(c):
    seen = 0
    for n, length in _lens(c):
        for p in range(length - n, length):
            seen += min(p + 1, c["window"]) if c["window"] else p + 1
    return 4 * DIM * c["heads"] * seen


def _admit_counts(c):
    """Token counts of the prompts that an "admit" case brings in, one per op."""
    r = random.Random("%d %d %d" % (c["seqs"], c["len"], c["ops"]))
    return [max(1, int(c["len"] * r.uniform(0.1, 1))) for _ in range(c["ops"])]


def _page_state(c):
    """Tables, lengths and reference counts (lists) of a "fork", "compact" or "admit" case, the same
    for every seed, and the ops' destinations and sources.

    The first half of the slots are prompts; the others hold samples that share their prompt's full
    pages and own a copy of its partial one, as earlier forks left them."""
    r = random.Random("%d %d %d %d" % (c["pages"], c["seqs"], c["len"], c["page"]))
    page, half = c["page"], max(1, c["seqs"] // 2)
    free = list(range(c["pages"]))
    r.shuffle(free)
    rows, lens, refs = [], [], [0] * c["pages"]
    for s in range(c["seqs"]):
        if s < half:
            length = max(1, int(c["len"] * r.uniform(0.2, 1)))
            want = -(-length // page)
            if want + c["ops"] > len(free):  # the ops may need a page each on top
                length, want = 0, 0
            row = [free.pop() for _ in range(want)]
        else:
            p = r.randrange(half)
            length = lens[p]
            row = rows[p][:length // page]
            if length % page:
                if len(free) > c["ops"]:
                    row = row + [free.pop()]
                else:
                    length, row = 0, []
        for q in row:
            refs[q] += 1
        rows.append(row)
        lens.append(length)
    width = -(-c["len"] // page) + 1
    if c["op"] == "compact":
        for s in range(0, c["seqs"], 3):  # a third of the sequences have finished
            for q in rows[s]:
                refs[q] -= 1
            rows[s], lens[s] = [], 0
    table = [row + [-1] * (width - len(row)) for row in rows]
    dst = list(range(half, c["seqs"]))
    r.shuffle(dst)
    dst = dst[:c["ops"]]
    # one in sixteen has finished and is only given back
    src = [-1 if i % 16 == 15 or c["op"] == "admit" else r.randrange(half) for i in range(len(dst))]
    return table, lens, refs, dst, src


def work(c):
    if c["op"] == "attn":
        keys = sum(b - a for a, b in (_span(c, n, L) for n, L in _lens(c)))
        new = sum(n for n, _ in _lens(c))
        return {"bytes": keys * ROW_BYTES + new * (c["heads"] * (2 * 2 * DIM + 4) + 4 * ROPE)
                + 4 * (keys // c["page"] + c["seqs"]),
                "flops": _attn_flops(c)}
    if c["op"] == "logprob":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["rows"] * (c["vocab"] * size + 4 * 4 + 8 * c["top"]),
                "flops": 4 * c["rows"] * c["vocab"]}
    table, lens, refs, dst, src = _page_state(c)
    held = sum(q >= 0 for row in table for q in row)
    if c["op"] == "compact":
        live = sum(x > 0 for x in refs)
        moves = sum(x > 0 for x in refs[live:])
        return {"bytes": 2 * moves * c["page"] * c["layers"] * ROW_BYTES + 8 * len(refs) + 8 * held,
                "flops": 0}
    if c["op"] == "admit":
        return {"bytes": 4 * len(refs) + 8 * sum(_admit_counts(c)[:len(dst)])
                + 8 * sum(len(table[d]) for d in dst), "flops": 0}
    rows = sum(lens[s] % c["page"] for s in src if s >= 0)
    return {"bytes": 2 * rows * c["layers"] * ROW_BYTES + 4 * len(refs)
            + 12 * sum(len(table[d]) for d in dst), "flops": 0}


# ----------------------------------------------------------------- inputs --


def _latents(shape, g):
    """Random cache contents: codes, scales, RoPE values of `shape` rows."""
    codes = torch.empty(*shape, NOPE, dtype=torch.uint8, device="cuda")
    rope = torch.empty(*shape, ROPE, dtype=torch.bfloat16, device="cuda")
    scales = torch.randint(119, 123, (*shape, 8), dtype=torch.uint8, device="cuda", generator=g)
    flat, frope = codes.view(-1, NOPE), rope.view(-1, ROPE)
    step = 1 << 18
    for i in range(0, flat.shape[0], step):
        x = torch.randn(flat[i:i + step].shape, device="cuda", generator=g) * 100
        flat[i:i + step] = x.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        frope[i:i + step] = torch.randn(frope[i:i + step].shape, device="cuda", generator=g)
    return codes, scales, rope


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "logprob":
        width = c["vocab"] + c["pad"]
        dtype = torch.float32 if c["dtype"] == "f32" else torch.bfloat16
        x = torch.empty(c["rows"], width, dtype=dtype, device="cuda")
        for i in range(0, c["rows"], 256):
            y = torch.randn(x[i:i + 256].shape, device="cuda", generator=g) * 2.5
            if c["masked"]:
                hide = torch.rand(y.shape, device="cuda", generator=g) < c["masked"]
                y = torch.where(hide, -math.inf, y)
            x[i:i + 256] = y
        x[:, c["vocab"]:] = 1e30  # what lies behind a row is not the row's
        tokens = torch.randint(0, c["vocab"], (c["rows"],), device="cuda", generator=g,
                               dtype=torch.int32)
        likely = torch.rand(c["rows"], device="cuda", generator=g) < 0.5
        tokens = torch.where(likely, x[:, :c["vocab"]].max(dim=1).indices.int(), tokens)
        tokens[7::16] = -1  # padding: no token is asked for
        f32 = dict(dtype=torch.float32, device="cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        s.update(logits=x[:, :c["vocab"]], tokens=tokens, logprob=torch.empty(c["rows"], **f32),
                 entropy=torch.empty(c["rows"], **f32), rank=torch.empty(c["rows"], **i32),
                 top_id=torch.empty(c["rows"], c["top"], **i32),
                 top_logprob=torch.empty(c["rows"], c["top"], **f32))
        if own:
            s["lib"] = _binding()
        return s
    if c["op"] == "attn":
        lens = _lens(c)
        spans = [_span(c, n, L) for n, L in lens]
        held = [-(-L // c["page"]) for _, L in lens]
        gone = [a // c["page"] if c["freed"] else 0 for a, _ in spans]
        pages = sum(held) - sum(gone) + 3
        width = max(held) + 1
        order = torch.randperm(pages, device="cuda", generator=g).tolist()
        table = []
        for h, b in zip(held, gone):
            table.append([-1] * b + [order.pop() for _ in range(h - b)] + [-1] * (width - h))
        total = sum(n for n, _ in lens)
        pos = torch.cat([torch.arange(L - n, L) for n, L in lens]).cuda()
        freq = 10000.0 ** (-torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float64) / ROPE)
        angle = pos[:, None].double() * freq[None]
        bf = dict(dtype=torch.bfloat16, device="cuda")
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        codes, scales, rope = _latents((1, pages * c["page"]), g)
        refs = [0] * pages
        for row in table:
            for q in row:
                if q >= 0:
                    refs[q] += 1
        s.update(codes=codes, scales=scales, rope=rope, table=_ints(table),
                 length=_ints([L for _, L in lens]), refs=_ints(refs), q_start=_ints(starts),
                 q=torch.randn(total, c["heads"], DIM, device="cuda", generator=g).bfloat16() * 1.5,
                 sink=torch.randn(c["heads"], device="cuda", generator=g),
                 cos=angle.cos().float(), sin=angle.sin().float(),
                 out=torch.empty(total, c["heads"], DIM, **bf),
                 lse=torch.empty(total, c["heads"], dtype=torch.float32, device="cuda"),
                 max_new=max(n for n, _ in lens), max_len=max(L for _, L in lens),
                 max_keys=sum(b - a for a, b in spans))
    else:
        table, lens, refs, dst, src = _page_state(c)
        # which pages hold what is the seed's; how many lie beyond the live count (what compaction
        # moves) is not
        live = sum(x > 0 for x in refs)
        to = torch.randperm(live, device="cuda", generator=g).tolist()
        to += [live + i for i in
               torch.randperm(c["pages"] - live, device="cuda", generator=g).tolist()]
        table = [[to[q] if q >= 0 else -1 for q in row] for row in table]
        moved = [0] * len(refs)
        for i, x in enumerate(refs):
            moved[to[i]] = x
        refs = moved
        codes, scales, rope = _latents((c["layers"], c["pages"] * c["page"]), g)
        # who forks from whom is the seed's; how many rows that copies is not
        if c["op"] == "fork":
            turn = torch.randperm(len(dst), device="cuda", generator=g).tolist()
            src = [src[i] for i in turn]
        elif c["op"] == "admit":
            turn = torch.randperm(len(dst), device="cuda", generator=g).tolist()
            dst = [dst[i] for i in turn]
        s.update(codes=codes, scales=scales, rope=rope, table=_ints(table), length=_ints(lens),
                 refs=_ints(refs), dst=_ints(dst), src=_ints(src))
        if c["op"] == "admit":
            counts = _admit_counts(c)[:len(dst)]
            s.update(counts=_ints(counts),
                     rows=torch.empty(sum(counts), dtype=torch.int64, device="cuda"))
        if c["op"] == "compact":
            s.update(table_out=torch.empty_like(s["table"]), refs_out=torch.empty_like(s["refs"]))
    if own:
        lib = _binding()
        caches = [lib.LatentCache.from_tensors(s["codes"][i], s["scales"][i],
                                               s["rope"][i].view(torch.int16))
                  for i in range(s["codes"].shape[0])]
        s["paged"] = lib.PagedCache(caches, c["page"], s["table"], s["length"], s["refs"])
        s["lib"] = lib
    return s


# ------------------------------------------------------------ one pass --


def run(s):
    op = s["case"]["op"]
    if op == "attn":
        if own:
            s["lib"].paged_attn(s["out"], s["q"], s["paged"], 0, s["q_start"], s["max_new"],
                                s["max_len"], DIM ** -0.5, sink=s["sink"],
                                window=s["case"]["window"], rope_cos=s["cos"], rope_sin=s["sin"],
                                lse=s["lse"], max_keys=s["max_keys"])
            return s["out"], s["lse"]
        return _attn_plain(s, torch.float32)
    if op == "logprob":
        if own:
            s["lib"].token_logprobs(s["logits"], s["tokens"], s["logprob"], s["entropy"], s["rank"],
                                    s["top_id"], s["top_logprob"])
            return s["logprob"], s["entropy"], s["rank"], s["top_id"], s["top_logprob"]
        return _logprob_plain(s["logits"].float(), s["tokens"], s["case"]["top"])
    if op == "admit":
        # finished sequences given back, then the new prompts' pages taken
        if own:
            s["paged"].fork(s["dst"], s["src"])
            s["paged"].append(s["dst"], s["counts"], s["rows"])
        else:
            _fork_plain(s)
            _append_plain(s)
        return s["table"], s["length"], s["refs"], s["rows"]
    if op == "fork":
        if own:
            s["paged"].fork(s["dst"], s["src"])
        else:
            _fork_plain(s)
        return (s["table"], s["length"], s["refs"]) + _contents(s)
    # the tables before the move stay as they are (steps in flight read them), so that the pass can
    # be made again
    if own:
        s["paged"].compact(s["table_out"], s["refs_out"])
    else:
        _compact_plain(s)
    return (s["table_out"], s["refs_out"]) + _contents(s)


def _contents(s):
    return s["codes"].view(torch.float8_e4m3fn), s["scales"], s["rope"]


def _attn_plain(s, dtype):
    """All sequences padded to the longest: scores, masked softmax with the sink, values, inverse RoPE."""
    c = s["case"]
    q_start, length = s["q_start"].long(), s["length"].long()
    new = q_start[1:] - q_start[:-1]
    first = length - new
    low = (first - c["window"] + 1).clamp(min=0) if c["window"] else torch.zeros_like(first)
    n_max, k_max = s["max_new"], max(b - a for a, b in (_span(c, n, L) for n, L in _lens(c)))
    # keys of each sequence from its first visible position on
    pos = low[:, None] + torch.arange(k_max, device="cuda")[None]
    page = torch.gather(s["table"].long(), 1, (pos // c["page"]).clamp(max=s["table"].shape[1] - 1))
    there = (pos < length[:, None]) & (page >= 0)
    row = torch.where(there, page * c["page"] + pos % c["page"], 0)
    scale = torch.exp2(s["scales"][0][row][..., :NOPE // 64].to(dtype) - 127)
    codes = s["codes"].view(torch.float8_e4m3fn)[0][row].to(dtype)
    k = torch.cat([codes * scale.repeat_interleave(64, dim=-1), s["rope"][0][row].to(dtype)], dim=-1)
    # queries of each sequence
    i = torch.arange(n_max, device="cuda")
    mine = i[None] < new[:, None]
    at = torch.where(mine, q_start[:-1, None] + i[None], 0)
    q = s["q"][at].to(dtype).flatten(1, 2)
    x = torch.matmul(q, k.transpose(1, 2)) * DIM ** -0.5
    x = x.view(len(new), n_max, c["heads"], k_max)
    p = (first[:, None] + i[None])[:, :, None]
    seen = there[:, None, :] & (pos[:, None, :] <= p)
    if c["window"]:
        seen = seen & (pos[:, None, :] > p - c["window"])
    x = x.masked_fill_(~seen[:, :, None, :], -math.inf)
    sink = s["sink"].to(dtype)[None, None, :, None]
    m = torch.maximum(x.amax(dim=-1, keepdim=True), sink)
    e = torch.exp(x.sub_(m))
    den = e.sum(dim=-1, keepdim=True) + torch.exp(sink - m)
    o = torch.matmul(e.flatten(1, 2), k).view(len(new), n_max, c["heads"], DIM) / den
    o, lse = o[mine], (m + torch.log(den))[..., 0][mine]
    a, b = o[..., NOPE::2].clone(), o[..., NOPE + 1::2].clone()
    cos, sin = s["cos"].to(dtype)[:, None], s["sin"].to(dtype)[:, None]
    o[..., NOPE::2] = a * cos + b * sin
    o[..., NOPE + 1::2] = b * cos - a * sin
    return (o.bfloat16(), lse) if dtype == torch.float32 else (o, lse)


def _logprob_plain(x, tokens, top):
    t = tokens.long()
    asked = (t >= 0) & (t < x.shape[1])
    t = torch.where(asked, t, 0)
    m = x.amax(dim=1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)  # a row with nothing left: all log probabilities -inf
    z = x - m
    e = torch.exp(z)
    total = e.sum(dim=1)
    total = torch.where(total == 0, 1.0, total)
    log_z = torch.log(total)
    xt = x.gather(1, t[:, None])
    logprob = torch.where(asked, (xt - m)[:, 0] - log_z, 0.0)
    entropy = log_z - torch.where(e > 0, e * z, 0.0).sum(dim=1) / total
    before = torch.arange(x.shape[1], device=x.device)[None] < t[:, None]
    rank = ((x > xt) | ((x == xt) & before)).sum(dim=1)
    value, order = torch.sort(x, dim=1, descending=True, stable=True)
    value, order = value[:, :top], order[:, :top]
    return (logprob, entropy, torch.where(asked, rank, -1).int(), order.int(),
            value - m - log_z[:, None])


def _fork_plain(s):
    page, table, length, refs = s["case"]["page"], s["table"], s["length"], s["refs"]
    dst, src = s["dst"].long(), s["src"].long()
    old = table[dst]
    refs.index_add_(0, old.clamp(min=0).flatten(), -(old >= 0).int().flatten())
    free = (refs == 0).nonzero()[:, 0]
    size = torch.where(src >= 0, length[src.clamp(min=0)], 0)
    full = (size // page).long()
    from_ = table[src.clamp(min=0)]
    keep = torch.arange(table.shape[1], device="cuda")[None] < full[:, None]
    rows = torch.where(keep, from_, -1)
    refs.index_add_(0, rows.clamp(min=0).flatten(), (rows >= 0).int().flatten())
    part = (size % page > 0).nonzero()[:, 0]
    taken = free[:part.shape[0]]
    rows[part, full[part]] = taken.int()
    refs[taken] = 1
    table[dst], length[dst] = rows, size
    # the used rows of the partial pages, through all layers
    at = torch.arange(page, device="cuda")[None]
    used = at < (size % page)[part][:, None]
    a = (from_[part, full[part]].long()[:, None] * page + at)[used]
    b = (taken[:, None] * page + at)[used]
    for t in (s["codes"], s["scales"], s["rope"]):
        t[:, b] = t[:, a]


def _append_plain(s):
    page, table, length, refs = s["case"]["page"], s["table"], s["length"], s["refs"]
    dst, counts = s["dst"].long(), s["counts"].long()
    old = length[dst].long()
    have, want = (old + page - 1) // page, (old + counts + page - 1) // page
    free = (refs == 0).nonzero()[:, 0]
    j = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (j >= have[:, None]) & (j < want[:, None])
    taken = free[:int((want - have).sum())]
    rows = table[dst]
    rows[fresh] = taken.int()
    refs[taken] = 1
    table[dst], length[dst] = rows, (old + counts).int()
    op = torch.repeat_interleave(torch.arange(len(dst), device="cuda"), counts)
    at = torch.arange(op.shape[0], device="cuda") - (counts.cumsum(0) - counts)[op] + old[op]
    s["rows"].copy_(rows[op, at // page].long() * page + at % page)


def _compact_plain(s):
    page, table, refs = s["case"]["page"], s["table"], s["refs"]
    live = refs > 0
    n = live.sum()
    i = torch.arange(refs.shape[0], device="cuda")
    holes = (~live & (i < n)).nonzero()[:, 0]
    moved = (live & (i >= n)).nonzero()[:, 0]
    to = i.clone()
    to[moved] = holes
    for t in (s["codes"], s["scales"], s["rope"]):
        v = t.view(t.shape[0], refs.shape[0], page, t.shape[2])
        v[:, holes] = v[:, moved]
    s["table_out"].copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), -1))
    s["refs_out"].copy_(refs)
    s["refs_out"][holes] = refs[moved]
    s["refs_out"][moved] = 0


# ------------------------------------------------------------ 64 bits --


def exact(case, seed):
    """The computed outputs from their definitions in 64 bits: attention one sequence and a few heads
    at a time, log probabilities some rows at a time. Page operations compute no numbers."""
    if case["op"] not in ("attn", "logprob"):
        return None
    s = prepare(case, seed)
    if case["op"] == "logprob":
        got = [[], [], []]
        step = max(1, (1 << 27) // case["vocab"])
        for i in range(0, case["rows"], step):
            x = s["logits"][i:i + step].double()
            dead = (x == -math.inf).all(dim=1, keepdim=True)
            lp = torch.where(dead, -math.inf, torch.log_softmax(x, dim=1))
            t = s["tokens"][i:i + step].long()
            picked = lp.gather(1, t.clamp(0, case["vocab"] - 1)[:, None])[:, 0]
            got[0].append(torch.where((t >= 0) & (t < case["vocab"]), picked, 0.0))
            got[1].append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(dim=1))
            got[2].append(lp.topk(case["top"], dim=1).values)
        a, b, d = (torch.cat(v) for v in got)
        return a, b, None, None, d
    outs, lses = [], []
    value = s["codes"][0].view(torch.float8_e4m3fn)
    for i, (n, length) in enumerate(_lens(case)):
        lo, hi = _span(case, n, length)
        pos = torch.arange(lo, hi, device="cuda")
        page = s["table"][i][pos // case["page"]].long()
        row = page.clamp(min=0) * case["page"] + pos % case["page"]
        k = value[row].double().view(-1, NOPE // 64, 64)
        k = k * (2.0 ** (s["scales"][0][row][:, :NOPE // 64].double() - 127))[:, :, None]
        k = torch.cat([k.flatten(1), s["rope"][0][row].double()], dim=1)
        first = int(sum(m for m, _ in _lens(case)[:i]))
        q = s["q"][first:first + n].double()
        p = torch.arange(length - n, length, device="cuda")
        hide = (pos[None] > p[:, None]) | (page < 0)[None]
        if case["window"]:
            hide = hide | (p[:, None] - pos[None] >= case["window"])
        o, lse = [], []
        step = max(1, (1 << 28) // (n * (hi - lo)))
        for h in range(0, case["heads"], step):
            x = torch.einsum("nhd,kd->hnk", q[:, h:h + step], k) / math.sqrt(DIM)
            x = x.masked_fill(hide[None], -math.inf)
            sink = s["sink"][h:h + step].double()[:, None, None].expand(-1, n, 1)
            x = torch.cat([x, sink], dim=2)
            lse.append(torch.logsumexp(x, dim=2).T)
            o.append(torch.einsum("hnk,kd->nhd", torch.softmax(x, dim=2)[..., :-1], k))
        o = torch.cat(o, dim=1)
        z = torch.view_as_complex(o[..., NOPE:].reshape(n, case["heads"], ROPE // 2, 2).contiguous())
        turn = torch.complex(s["cos"][first:first + n].double(), -s["sin"][first:first + n].double())
        o[..., NOPE:] = torch.view_as_real(z * turn[:, None]).flatten(-2)
        outs.append(o)
        lses.append(torch.cat(lse, dim=1))
    return torch.cat(outs), torch.cat(lses)
