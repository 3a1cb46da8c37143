"""Cases of the operators that a step of many rows runs beside its attention: the routed experts and
the products grouped by expert under them, the norm that makes their 8-bit input, the write of new
latents into their pages, and the selection of beams.

`run` computes one call in plain torch operations, or with the framework's operators where `own` is
true; `exact` computes it in 64 bits. Layouts are the framework's: E2M1 codes two a byte (the low
nibble first) with one E8M0 scale per 32, E4M3 activations with one E8M0 scale per 128, E4M3 weights
with one per 128 x 128, latent rows of 448 E4M3 codes with one scale per 64 and 64 BF16 RoPE values.
"""
import math
import os
import random
import sys

import torch

own = False

NOPE, ROPE, DIM = 448, 64, 512
VOCAB = 129280
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _binding():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "deepseek-v4-flash-0731-in-c_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import dsv4cuda
    return dsv4cuda


def listed():
    return [
        # one token through the routed experts of the benchmark's model: latency of reading six of them
        dict(name="experts_token", op="experts", n=1, hidden=4096, inter=2048, experts=256, topk=6,
             skew=0.0, limit=10),
        # a decode step of 32 sequences, experts of 7168 x 2048: most experts have a row or two
        dict(name="experts_batch", op="experts", n=32, hidden=7168, inter=2048, experts=256, topk=8,
             skew=0.0, limit=10),
        # a prompt's chunk of 2,000 tokens (ragged): every expert is read for some 47 rows
        dict(name="experts_chunk", op="experts", n=2000, hidden=4096, inter=2048, experts=256, topk=6,
             skew=0.5, limit=10),
        # several prompts at once, the experts' popularity uneven: the products outweigh the weights
        dict(name="experts_prompts", op="experts", n=8192, hidden=4096, inter=2048, experts=256, topk=6,
             skew=0.5, limit=10),
        # ragged groups, some empty, of a narrow expert with an odd number of outputs
        dict(name="grouped_ragged", op="grouped", rows=777, outs=1003, width=1152, experts=24, fp8=False,
             f32=True, gather=True, skew=1.0),
        # a prompt chunk through a dense FP8 projection (the query's, 64 heads x 512 from 1,024)
        dict(name="grouped_dense", op="grouped", rows=2048, outs=32768, width=1024, experts=1, fp8=True,
             f32=False, gather=False, skew=0.0),
        # the decode step's row
        dict(name="norm_token", op="norm", rows=1, width=4096, f32=False, residual=True, pad=0),
        # a prompt chunk's rows at the wide model's size
        dict(name="norm_chunk", op="norm", rows=4096, width=7168, f32=False, residual=True, pad=0),
        # the new latents of a decode step of 32 sequences
        dict(name="write_step", op="write", rows=32, pages=2048, page=64, f32=False, normed=True, absent=0),
        # the new latents of several prompts' chunks, with the padding of a captured step
        dict(name="write_chunk", op="write", rows=16000, pages=1024, page=64, f32=False, normed=True,
             absent=384),
        # one prompt's four beams
        dict(name="beam_few", op="beam", groups=1, beams=4, cands=8, vocab=VOCAB, f32=True, pad=0,
             masked=0.0),
        # a batch of 64 prompts with eight beams each
        dict(name="beam_batch", op="beam", groups=64, beams=8, cands=16, vocab=VOCAB, f32=False, pad=8,
             masked=0.2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["experts", "experts", "experts", "grouped", "grouped", "norm", "write", "beam"])
    if op == "experts":
        while True:
            c = dict(op=op, n=_log_int(rng, 1, 8192), hidden=128 * _log_int(rng, 2, 56),
                     inter=128 * _log_int(rng, 1, 16), experts=_log_int(rng, 4, 256),
                     topk=rng.randint(1, 8), skew=rng.choice([0.0, 0.5, 1.0]), limit=rng.choice([7, 10]))
            c["topk"] = min(c["topk"], c["experts"])
            if (c["n"] * c["topk"] * c["hidden"] * c["inter"] <= 8192 * 6 * 4096 * 2048
                    and c["experts"] * c["hidden"] * c["inter"] <= 256 * 7168 * 2048
                    and max(_counts(c)) * c["experts"] * c["hidden"] <= 1 << 32):
                return c
    if op == "grouped":
        while True:
            c = dict(op=op, rows=_log_int(rng, 1, 16384), outs=_log_int(rng, 16, 32768),
                     width=128 * _log_int(rng, 1, 64), experts=rng.choice([1, _log_int(rng, 2, 256)]),
                     fp8=rng.random() < 0.5, f32=rng.random() < 0.4, gather=rng.random() < 0.5,
                     skew=rng.choice([0.0, 0.5, 1.5]))
            if (c["rows"] * c["outs"] <= 1 << 28 and c["rows"] * c["outs"] * c["width"] <= 1 << 37
                    and c["experts"] * c["outs"] * c["width"] <= 1 << 31
                    and max(_counts(c)) * c["experts"] * max(c["width"], c["outs"]) <= 1 << 32):
                return c
    if op == "norm":
        rows = _log_int(rng, 1, 16384)
        return dict(op=op, rows=rows, width=min(_log_int(rng, 16, 16384), (1 << 25) // rows),
                    f32=rng.random() < 0.3, residual=rng.random() < 0.7, pad=rng.choice([0, 8, rng.randint(1, 64)]))
    if op == "write":
        page = rng.choice([16, 64, rng.randint(1, 200)])
        rows = _log_int(rng, 1, 32768)
        return dict(op=op, rows=rows, pages=-(-rows // page) + rng.randint(1, 400), page=page,
                    f32=rng.random() < 0.3, normed=rng.random() < 0.8, absent=rng.choice([0, rows // 7]))
    while True:
        beams = rng.randint(1, 16)
        c = dict(op=op, groups=_log_int(rng, 1, 128), beams=beams, cands=rng.randint(beams, 2 * beams),
                 vocab=rng.choice([VOCAB, _log_int(rng, 100, 260000)]), f32=rng.random() < 0.5,
                 pad=rng.choice([0, 8, rng.randint(1, 64)]), masked=rng.choice([0.0, 0.2, 0.95]))
        if c["groups"] * c["beams"] * c["vocab"] * (2 if c["f32"] else 1) <= 512 * VOCAB:
            return c


# ------------------------------------------------------------------ sizes --


def _weights_of(c):
    """How often each expert is taken, most first (relative)."""
    return [(i + 1.0) ** -c["skew"] for i in range(c["experts"])]


def _routes(c):
    """Experts of each token [n][topk], ascending, the same for every seed; and, of grouped rows, how
    many each expert has."""
    g = torch.Generator()
    if c["op"] == "grouped":
        g.manual_seed(c["rows"] * 31 + c["experts"])
        share = torch.tensor(_weights_of(c), dtype=torch.float64)
        if c["experts"] > 3:
            share[torch.randperm(c["experts"], generator=g)[:c["experts"] // 6]] = 0  # nobody's
        return torch.bincount(torch.multinomial(share, c["rows"], replacement=True, generator=g),
                              minlength=c["experts"])
    g.manual_seed(c["n"] * 31 + c["experts"])
    share = torch.tensor(_weights_of(c), dtype=torch.float64).log()
    noise = torch.rand(c["n"], c["experts"], dtype=torch.float64, generator=g).log().neg().log().neg()
    return (share[None] + noise).topk(c["topk"], dim=1).indices.sort(dim=1).values


def _counts(c):
    r = _routes(c)
    return (r if c["op"] == "grouped" else torch.bincount(r.flatten(), minlength=c["experts"])).tolist()


def work(c):
    if c["op"] == "experts":
        live = sum(x > 0 for x in _counts(c))
        matrix = c["hidden"] * c["inter"]
        return {"bytes": live * 3 * (matrix // 2 + matrix // 32)
                + c["n"] * (c["hidden"] + c["hidden"] // 128 + 8 * c["topk"] + 2 * c["hidden"]),
                "flops": 6 * c["n"] * c["topk"] * matrix}
    if c["op"] == "grouped":
        live = sum(x > 0 for x in _counts(c))
        k, m = c["width"], c["outs"]
        one = m * k + -(-m // 128) * (k // 128) if c["fp8"] else m * k // 2 + m * k // 32
        return {"bytes": live * one + c["rows"] * (k + k // 128 + m * (4 if c["f32"] else 2)),
                "flops": 2 * c["rows"] * k * m}
    if c["op"] == "norm":
        size = 4 if c["f32"] else 2
        each = c["width"] * (size * (2 + 2 * c["residual"]) + 1) + -(-c["width"] // 128)
        return {"bytes": c["rows"] * each + 2 * c["width"], "flops": 8 * c["rows"] * c["width"]}
    if c["op"] == "write":
        live = c["rows"] - c["absent"]
        return {"bytes": live * (DIM * (4 if c["f32"] else 2) + NOPE + NOPE // 64 + 2 * ROPE + 4 * ROPE)
                + 8 * c["rows"] + 2 * DIM, "flops": 8 * live * DIM}
    rows = c["groups"] * c["beams"]
    return {"bytes": rows * (c["vocab"] * (4 if c["f32"] else 2) + 4 + 16) + c["groups"] * c["cands"] * 12,
            "flops": 4 * rows * c["vocab"]}


# ----------------------------------------------------------------- inputs --


def _activations(rows, width, g):
    """E4M3 codes and E8M0 scales of rows such as a norm's output has."""
    codes = torch.empty(rows, width, dtype=torch.uint8, device="cuda")
    for i in range(0, rows, 4096):
        x = torch.randn(codes[i:i + 4096].shape, device="cuda", generator=g) * 110
        codes[i:i + 4096] = x.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.randint(118, 122, (rows, width // 128), dtype=torch.uint8, device="cuda", generator=g)
    return codes, scales


def _fp4(experts, outs, width, g):
    """Random codes, and scales that make outputs of the inputs' size."""
    w = torch.randint(0, 256, (experts, outs, width // 2), dtype=torch.uint8, device="cuda", generator=g)
    s = torch.randint(0, 3, (experts, outs, width // 32), dtype=torch.uint8, device="cuda", generator=g)
    return w, s + (125 - int(round(math.log2(width) / 2)))


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    f32 = dict(dtype=torch.float32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    u8 = dict(dtype=torch.uint8, device="cuda")
    kind = dict(dtype=torch.float32 if c.get("f32") else torch.bfloat16, device="cuda")
    if c["op"] == "experts":
        h, i, e, n, k = c["hidden"], c["inter"], c["experts"], c["n"], c["topk"]
        s["w1"], s["s1"] = _fp4(e, i, h, g)
        s["w3"], s["s3"] = _fp4(e, i, h, g)
        s["w2"], s["s2"] = _fp4(e, h, i, g)
        # which expert is the popular one, and which token takes which, are the seed's
        name = torch.randperm(e, device="cuda", generator=g)
        order = torch.randperm(n, device="cuda", generator=g)
        s["idx"] = name[_routes(c).cuda()[order]].sort(dim=1).values.int()
        wt = torch.rand(n, k, device="cuda", generator=g) + 0.1
        s["wt"] = 1.5 * wt / wt.sum(dim=1, keepdim=True)
        s["xq"], s["xs"] = _activations(n, h, g)
        s["out"] = torch.empty(n, h, dtype=torch.bfloat16, device="cuda")
        if own:
            weights = dict(hidden=h, moe_inter=i, n_experts=e, topk=k, swiglu_limit=c["limit"],
                           route_scale=1.5, gate_w=torch.zeros(e, h, dtype=torch.int16, device="cuda"),
                           **{m: s[m] for m in ("w1", "s1", "w3", "s3", "w2", "s2")})
            s["layer"] = _binding().MoeLayer(weights, max_tokens=1, device=True)
        return s
    if c["op"] == "grouped":
        e, m, k, rows = c["experts"], c["outs"], c["width"], c["rows"]
        if c["fp8"]:
            s["w"] = torch.empty(e, m, k, **u8)
            flat = s["w"].view(-1)
            for j in range(0, flat.shape[0], 1 << 28):
                x = torch.randn(flat[j:j + (1 << 28)].shape, device="cuda", generator=g) * 110
                flat[j:j + (1 << 28)] = x.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            s["ws"] = torch.randint(0, 3, (e, -(-m // 128), k // 128), **u8, generator=g) + 112
        else:
            s["w"], s["ws"] = _fp4(e, m, k, g)
        count = _routes(c).cuda()[torch.randperm(e, device="cuda", generator=g)]
        s["offsets"] = torch.zeros(e + 1, **i32)
        s["offsets"][1:] = count.cumsum(0)
        s["most"] = max(_counts(c))
        held = max(1, rows // 2) if c["gather"] else rows  # tokens that several experts take
        s["xq"], s["xs"] = _activations(held, k, g)
        s["src"] = s["dst"] = None
        if c["gather"]:
            s["src"] = torch.randint(0, held, (rows,), **i32, generator=g)
            s["dst"] = torch.randperm(rows, device="cuda", generator=g).int()
        s["out"] = torch.empty(rows, m, **kind)
    elif c["op"] == "norm":
        rows, width = c["rows"], c["width"]
        s["x"] = torch.randn(rows, width + c["pad"], device="cuda", generator=g).to(kind["dtype"])[:, :width]
        s["residual"] = None
        s["sum"] = None
        if c["residual"]:
            s["residual"] = (torch.randn(rows, width, device="cuda", generator=g) * 3).to(kind["dtype"])
            s["sum"] = torch.empty(rows, width, **kind)
        s["gain"] = (1 + 0.1 * torch.randn(width, device="cuda", generator=g)).bfloat16()
        s["codes"] = torch.empty(rows, width, **u8)
        s["scales"] = torch.empty(rows, -(-width // 128), **u8)
        s["out"] = torch.empty(rows, width, **kind)
    elif c["op"] == "write":
        rows, total = c["rows"], c["pages"] * c["page"]
        s["kv"] = torch.randn(rows, DIM, device="cuda", generator=g).to(kind["dtype"])
        # whole pages in the tables' order, and -1 behind the last new token
        page = torch.randperm(c["pages"], device="cuda", generator=g)
        at = (page[:, None] * c["page"] + torch.arange(c["page"], device="cuda")[None]).flatten()[:rows]
        s["rows"] = torch.where(torch.arange(rows, device="cuda") < rows - c["absent"], at, -1)
        pos = torch.arange(rows, device="cuda") % 8192 + 5
        freq = 10000.0 ** (-torch.arange(0, ROPE, 2, device="cuda", dtype=torch.float64) / ROPE)
        angle = pos[:, None].double() * freq[None]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["gain"] = None
        if c["normed"]:
            s["gain"] = (1 + 0.1 * torch.randn(DIM, device="cuda", generator=g)).bfloat16()
        s["codes"] = torch.randint(0, 127, (total, NOPE), **u8, generator=g)
        s["scales"] = torch.randint(119, 123, (total, 8), **u8, generator=g)
        s["rope"] = torch.randn(total, ROPE, device="cuda", generator=g).bfloat16()
        if own:
            lib = _binding()
            cache = lib.LatentCache.from_tensors(s["codes"], s["scales"], s["rope"].view(torch.int16))
            s["pool"] = lib.PagedCache([cache], c["page"], torch.full((1, c["pages"]), -1, **i32),
                                       torch.zeros(1, **i32), torch.zeros(c["pages"], **i32))
    else:
        rows, width = c["groups"] * c["beams"], c["vocab"] + c["pad"]
        x = torch.empty(rows, width, **kind)
        for i in range(0, rows, 256):
            y = torch.randn(x[i:i + 256].shape, device="cuda", generator=g) * 2.5
            if c["masked"]:
                y = torch.where(torch.rand(y.shape, device="cuda", generator=g) < c["masked"], -math.inf, y)
            x[i:i + 256] = y
        x[:, c["vocab"]:] = 1e30  # what lies behind a row is not the row's
        s["logits"] = x[:, :c["vocab"]]
        score = -torch.rand(c["groups"], c["beams"], device="cuda", generator=g) * 6 - 1
        if c["groups"] > 3:
            score[::4, 1:] = -math.inf  # prompts just begun: one beam lives
        s["score"] = score
        # a slot of the pool for each beam
        s["slot"] = torch.randperm(rows, device="cuda", generator=g).int().view(c["groups"], c["beams"])
        # the sequence's end, which some candidate reaches
        s["eos"] = int(s["logits"][0].float().argmax())
        s["parent"] = torch.empty(c["groups"], c["cands"], **i32)
        s["token"] = torch.empty(c["groups"], c["cands"], **i32)
        s["total"] = torch.empty(c["groups"], c["cands"], **f32)
        s["next"] = torch.empty(c["groups"], c["beams"], **i32)
        s["to"] = torch.empty(c["groups"], c["beams"], **i32)
        s["from"] = torch.empty(c["groups"], c["beams"], **i32)
    if own:
        s["lib"] = _binding()
    return s


# ------------------------------------------------------------ one pass --


def run(s):
    op = s["case"]["op"]
    if op == "experts":
        if own:
            s["layer"].experts(s["xq"], s["xs"], s["idx"], s["wt"], s["out"])
            return s["out"]
        return _experts_plain(s)
    if op == "grouped":
        if own:
            s["lib"].grouped_gemm(s["out"], s["xq"], s["xs"], s["w"], s["ws"], s["offsets"], src=s["src"],
                                  dst=s["dst"])
            return s["out"]
        return _grouped_plain(s)
    if op == "norm":
        if own:
            s["lib"].norm_quant(s["x"], s["gain"], s["codes"], s["scales"], eps=1e-6,
                                residual=s["residual"], sum_out=s["sum"], out=s["out"])
        else:
            _norm_plain(s)
        return (s["codes"].view(torch.float8_e4m3fn), s["scales"].view(torch.float8_e8m0fnu), s["out"],
                s["sum"])
    if op == "write":
        if own:
            s["pool"].write(0, s["kv"], s["rows"], gain=s["gain"], eps=1e-6, rope_cos=s["cos"],
                            rope_sin=s["sin"])
        else:
            _write_plain(s)
        return s["codes"].view(torch.float8_e4m3fn), s["scales"].view(torch.float8_e8m0fnu), s["rope"]
    if own:
        s["lib"].beam_select(s["logits"], s["score"], s["parent"], s["token"], s["total"], s["next"],
                             slot=s["slot"], dst=s["to"], src=s["from"], eos=s["eos"])
        return s["parent"], s["token"], s["total"], s["next"], s["to"], s["from"]
    return _beam_plain(s)


def _scale_of(codes, each):
    return torch.exp2(codes.float() - 127).repeat_interleave(each, dim=-1)


def _fp4_values(w, ws):
    pairs = torch.tensor([[E2M1[b & 15], E2M1[b >> 4]] for b in range(256)], device="cuda")
    v = pairs[w.int()].flatten(-2)
    return v.view(*ws.shape, 32).mul_(torch.exp2(ws.float() - 127)[..., None]).flatten(-2)


def _fp8_values(w, ws):
    v = w.view(torch.float8_e4m3fn).float()
    return v * _scale_of(ws, 128).repeat_interleave(128, dim=-2)[..., :w.shape[-2], :]


def _pow2_scale(amax):
    """The smallest power of two that brings amax (1e-4 at least) to 448 or below."""
    m, e = torch.frexp(amax.clamp(min=1e-4))
    return torch.exp2((torch.where(m > 0.875, e + 1, e) - 9).to(amax.dtype))


def _quantised(v, each):
    """E4M3 codes and E8M0 codes of rows v, one scale per `each` values (the last of a row may have
    fewer)."""
    n = v.shape[-1]
    pad = -n % each
    b = torch.nn.functional.pad(v, (0, pad)).unflatten(-1, (-1, each))
    scale = _pow2_scale(b.abs().amax(dim=-1))
    q = (b / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q.flatten(-2)[..., :n], (torch.log2(scale) + 127).to(torch.uint8)


def _padded_rows(offsets, experts, most):
    """Row of the i-th of expert e's group [experts][most] and which of them there are."""
    at = offsets[experts].long()[:, None] + torch.arange(most, device="cuda")[None]
    there = at < offsets[experts + 1].long()[:, None]
    return torch.where(there, at, 0), there


def _experts_plain(s):
    c = s["case"]
    n, k = c["n"], c["topk"]
    order = torch.sort(s["idx"].flatten(), stable=True).indices
    count = torch.bincount(s["idx"].flatten(), minlength=c["experts"])
    offsets = torch.nn.functional.pad(count.cumsum(0), (1, 0))
    live = count.nonzero()[:, 0]
    at, there = _padded_rows(offsets, live, int(count.max()))
    slot = order[at]
    x = s["xq"].view(torch.float8_e4m3fn).float() * _scale_of(s["xs"], 128)
    x = x[slot // k]
    gate = torch.bmm(x, _fp4_values(s["w1"][live], s["s1"][live]).transpose(1, 2))
    up = torch.bmm(x, _fp4_values(s["w3"][live], s["s3"][live]).transpose(1, 2))
    gate, up = gate.clamp(max=c["limit"]), up.clamp(-c["limit"], c["limit"])
    h = gate / (1 + torch.exp(-gate)) * up * s["wt"].flatten()[slot][..., None]
    q, e8 = _quantised(h, 128)
    y = torch.bmm(q.float() * _scale_of(e8, 128),
                  _fp4_values(s["w2"][live], s["s2"][live]).transpose(1, 2))
    slots = torch.empty(n * k, c["hidden"], device="cuda")
    slots[slot[there]] = y[there]
    return slots.view(n, k, -1).sum(dim=1).bfloat16()


def _grouped_plain(s):
    c = s["case"]
    offsets = s["offsets"]
    live = (offsets[1:] > offsets[:-1]).nonzero()[:, 0]
    at, there = _padded_rows(offsets, live, s["most"])
    x = s["xq"].view(torch.float8_e4m3fn).float() * _scale_of(s["xs"], 128)
    x = x[s["src"][at]] if c["gather"] else x[at]
    values = _fp8_values if c["fp8"] else _fp4_values
    y = torch.bmm(x, values(s["w"][live], s["ws"][live]).transpose(1, 2))[there].to(s["out"].dtype)
    row = at[there]
    out = torch.empty_like(s["out"])
    out[s["dst"][row] if c["gather"] else row] = y
    return out


def _norm_plain(s):
    v = s["x"].float()
    if s["residual"] is not None:
        v = v + s["residual"].float()
        s["sum"].copy_(v)
    y = v * torch.rsqrt(v.square().mean(dim=1, keepdim=True) + 1e-6) * s["gain"].float()
    q, e8 = _quantised(y, 128)
    s["codes"].copy_(q.view(torch.uint8))
    s["scales"].copy_(e8)
    s["out"].copy_(y)


def _write_plain(s):
    v = s["kv"].float()
    if s["gain"] is not None:
        v = v * torch.rsqrt(v.square().mean(dim=1, keepdim=True) + 1e-6) * s["gain"].float()
    a, b = v[:, NOPE::2].clone(), v[:, NOPE + 1::2].clone()
    rope = torch.stack([a * s["cos"] - b * s["sin"], a * s["sin"] + b * s["cos"]], dim=2).flatten(1)
    q, e8 = _quantised(v[:, :NOPE], 64)
    live = s["rows"] >= 0
    row = s["rows"][live]
    s["codes"][row] = q.view(torch.uint8)[live]
    s["scales"][row, :NOPE // 64] = e8[live]
    s["rope"][row] = rope[live].bfloat16()


def _beam_plain(s):
    c = s["case"]
    beams, cands, vocab = c["beams"], c["cands"], c["vocab"]
    # differences between candidates of two beams may be small: 64 bits
    x = s["logits"].double()
    m = x.amax(dim=1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    lse = m + torch.log(torch.exp(x - m).sum(dim=1, keepdim=True))
    lse = torch.where(lse == -math.inf, 0.0, lse)
    total = (s["score"].double().view(-1, 1) + (x - lse)).view(c["groups"], beams * vocab)
    value, order = torch.sort(total, dim=1, descending=True, stable=True)
    value, order = value[:, :cands], order[:, :cands]
    live = value > -math.inf
    parent = torch.where(live, order // vocab, -1)
    token = torch.where(live, order % vocab, -1)
    # the beams that go on: the best that have not ended
    on = live & (token != s["eos"])
    place = torch.where(on, on.cumsum(dim=1) - 1, cands)
    following = torch.full((c["groups"], cands + 1), -1, device="cuda")
    which = torch.arange(cands, device="cuda").expand(c["groups"], -1)
    following.scatter_(1, place, which)
    following = following[:, :beams]
    mother = torch.where(following >= 0, parent.gather(1, following.clamp(min=0)), -1)
    # a beam's first child stays in its slot; the others take the slots of beams without one
    earlier = torch.ones(beams, beams, device="cuda").tril(-1).bool()
    again = ((mother[:, :, None] == mother[:, None, :]) & earlier[None]).any(dim=2) | (mother < 0)
    lost = ~(mother[:, :, None] == torch.arange(beams, device="cuda")).any(dim=1)
    heir = torch.sort((~lost).int(), dim=1, stable=True).indices  # beams without children first
    turn = (again.cumsum(dim=1) - 1).clamp(min=0)
    home = torch.where(again, heir.gather(1, turn), mother.clamp(min=0))
    to = s["slot"].gather(1, home)
    source = torch.where(mother >= 0, s["slot"].gather(1, mother.clamp(min=0)), -1)
    return parent.int(), token.int(), value.float(), following.int(), to, source


# ------------------------------------------------------------ 64 bits --


def _e8m0(codes):
    return torch.ldexp(torch.ones_like(codes, dtype=torch.float64), codes.int() - 127)


def _exact_fp4(w, ws):
    code = torch.stack([w & 15, w >> 4], dim=-1).flatten(-2).int()
    exponent, half = (code & 7) >> 1, (code & 1).double()
    size = torch.where(exponent > 0, torch.ldexp(1 + half / 2, exponent - 1), half / 2)
    size = torch.where(code > 7, -size, size)
    return (size.view(*ws.shape, 32) * _e8m0(ws)[..., None]).view(size.shape)


def _exact_rows(codes, scales, each):
    v = codes.view(torch.float8_e4m3fn).double()
    return (v.view(*scales.shape, each) * _e8m0(scales)[..., None]).view(v.shape)


def _exact_e4m3(v, each):
    """Values on the E4M3 grid of each block's scale, and the scales: (codes' values, scales)."""
    codes, scales = [], []
    for b in v.split(each, dim=-1):
        top = b.abs().amax(dim=-1, keepdim=True).clamp(min=1e-4)
        power = torch.ceil(torch.log2(top / 448))
        power = torch.where(torch.ldexp(torch.full_like(top, 448.0), power.int()) < top, power + 1, power)
        b = torch.ldexp(b, -power.int())
        step = torch.ldexp(torch.ones_like(b), torch.floor(torch.log2(b.abs().clamp(min=2.0 ** -6))).int() - 3)
        codes.append((torch.round(b / step) * step).clamp(-448, 448))
        scales.append(torch.ldexp(torch.ones_like(power), power.int()))
    return torch.cat(codes, dim=-1), torch.cat(scales, dim=-1)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] == "experts":
        x = _exact_rows(s["xq"], s["xs"], 128)
        out = torch.zeros(c["n"], c["hidden"], dtype=torch.float64, device="cuda")
        for e in sorted(set(s["idx"].flatten().tolist())):
            t, j = (s["idx"] == e).nonzero(as_tuple=True)
            gate = (x[t] @ _exact_fp4(s["w1"][e], s["s1"][e]).T).clamp(max=c["limit"])
            up = (x[t] @ _exact_fp4(s["w3"][e], s["s3"][e]).T).clamp(-c["limit"], c["limit"])
            h = gate * torch.sigmoid(gate) * up * s["wt"][t, j].double()[:, None]
            q, scale = _exact_e4m3(h, 128)
            h = (q.unflatten(1, (-1, 128)) * scale[..., None]).flatten(1)
            out.index_add_(0, t, h @ _exact_fp4(s["w2"][e], s["s2"][e]).T)
        return out
    if c["op"] == "grouped":
        x = _exact_rows(s["xq"], s["xs"], 128)
        out = torch.zeros(c["rows"], c["outs"], dtype=torch.float64, device="cuda")
        edge = s["offsets"].tolist()
        for e in range(c["experts"]):
            if edge[e + 1] == edge[e]:
                continue
            r = torch.arange(edge[e], edge[e + 1], device="cuda")
            if c["fp8"]:
                w = s["w"][e].view(torch.float8_e4m3fn).double()
                grid = _e8m0(s["ws"][e])
                w = w * torch.kron(grid, torch.ones(128, 128, dtype=torch.float64, device="cuda"))[:c["outs"]]
            else:
                w = _exact_fp4(s["w"][e], s["ws"][e])
            y = x[s["src"][r].long() if c["gather"] else r] @ w.T
            out[s["dst"][r].long() if c["gather"] else r] = y
        return out
    if c["op"] == "norm":
        v = s["x"].double()
        if c["residual"]:
            v = v + s["residual"].double()
        y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * s["gain"].double()
        q, scale = _exact_e4m3(y, 128)
        return q, scale, y, v if c["residual"] else None
    if c["op"] == "write":
        v = s["kv"].double()
        if c["normed"]:
            v = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * s["gain"].double()
        turned = torch.view_as_complex(v[:, NOPE:].reshape(-1, ROPE // 2, 2).contiguous())
        turned = torch.view_as_real(turned * torch.complex(s["cos"].double(), s["sin"].double())).flatten(1)
        q, scale = _exact_e4m3(v[:, :NOPE], 64)
        codes = s["codes"].view(torch.float8_e4m3fn).double()
        scales, rope = _e8m0(s["scales"]), s["rope"].double()
        live = s["rows"] >= 0
        row = s["rows"][live]
        codes[row], scales[row, :NOPE // 64], rope[row] = q[live], scale[live], turned[live]
        return codes, scales, rope
    x = s["logits"].double()
    lp = torch.where((x == -math.inf).all(dim=1, keepdim=True), -math.inf, torch.log_softmax(x, dim=1))
    total = (s["score"].double().view(-1, 1) + lp).view(c["groups"], -1)
    return None, None, total.topk(c["cands"], dim=1).values, None, None, None
