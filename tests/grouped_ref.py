"""64-bit forms of the grouped products' formats, for the tests: E2M1, E4M3 and E8M0 decoded,
blocks quantised, and the bound of a product's fp32 sum.

The bound: an instruction adds 32 exact products to its fp32 sum; products and sum are aligned to
the largest of them and cut off below its last place, so that an instruction errs by at most four
units of 2^-24 of sum |x w|, and parts of a tile that several blocks bring add a rounding each:
(width / 32 + 8) 2^-22 sum |x w|."""
import torch

MAG = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def e8m0(c):
    return torch.where(c == 255, torch.nan, torch.exp2(c.double() - 127))


def e2m1(w):
    """[..., k / 2] packed bytes to [..., k]."""
    code = torch.stack([w & 15, w >> 4], dim=-1).flatten(-2).long()
    v = MAG.to(w.device)[code & 7]
    return torch.where(code > 7, -v, v)


def e4m3(c):
    return c.view(torch.float8_e4m3fn).double()


def rows_of(xq, xs):
    """[rows][k] values of codes with a scale per 128."""
    return e4m3(xq) * e8m0(xs).repeat_interleave(128, dim=-1)


def fp4_of(w, ws):
    return e2m1(w) * e8m0(ws).repeat_interleave(32, dim=-1)


def fp8_of(w, ws):
    s = e8m0(ws).repeat_interleave(128, dim=-1).repeat_interleave(128, dim=-2)
    return e4m3(w) * s[..., :w.shape[-2], :]


def sum_bound(x, w):
    return (x.shape[-1] / 32 + 8) * 2.0 ** -22 * (x.abs() @ w.abs().transpose(-1, -2))


def scale_of(amax):
    """The smallest power of two 2^e with max(amax, 1e-4) <= 448 2^e."""
    m, e = torch.frexp(amax.clamp(min=1e-4))
    return torch.exp2((e - 9 + (m > 0.875)).double())


def on_grid(v, scale):
    """v rounded to E4M3 times scale, half to even."""
    q = (v / scale).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(q / step) * step * scale


def quantised(v, each=128):
    """(values on the grid, scales) of rows of blocks of `each` (a last one may be shorter)."""
    got, scales = [], []
    for b in v.split(each, dim=-1):
        s = scale_of(b.abs().amax(dim=-1, keepdim=True))
        got.append(on_grid(b, s))
        scales.append(s)
    return torch.cat(got, -1), torch.cat(scales, -1)


def quantised_range(v, eps, each=128):
    """Lowest and highest value that rounding v + d, |d| <= eps, may give, whichever scale the
    block then has."""
    lo, hi = [], []
    for b, d in zip(v.split(each, dim=-1), eps.split(each, dim=-1)):
        scales = [scale_of(((b.abs() + s * d).clamp(min=0)).amax(dim=-1, keepdim=True)) for s in (-1, 1)]
        ends = [on_grid(e, s) for e in (b - d, b + d) for s in scales]
        lo.append(torch.stack(ends).amin(0))
        hi.append(torch.stack(ends).amax(0))
    return torch.cat(lo, -1), torch.cat(hi, -1)


def activations(rows, width, g, device="cuda"):
    x = torch.randn(rows, width, device=device, generator=g) * 110
    xs = torch.randint(116, 124, (rows, width // 128), dtype=torch.uint8, device=device, generator=g)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), xs


def fp4(groups, outs, width, g, device="cuda"):
    w = torch.randint(0, 256, (groups, outs, width // 2), dtype=torch.uint8, device=device, generator=g)
    ws = torch.randint(117, 124, (groups, outs, width // 32), dtype=torch.uint8, device=device, generator=g)
    return w, ws


def fp8(groups, outs, width, g, device="cuda"):
    w = torch.randn(groups, outs, width, device=device, generator=g) * 110
    ws = torch.randint(112, 118, (groups, -(-outs // 128), width // 128), dtype=torch.uint8,
                       device=device, generator=g)
    return w.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), ws
