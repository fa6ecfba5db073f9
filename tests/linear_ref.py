"""Plain 64-bit forms of the block-FP8 operators, and how far a kernel may be from them."""
import torch

E4M3 = torch.float8_e4m3fn
HALF8, HALF16, HALF32 = 2.0 ** -4, 2.0 ** -8, 2.0 ** -24     # half a step of e4m3, bf16, fp32, relative to the value
LEAST8 = 2.0 ** -10                                         # half a step of e4m3 below 2^-6


def groups_of(x):
    """[..., K] as [..., groups, 128], zeros behind the last value."""
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % 128)).unflatten(-1, (-1, 128))


def spread(s, n):
    """One number for 128 columns -> one for each of n."""
    return s.repeat_interleave(128, -1)[..., :n]


def tops(x):
    m = groups_of(x).abs().amax(-1)
    return torch.where(m < 2.0 ** -100, torch.ones_like(m), m)


def codes32(x):
    """Codes and scales of fp32 rows by the operations of the definition, each rounded to fp32: what the kernel has to give, bit for bit."""
    m = tops(x)
    q = (x * spread(torch.full_like(m, 448.0) / m, x.shape[-1])).clamp(-448, 448).to(E4M3)
    return q, m / torch.full_like(m, 448.0)


def values(q, s, blocks=False):
    if blocks:
        s = s.repeat_interleave(128, -2)[..., :q.shape[-2], :]
    return q.view(E4M3).double() * spread(s.double(), q.shape[-1])


def gated(y):
    a, b = y.chunk(2, -1)
    return a * torch.sigmoid(a) * b


def product(q, s, w, ws):
    """(y, how far fp32 sums may be from it): q [M, K] x w [N, K] with their scales.

    A group's products are exact in fp32 and summed by the tensor core, 128 of them, with at most 2^-23 of the sum of their magnitudes lost
    at each addition (it may cut instead of rounding); each group's sum is then multiplied by a product of two scales (one rounding)
    and added (one rounding, of a sum that is at most the sum of all magnitudes)."""
    a, b = values(q, s), values(w, ws, True)
    y, size = a @ b.T, a.abs() @ b.abs().T
    groups = s.shape[-1]
    return y, size * (128 * 2.0 ** -23 + (groups + 2) * HALF32)


def weight(n, k, gen, lead=()):
    w = 0.02 * torch.randn(*lead, n, k, generator=gen)
    g = groups_of(torch.nn.functional.pad(w, (0, 0, 0, -n % 128))).unflatten(-3, (-1, 128))
    s = (g.abs().amax((-3, -1)) / 448.0).clamp(min=1e-12)
    q = (w / spread(s.repeat_interleave(128, -2)[..., :n, :], k)).clamp(-448, 448).to(E4M3)
    return q, s


def states(m, k, gen):
    return (torch.randn(m, k, generator=gen) * torch.exp(0.5 * torch.randn(k, generator=gen))).to(torch.bfloat16)


def near(got, want, off, half):
    """Whether `got` (of a type with this half step) is `want` to within `off` before its rounding."""
    got = got.double()
    return bool(((got - want).abs() <= off + half * (want.abs() + off)).all())


def gate_near(q, s, y, off):
    """Whether codes q and scales s stand for the gated halves of a result that is y to within off.

    silu has a slope of at most 1.1, so half a's error reaches the product at most 1.1 |b| times and b's |silu(a)| times, both together 1.1 times their
    product; exp, quotient and product of the gate lose at most (8 + 1.2 |a|) 2^-23 of it (2 + 1.173 |a| units for the exponential, 2 for the quotient,
    one rounding each for the sum, the product, and two for the scale and its application)."""
    a, b = y.chunk(2, -1)
    da, db = off.chunk(2, -1)
    v = gated(y)
    slack = 1.1 * da * b.abs() + (a * torch.sigmoid(a)).abs() * db + 1.1 * da * db + v.abs() * (8 + 1.2 * a.abs()) * 2.0 ** -23
    m, worst = tops(v), groups_of(slack).amax(-1)
    scale_ok = ((s.double() - m / 448).abs() <= worst / 448 + m / 448 * 2.0 ** -22).all()
    per = spread(s.double(), v.shape[-1])
    got = q.double() * per
    step = torch.maximum(HALF8 * (v.abs() + slack), LEAST8 * per)
    return bool(scale_ok) and bool(((got - v).abs() <= slack + step * (1 + 2.0 ** -20)).all())


def plan(ids, n):
    """Offsets, tokens, positions by a loop."""
    flat = ids.flatten().tolist()
    runs = [[i for i, e in enumerate(flat) if e == x] for x in range(n)]
    offsets, tokens, positions = [0], [], [-1] * len(flat)
    for run in runs:
        for i in run:
            positions[i] = len(tokens)
            tokens.append(i // ids.shape[1])
        offsets.append(len(tokens))
    tokens += [-1] * (len(flat) - len(tokens))
    return torch.tensor(offsets), torch.tensor(tokens, dtype=torch.int64), torch.tensor(positions, dtype=torch.int64).view(ids.shape)


def combine(partial, positions, weights, residual=None):
    """(sum, sum of magnitudes)."""
    p = positions.long()
    w = weights.double()[..., None] * (p >= 0)[..., None]
    rows = partial.double()[p.clamp(min=0)] if len(partial) else torch.zeros(*p.shape, partial.shape[1], dtype=torch.float64)
    r = torch.zeros(1, dtype=torch.float64) if residual is None else residual.double()
    return (w * rows).sum(1) + r, (w * rows).abs().sum(1) + r.abs()
