"""Rows of 8-bit numbers and their products in double precision, from the definitions alone."""
import torch

TOP, LEAST = 448.0, 2.0 ** -100


def codes() -> torch.Tensor:
    """Values of the codes 0 to 126 (sign clear, 127 is NaN), in order: four bits of exponent with a bias of 7, three of fraction."""
    v = []
    for c in range(127):
        e, f = c >> 3, c & 7
        v.append((8 + f) * 2.0 ** (e - 10) if e else f * 2.0 ** -9)
    return torch.tensor(v, dtype=torch.float64)


def rounded(x: torch.Tensor) -> torch.Tensor:
    """x (double) to the nearest number of the format, ties to the even code, what is larger than the largest to that one; as doubles."""
    v = codes()
    a = x.abs().clamp(max=TOP)
    hi = torch.searchsorted(v, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up = (v[hi] - a < a - v[lo]) | ((v[hi] - a == a - v[lo]) & (hi % 2 == 0))
    return torch.where(up, v[hi], v[lo]) * x.sign()


def quantized(g: torch.Tensor, slack: float):
    """Of rows g (double): the scales a / 448, and the least and largest 8-bit numbers that 448 g / a can be rounded to when it is off by a
    factor of up to 1 +- slack."""
    a = g.abs().amax(-1, keepdim=True).clamp(min=LEAST)
    v = g * TOP / a
    one, two = rounded(v * (1 - slack)), rounded(v * (1 + slack))
    return a[:, 0] / TOP, torch.minimum(one, two), torch.maximum(one, two)


def gelu(z):
    return 0.5 * z * (1 + torch.erf(z / 2 ** 0.5))


def gelu_tanh(z):
    return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))


PLAIN = {"gelu": gelu, "relu_squared": lambda z: z.clamp(min=0) ** 2, "gelu_tanh": gelu_tanh, "silu": lambda z: z * torch.sigmoid(z)}


def gated(z, act, limit=0.0):
    """Columns in blocks of 16 gate and 16 up values -> act(gate) * up."""
    b = z.reshape(z.shape[0], -1, 2, 16)
    g, u = b[:, :, 0].reshape(z.shape[0], -1), b[:, :, 1].reshape(z.shape[0], -1)
    if act == "clamped":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        return g * torch.sigmoid(1.702 * g) * (u + 1)
    return (g * torch.sigmoid(g) if act == "silu" else gelu_tanh(g)) * u


def product(x, sx, w, sw, offsets=None):
    """(sum, sum of magnitudes) of the scaled product in double; grouped where offsets are given, zero behind the last."""
    if offsets is None:
        f = lambda a, b: (a @ b.T) * sx[:, None].double() * sw.double()  # noqa: E731
        return f(x.double(), w.double()), f(x.double().abs(), w.double().abs())
    z, m = (torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64) for _ in range(2))
    for e in range(w.shape[0]):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        z[lo:hi], m[lo:hi] = product(x[lo:hi], sx[lo:hi], w[e], sw[e])
    return z, m
