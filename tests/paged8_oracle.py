"""The 8-bit paged KV cache in 64 bits, token by token, for the tests: no code of the package."""
import math

import torch

PAGE = 16
LEVELS = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def f64(t):
    return (t.float() if t.dtype == torch.float8_e4m3fn else t).double().cpu()


def half_ulp(x, dtype):
    """Half the distance between neighbouring codes around x (codes are 64-bit values)."""
    if dtype == torch.int8:
        return torch.full_like(x, 0.5)
    a = x.abs().clamp_min(2.0 ** -6)
    return torch.exp2(torch.floor(torch.log2(a)) - 4)


class Layer:
    """One layer of a cache on ``device`` with sequences of the given lengths."""

    def __init__(self, lens, hkv, d, dtype, device, extra_pages=3, seed=0, width=None, layers=None,
                 fill=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.d, self.dtype, self.device = list(lens), hkv, d, dtype, device
        need = [-(-n // PAGE) for n in lens]
        self.num_pages = sum(need) + extra_pages
        order = torch.randperm(self.num_pages, generator=g).tolist()
        w = max(1, max(need)) if width is None else width
        table = torch.zeros(len(lens), w, dtype=torch.int32)
        at = 0
        for i, k in enumerate(need):
            table[i, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
            at += k
        self.spare = order[at:]
        lead = () if layers is None else (layers,)
        shape = (*lead, self.num_pages, hkv, 2, PAGE, d)
        if fill:
            if dtype == torch.int8:
                codes = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)
            else:
                codes = (torch.randn(shape, generator=g) * 100).clamp(-448, 448).to(dtype)
            scales = (0.25 + torch.rand(shape[:-2], generator=g)) * 3 / LEVELS[dtype]
        else:
            codes = torch.zeros(shape, dtype=dtype)
            scales = torch.zeros(shape[:-2])
        self.codes, self.scales = codes.to(device), scales.to(device)
        self.table = table.to(device)
        self.kv_lens = torch.tensor(self.lens, dtype=torch.int32, device=device)

    def values(self, i, n=None, layer=None):
        """[2, Hkv, n, D] of sequence i in 64 bits."""
        n = self.lens[i] if n is None else n
        c = self.codes if layer is None else self.codes[layer]
        s = self.scales if layer is None else self.scales[layer]
        p = self.table[i, :-(-n // PAGE)].long()
        x = f64(c[p]) * f64(s[p])[..., None, None]
        return x.permute(2, 1, 0, 3, 4).reshape(2, self.hkv, -1, self.d)[:, :, :n]


def attention(layer, q, cu, scale):
    """(out, sum of p|v|, weights per sequence [Hkv, n], largest sum of |q k| scale)."""
    G = q.shape[1] // layer.hkv
    q = f64(q)
    out, spread, weights, mag = torch.zeros_like(q), torch.zeros_like(q), [], 0.0
    for i, n in enumerate(layer.lens):
        rows = cu[i + 1] - cu[i]
        w = torch.zeros(layer.hkv, n, dtype=torch.float64)
        k, v = layer.values(i)
        for t in range(rows):
            seen = n - rows + t + 1
            if seen <= 0:
                continue
            for h in range(q.shape[1]):
                x = q[cu[i] + t, h]
                s = (k[h // G, :seen] @ x) * scale
                mag = max(mag, float((k[h // G, :seen].abs() @ x.abs()).max()) * scale)
                p = torch.softmax(s, 0)
                out[cu[i] + t, h] = p @ v[h // G, :seen]
                spread[cu[i] + t, h] = p @ v[h // G, :seen].abs()
                w[h // G, :seen] += p
        weights.append(w)
    return out, spread, weights, mag


def keep_order(mass, budget, recent):
    """Indices kept of one head's masses (a list of floats)."""
    n = len(mass)
    if n <= budget:
        return list(range(n))
    old = sorted(range(n - recent), key=lambda j: (-mass[j], j))[:budget - recent]
    return sorted(old) + list(range(n - recent, n))


def score_error(mag):
    """Bound of the error of a score in log2 units: a dot product of exact factors in 32 bits
    whose magnitudes add up to mag (natural units), and three more roundings."""
    return mag * math.log2(math.e) * 2.0 ** -20
