"""The paged cache's operators in 64 bits, written plainly, and how far 32-bit arithmetic with the stated roundings may be from them."""
import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def make_rows(q, new, lengths, page, pages_extra=3, seed=0, stride_extra=0, max_length=None, max_new=None):
    """PagedRows of sequences with these new tokens and lengths, pages in a random order; returns (rows, number of pages, table on the host)."""
    g = torch.Generator().manual_seed(seed)
    per = [max(1, -(-n // page)) for n in lengths]
    pages = sum(per) + pages_extra
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(per) + stride_extra), -7, dtype=torch.int32)  # what is not a sequence's is no page
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    dev = "cuda"
    tokens = int(starts[-1])
    rows = q.PagedRows(starts.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev), table.to(dev), tokens, max_new or max(new), max_length or max(lengths))
    return rows, pages, table


def whole(q, rows):
    """The same sequences with everything they hold as new tokens."""
    n = rows.lengths.to(torch.int64)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=n.device), n.cumsum(0)]).to(torch.int32)
    return q.PagedRows(starts, rows.lengths, rows.table, int(starts[-1]), int(n.max()), int(n.max()))


def places(rows):
    """(sequence, position) of every packed token, as lists."""
    starts, lengths = rows.starts.tolist(), rows.lengths.tolist()
    out = []
    for s, length in enumerate(lengths):
        n = starts[s + 1] - starts[s]
        out += [(s, length - n + i) for i in range(n)]
    return out


def written(x, weights, eps, cos_sin, neox, positions):
    """Heads [tokens][heads][size] normalised and rotated, in 64 bits."""
    x = x.double().clone()
    if weights is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weights.double()
    if cos_sin is not None:
        r = cos_sin.shape[1]
        cs = cos_sin.double()[positions]
        c, s = cs[:, None, 0::2], cs[:, None, 1::2]
        i0 = torch.arange(r // 2, device=x.device) if neox else torch.arange(0, r, 2, device=x.device)
        i1 = i0 + r // 2 if neox else i0 + 1
        a, b = x[..., i0].clone(), x[..., i1].clone()
        x[..., i0], x[..., i1] = a * c - b * s, a * s + b * c
    return x


def attention(qs, rows, keys, values, starts_all, scale, cap=0.0, window=0):
    """(out, bound): out [tokens][heads][size] in 64 bits from dense keys and values of whole sequences; what the bounds below need per output."""
    T, H, D = qs.shape
    G = H // keys.shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64, device=qs.device)
    mass = torch.zeros_like(out)            # sum of weight times |value|
    size = torch.zeros(T, H, 1, dtype=torch.float64, device=qs.device)  # the largest scale * sum |q| |k|
    for t, (s, p) in enumerate(places(rows)):
        if p < 0:
            continue
        lo = max(0, p - window + 1) if window else 0
        k = keys[starts_all[s] + lo:starts_all[s] + p + 1].double().repeat_interleave(G, 1)
        v = values[starts_all[s] + lo:starts_all[s] + p + 1].double().repeat_interleave(G, 1)
        x = qs[t].double()
        z = torch.einsum("hd,jhd->hj", x, k) * scale
        if cap:
            z = cap * torch.tanh(z / cap)
        w = torch.softmax(z, -1)
        out[t] = torch.einsum("hj,jhd->hd", w, v)
        mass[t] = torch.einsum("hj,jhd->hd", w, v.abs())
        size[t, :, 0] = torch.einsum("hd,jhd->hj", x.abs(), k.abs()).amax(-1) * abs(scale)
    return out, mass, size


def attention_bound(out, mass, size, length, head_dim, weight_type, out_type, values, q8=False, q_type=None, cap=0.0):
    """|kernel - exact| for each output. A weight is off by its rounding (half a step of weight_type) and by what its exponent is off: 32-bit sums of head_dim exact
    products (head_dim half steps of the sum of their magnitudes), the scale, the cap (2^-22 of the cap: two approximate functions) and the exponential (2^-21); Q8 adds
    the logarithm of a scale (2^-22 of a magnitude of at most 24 here, twice), and queries wider than F16 their rounding. Both sums are 32-bit sums of `length` terms.
    Errors of the weights count twice (numerator and denominator). F16 weights below 2^-14 are off by up to 2^-25 whatever their size, relative to a largest weight of one or
    more: the largest of a row's weights, for Q8 of its weights times scales. Each adds at most 2^-25 of the largest value, where the products that count may be as
    small as zero."""
    u = 2.0 ** -24
    z = size * (head_dim + 8) * u + cap * 2.0 ** -22
    if q8:
        z = z + 48 * 2.0 ** -22
        if q_type is torch.float32:
            z = z + size * EPS[torch.float16]
    w = 2.0 * torch.expm1(z) + 2.0 ** -20 + 2.0 * (length + 16) * u + EPS[weight_type]
    tiny = length * 2.0 ** -25 * float(values.abs().max()) if weight_type is torch.float16 else 0.0
    return mass * w + tiny + out.abs() * EPS[out_type] + 1e-30 + (2.0 ** -25 if out_type is torch.float16 else 0.0)
