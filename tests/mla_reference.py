"""Latent attention from its definition, in float64, with bounds on what the kernels' roundings may add.

u is half a step of a 16-bit type, relative (bf16 2^-8, fp16 2^-11); e = 2^-24 that of float32.

An attention result o = sum p v / sum p differs from the exact one by
* its own rounding, u |o|;
* the rounding of the exponentials for their product, u * a with a = sum p |v| / sum p; a float16 exponential below 2^-14 is off by up to
  2^-25 of the largest, which is at least 1 against a sum that is at least as large: 2^-25 * sum |v|;
* float32 sums of n terms in the numerator and the denominator, n e each (relative to a);
* errors of the scores, which multiply an exponential by exp(ds) and count in numerator and denominator: ds is at most
  (w + 8) e * sum |q k| * scale for a float32 dot product of w terms and the scaling's roundings, plus 2^-21 for the exponential
  itself and its argument's rounding near |s| <= 64 (2^-24 * 64 * 1.44 * 2 < 2^-16 is counted: |s| 2^-22).
"""
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


E = 2.0 ** -24


def softmax_rows(q, k, v, scale, limit, dtype):
    """q [m, w], k [n, w], v [n, d] float64, limit [m]: query i sees the first limit[i] keys.  -> out, lse, and their tolerances."""
    m, n = q.shape[0], k.shape[0]
    if n == 0:
        z = q.new_zeros((m, v.shape[1]))
        return z, q.new_full((m,), float("-inf")), z, q.new_zeros((m,))
    s = (q @ k.t()) * scale
    seen = torch.arange(n, device=q.device)[None] < limit[:, None]
    s = torch.where(seen, s, float("-inf"))
    some = seen.any(1)
    top = torch.where(some, s.max(1).values, 0.0)
    p = torch.exp(s - top[:, None])
    total = p.sum(1)
    div = torch.where(some, total, 1.0)
    out, mean = (p @ v) / div[:, None], (p @ v.abs()) / div[:, None]
    lse = torch.log(total) + top
    ds = torch.where(seen, (q.abs() @ k.abs().t()) * scale * ((q.shape[1] + 8) * E) + torch.where(seen, s, 0.0).abs() * 2.0 ** -22, 0.0).max(1).values + 2.0 ** -21
    u = half_step(dtype)
    tol = u * out.abs() + (u + 2 * n * E + 2 * ds)[:, None] * mean + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (seen.double() @ v.abs()) + 2.0 ** -25
    lse_tol = ds + n * E + torch.where(some, lse, 0.0).abs() * 4 * E + 2.0 ** -20
    return out, lse, tol, lse_tol


def close(got, want, tol, what=""):
    """Every element within its tolerance; the same infinities."""
    got = got.double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.where(finite, 0.0, want), torch.where(finite, 0.0, got)), what + ": infinities"
    err = torch.where(finite, (got - want).abs(), 0.0)
    over = err / torch.where(finite, tol, 1.0).clamp(min=1e-300)
    assert bool((over <= 1.0).all()), "%s: %.3g times the tolerance at %s" % (what, float(over.max()), tuple(int(i) for i in (over == over.max()).nonzero()[0]))


def rows_of(cache, table, length, scale):
    """The first `length` rows of a request, float64: cache [pages, page, 576], table a list of page numbers."""
    page = cache.shape[1]
    t = torch.arange(length, device=cache.device)
    flat = cache.reshape(-1, cache.shape[-1])
    index = torch.as_tensor(table, device=cache.device, dtype=torch.int64)[t // page] * page + t % page
    if cache.dtype == torch.float8_e4m3fn:
        return flat.view(torch.uint8)[index].view(torch.float8_e4m3fn).double() * (float(scale) if scale is not None else 1.0)
    return flat[index].double()


def decode(q_nope, q_pe, cache, table, lens, sm_scale, scale):
    """q_nope [B, n, H, 512], table and lens lists -> (out, lse, tolerances), as softmax_rows gives them, [B, n, H, ..]."""
    B, n, H, _ = q_nope.shape
    parts = []
    for b in range(B):
        rows = rows_of(cache, table[b], lens[b], scale)
        q = torch.cat((q_nope[b], q_pe[b]), -1).double().reshape(n * H, -1)
        limit = lens[b] - (n - 1) + torch.arange(n, device=q.device).repeat_interleave(H)
        parts.append([x.reshape((n, H) + x.shape[1:]) for x in softmax_rows(q, rows, rows[:, :512], sm_scale, limit, q_nope.dtype)])
    return [torch.stack(x) for x in zip(*parts)]


def prefill(q, k_nope, k_pe, v, cu_q, cu_k, sm_scale, causal):
    """Lists of bounds -> (out, lse, tolerances) of the queries that a sequence has, [cu_q[-1], H, ..]."""
    H = q.shape[1]
    parts = []
    for a, b, c, d in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        limit = torch.arange(b - a, device=q.device) + (d - c) - (b - a) + 1 if causal else torch.full((b - a,), d - c, device=q.device)
        heads = [softmax_rows(q[a:b, h].double(), torch.cat((k_nope[c:d, h], k_pe[c:d]), -1).double(), v[c:d, h].double(), sm_scale, limit, q.dtype)
                 for h in range(H)]
        parts.append([torch.stack(x, dim=1) for x in zip(*heads)])
    return [torch.cat(x) for x in zip(*parts)]


def rotate(x, cos_sin, neox):
    """x [.., 64], cos_sin [.., 64], float64."""
    cos, sin = cos_sin[..., :32], cos_sin[..., 32:]
    out = torch.empty_like(x)
    first = slice(0, 32) if neox else slice(0, None, 2)
    second = slice(32, 64) if neox else slice(1, None, 2)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size = torch.empty_like(x)
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size  # and what a float32 error is relative to
