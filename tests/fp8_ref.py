"""Plain 64-bit restatements of the block-scaled 8-bit formats for the tests."""
import torch

BLK = 128


def pad(x, dim):
    n = -x.shape[dim] % BLK
    if not n:
        return x
    shape = list(x.shape)
    shape[dim] = n
    return torch.cat([x, x.new_zeros(shape)], dim)


def exponent(amax):
    """Smallest e with amax <= 448 * 2^e (448 = 0.875 * 2^9), at least -127; 0 for no value."""
    m, ex = torch.frexp(amax)
    e = (ex - 9 + (m > 0.875).to(ex.dtype)).clamp(-127, 127)
    return torch.where(amax > 0, e, torch.zeros_like(e))


def _finite(x):
    return torch.where(torch.isfinite(x), x, torch.zeros_like(x))


def quantize(x, rows):
    """x [..,N,K] -> (e4m3, scale bytes) with 1 x 128 (rows) or 128 x 128 blocks, on x's device."""
    x = x.double()
    hi = 1 if rows else BLK
    p = pad(x, -1) if rows else pad(pad(x, -1), -2)
    lead, (n, k) = p.shape[:-2], p.shape[-2:]
    a = _finite(p).abs().reshape(*lead, n // hi, hi, k // BLK, BLK).amax(-1).amax(-2)
    e = exponent(a)
    full = e.repeat_interleave(hi, -2).repeat_interleave(BLK, -1)[..., :x.shape[-2], :x.shape[-1]]
    v = torch.ldexp(x, -full)
    v = torch.where(torch.isinf(v), torch.full_like(v, float("nan")), v)
    # |v| <= 448 has at most the bits of x, so going through fp32 rounds nothing that e4m3 keeps
    # (bf16 and fp32 inputs only)
    return v.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def values(q, scale_bytes, rows):
    """The 64-bit numbers that (q, scale) stand for."""
    hi = 1 if rows else BLK
    s = torch.exp2(scale_bytes.double() - 127)
    s = s.repeat_interleave(hi, -2).repeat_interleave(BLK, -1)
    return q.double() * s[..., :q.shape[-2], :q.shape[-1]]


def bytes_of(t):
    return t.view(torch.uint8)
