"""The 4-bit KV cache in 64 bits, from its definition: quantisation, the byte
address of every (token, channel), norm + rotary, and attention."""
import numpy as np
import torch

D, PAGE = 128, 256


def _addresses():
    t = torch.arange(PAGE)[:, None]
    c = torch.arange(D)[None, :]
    g, r, pair = c // 32, c % 32, t // 2
    k = t * 64 + (r // 8) * 16 + g * 4 + (r % 8) // 4 * 2 + (r % 4) // 2
    v = pair * 128 + ((r // 4) ^ (2 * (pair % 4))) * 16 + g * 4 + t % 2 * 2 + (r % 4) // 2
    return k, v, (4 * (c % 2)).expand(PAGE, D)


K_BYTE, V_BYTE, SHIFT = _addresses()


def read(codes, scales, byte):
    """Values (float64 [pages, heads, 256, 128]) that a cache tensor pair holds."""
    flat = codes.cpu().flatten(2)
    nibble = (flat[:, :, byte].int() >> SHIFT) & 15
    return (nibble.double() - 8) * scales.cpu().double().repeat_interleave(32, -1)


def read_k(cache):
    return read(cache.k_codes, cache.k_scales, K_BYTE)


def read_v(cache):
    return read(cache.v_codes, cache.v_scales, V_BYTE)


def bf16_of(x):
    """Round float64 to BF16 in one step (round-half-even on the exact value)."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(all="ignore"):
        m, e = np.frexp(x)
        step = np.ldexp(1.0, np.maximum(e - 8, -133))
        return np.where(np.isfinite(x) & (x != 0), np.rint(x / step) * step, x)


def quantise(x):
    """(codes int8 [..., 128], scales float64 [..., 4]) of float32 / float64 values."""
    g = np.asarray(x.double()).reshape(*x.shape[:-1], 4, 32)
    top = np.abs(g).max(-1)
    scale = np.maximum(bf16_of(top / 7), 2.0 ** -126)
    scale = np.where(top == 0, 1.0, scale)
    scale = np.where(np.isfinite(top), scale, np.nan)
    with np.errstate(all="ignore"):
        codes = np.clip(np.rint(g / scale[..., None]), -7, 7)
    return torch.from_numpy(codes.reshape(x.shape)), torch.from_numpy(scale)


def pack(codes, scales, device):
    """Kv4Cache halves from codes [pages, heads, 256, 128] in [-7, 7]: (k_codes, v_codes) bytes."""
    out = []
    for byte in (K_BYTE, V_BYTE):
        flat = torch.zeros(*codes.shape[:2], PAGE * 64, dtype=torch.int32)
        nib = ((codes.int() + 8) << SHIFT).int()
        flat.scatter_add_(2, byte.reshape(1, 1, -1).expand(*codes.shape[:2], -1), nib.flatten(2))
        out.append(flat.to(torch.uint8).view(*codes.shape[:2], PAGE, 64).to(device))
    return out


def norm_rope(x, w, cos_sin, positions, eps):
    """float64 RMSNorm then rotary of [T, H, 128]."""
    x = x.double().cpu()
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
    cos, sin = cos_sin.double().cpu()[positions.cpu()].unsqueeze(1).chunk(2, -1)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def attention(q, k, v, tables, lens, scale):
    """(out, sum p |v|) in float64 [B, Hq, 128]; k, v float64 [pages, heads, 256, 128]."""
    q, tables = q.double().cpu(), tables.cpu().long()
    b, hq, _ = q.shape
    hkv = k.shape[1]
    out, size = torch.zeros(b, hq, D, dtype=torch.float64), torch.zeros(b, hq, D, dtype=torch.float64)
    for i, n in enumerate(lens):
        if n <= 0:
            continue
        page = tables[i, :(n + PAGE - 1) // PAGE]
        kk = k[page].transpose(0, 1).reshape(hkv, -1, D)[:, :n]
        vv = v[page].transpose(0, 1).reshape(hkv, -1, D)[:, :n]
        p = torch.softmax(torch.einsum("hgd,htd->hgt", q[i].view(hkv, hq // hkv, D), kk) * scale, -1)
        out[i] = torch.einsum("hgt,htd->hgd", p, vv).reshape(hq, D)
        size[i] = torch.einsum("hgt,htd->hgd", p, vv.abs()).reshape(hq, D)
    return out, size


def assert_attention_close(got, ref, size):
    """The output's rounding to BF16 is off by 2^-8 |ref| at most, that of each
    probability times its value's scale by 2^-8 of its share of sum p |v|; 2^-10
    of that sum covers what is held in FP32 (scores, exponentials, sums)."""
    got = got.double().cpu()
    bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -10) * size + 1e-30
    worst = ((got - ref).abs() / bound).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, worst
