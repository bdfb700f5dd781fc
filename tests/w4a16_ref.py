"""Plain 64-bit forms of the weight-only operators, and inputs whose sums f32 holds exactly.

Exact inputs: activations are whole numbers up to 7, block scales powers of two from 1/4 to 2; then every product is a multiple of 1/8 and of at most
84, and a sum over k up to 4096 needs fewer than 24 bits, so that f32 sums are exact in whatever order they are taken."""
import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def values(codes, block, g):
    """f64 values of [E,N,K/2] codes, [E,N,K/16] scale bytes and [E,N] (or broadcastable) factors."""
    nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = MAGNITUDES.to(codes.device)[nib & 7] * torch.where(nib >= 8, -1.0, 1.0).double()
    return v * block.view(torch.float8_e4m3fn).double().repeat_interleave(16, -1) * g[..., None].double()


def make_weight(E, N, K, seed, exact=True, device="cuda"):
    """(codes u8 [E,N,K/2], scale bytes u8 [E,N,K/16]) with every code; scales powers of two, or any that are finite."""
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (E, N, K // 2), generator=gen, dtype=torch.uint8)
    if exact:
        block = torch.randint(5, 9, (E, N, K // 16), generator=gen, dtype=torch.uint8) * 8     # 2^(e - 7)
    else:
        block = torch.randint(0, 127, (E, N, K // 16), generator=gen, dtype=torch.uint8)
        block |= (torch.rand(block.shape, generator=gen) < 0.1).to(torch.uint8) * 128
    return codes.to(device), block.to(device)


def make_x(M, K, seed, dtype, exact=True, pad=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed + 1)
    x = torch.randint(-7, 8, (M, K + pad), generator=gen).double() if exact else torch.randn(M, K + pad, generator=gen).double()
    return x.to(dtype).to(device)[:, :K]


def moe(x, weights, ids, emap, w13, w2, on_input=False):
    """(out, size): the layer in 64 bits, and the same sum over magnitudes from the second projection on.  w13 [E,2I,H], w2 [E,H,I] values."""
    E, I = w13.shape[0], w13.shape[1] // 2
    out = torch.zeros(x.shape[0], w2.shape[1], dtype=torch.float64, device=x.device)
    size = out.clone()
    ids = ids.tolist()
    for m in range(x.shape[0]):
        for s, e in enumerate(ids[m]):
            if emap is not None:
                e = int(emap[e]) if 0 <= e < emap.numel() else -1
            if not 0 <= e < E:
                continue
            w = float(weights[m, s])
            h = w13[e] @ x[m].double() * (w if on_input else 1.0)
            a = h[:I] / (1.0 + torch.exp(-h[:I])) * h[I:]
            f = 1.0 if on_input else w
            out[m] += f * (w2[e] @ a)
            size[m] += abs(f) * (w2[e].abs() @ a.abs())
    return out, size
