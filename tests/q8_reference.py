"""What a matrix in 8 bits holds, in 64 bits and without the library: blocks of 128 elements of a
row share 2^e, e the smallest integer >= -127 with max|v| <= 448 * 2^e; an element is the e4m3
number nearest to v / 2^e, ties to the even code; infinities and NaN are NaN and count for no
maximum."""
import torch

# codes 0 .. 126: eighths of 2^-6, then eight steps an octave from 2^-6 to 448
E4M3 = torch.tensor([i * 2.0 ** -9 for i in range(8)] +
                    [(8 + i) * 2.0 ** (p - 10) for p in range(1, 16) for i in range(8)][:119],
                    dtype=torch.float64)
POWERS = torch.tensor([2.0 ** i for i in range(-127, 140)], dtype=torch.float64)


def held(v):
    """v (rows, K), any floating type -> (values (rows, K), powers (rows, blocks)) in 64 bits."""
    v = v.double().cpu()
    out, scales = torch.empty_like(v), []
    mids = (E4M3[:-1] + E4M3[1:]) / 2
    for k in range(0, v.shape[1], 128):
        b = v[:, k:k + 128]
        fin = torch.isfinite(b)
        top = torch.where(fin, b.abs(), torch.zeros_like(b)).amax(1)
        s = POWERS[torch.searchsorted(448.0 * POWERS, top)][:, None]
        a = (torch.where(fin, b.abs(), torch.zeros_like(b)) / s).contiguous()
        i = torch.searchsorted(mids, a)
        tie = (i < 126) & (mids[i.clamp(max=125)] == a)
        i = torch.where(tie & (i % 2 == 1), i + 1, i)
        h = torch.sign(b) * E4M3[i] * s
        out[:, k:k + 128] = torch.where(fin, h, torch.full_like(h, float("nan")))
        scales.append(s)
    return out, torch.cat(scales, 1)
