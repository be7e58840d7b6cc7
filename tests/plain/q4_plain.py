"""Weights of 4 bits in plain code: the stored form by its definition, quantization in float64."""
import numpy as np
import torch


def unpack(w):
    """(codes [n, k], scales [n, g], zeros [n, g] or None: 8) of a stored matrix, bit by bit from the description of the form."""
    n, k, group = w.n, w.k, w.group
    data = w.data.cpu().numpy()
    groups, size = 128 // group, w.scale_dtype.itemsize
    words = np.ascontiguousarray(data[:, :, :8192]).view(np.uint32).reshape(data.shape[0], data.shape[1], 4, 128, 4)
    nn, kk = np.meshgrid(np.arange(n), np.arange(k), indexing="ij")
    r = kk % 8
    bit = 16 * (r % 2) + 8 * (r // 4) + 4 * ((r // 2) % 2)
    codes = (words[nn // 128, kk // 128, (kk % 128) // 32, nn % 128, (kk % 32) // 8] >> bit.astype(np.uint32)) & 15
    at = 8192 + groups * 128 * size
    scales = torch.from_numpy(np.ascontiguousarray(data[:, :, 8192:at])).view(w.scale_dtype).reshape(data.shape[0], data.shape[1], groups, 128)
    nn, gg = np.meshgrid(np.arange(n), np.arange(-(-k // group)), indexing="ij")
    pick = lambda t: t[nn // 128, gg // groups, gg % groups, nn % 128]                  # noqa: E731
    zeros = torch.from_numpy(pick(data[:, :, at:].reshape(data.shape[0], data.shape[1], groups, 128)).astype(np.int64)) if w.zeros else None
    return torch.from_numpy(codes.astype(np.int64)), pick(scales), zeros


def values(w):
    """[n, k] float64."""
    codes, scales, zeros = unpack(w)
    spread = lambda t: t.repeat_interleave(w.group, dim=1)[:, :w.k]                      # noqa: E731
    return spread(scales.double()) * (codes - (spread(zeros) if zeros is not None else 8)).double()


def quantized(m, group, zeros, scale_dtype):
    """(codes, scales, zeros or None) of a matrix, group by group in float64."""
    m = m.cpu().double()
    n, k = m.shape
    codes, scales, zs = torch.empty((n, k), dtype=torch.int64), [], []
    for at in range(0, k, group):
        v = m[:, at:at + group]
        fine = torch.isfinite(v).all(dim=1)
        v = torch.where(fine[:, None], v, 0.0)
        lo, hi = v.amin(1).clamp_max(0), v.amax(1).clamp_min(0)
        s = ((hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7).float().to(scale_dtype).double()
        safe = torch.where(s > 0, s, 1.0)
        q = torch.where((s > 0)[:, None], torch.round(v / safe[:, None]), 0.0)
        z = torch.where(s > 0, torch.round(-lo / safe), 0.0).clamp(0, 15)
        codes[:, at:at + group] = ((q + z[:, None]).clamp(0, 15) if zeros else q.clamp(-7, 7) + 8).long()
        scales.append(torch.where(fine, s, float("nan")).to(scale_dtype))
        zs.append(z.long())
    return codes, torch.stack(scales, 1), torch.stack(zs, 1) if zeros else None
