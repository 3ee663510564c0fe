"""Blocks of 128 with a float32 scale each, in 64 bits, for the tests."""

import torch

B = 128


def plain_codes(x, rows):
    """Codes (as their values) and scales of x [R, K] by blocks of `rows` x 128: the definition, a block at a time."""
    R, K = x.shape
    codes = torch.empty((R, K), dtype=torch.float64)
    scales = torch.empty((-(-R // rows), -(-K // B)), dtype=torch.float32)
    x = x.cpu().double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            tile = x[i * rows:(i + 1) * rows, j * B:(j + 1) * B]
            a = torch.clamp(tile.abs().max(), min=2.0 ** -100)
            scales[i, j] = (a / 448).float()
            codes[i * rows:(i + 1) * rows, j * B:(j + 1) * B] = nearest_e4m3(448 * tile / a)
    return codes, scales


def nearest_e4m3(q):
    """The e4m3 nearest to q (up to 448), ties to the even one: steps of 2^-9 below 2^-6, else 2^-3 of the leading bit."""
    m, _ = torch.frexp(q)
    step = torch.where(q == 0, torch.zeros_like(q), q / m / 16).clamp(min=2.0 ** -9)
    return torch.round(q / step) * step


def values_of(codes, scales, rows):
    """What codes [.., R, K] and scales [.., R / rows, K / 128] stand for, in 64 bits."""
    R, K = codes.shape[-2:]
    return codes.double() * scales.double().repeat_interleave(rows, -2)[..., :R, :].repeat_interleave(B, -1)[..., :K]


def as_blocks(w):
    """A BlockMatrix of w from the definition's codes (a stack by its matrices)."""
    from rust_llm_inference_server_b200 import ops
    parts = [plain_codes(m, B) for m in (w if w.dim() == 3 else [w])]
    codes, scales = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    if w.dim() == 2:
        codes, scales = codes[0], scales[0]
    room = torch.zeros(codes.shape[:-1] + (-(-codes.shape[-1] // 16) * 16,), dtype=torch.float8_e4m3fn, device=w.device)
    room[..., :codes.shape[-1]] = codes.to(w.device).float().to(torch.float8_e4m3fn)
    return ops.BlockMatrix(room[..., :codes.shape[-1]], scales.to(w.device))
