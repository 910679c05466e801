"""Block-sparse 8-bit matrices from their definition, in 64 bits (torch, any device), for the tests of asp_b200_block8.h."""
import torch

BLOCK = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def blocks(n):
    return -(-n // BLOCK)


def groups_in_8_bits(v):
    """v: [groups, elements] of 32 bits at most; what e4m3 with a power-of-two scale for each group stands for, in 64 bits."""
    v = v.double()
    finite = torch.isfinite(v)
    most = torch.where(finite, v.abs(), 0.0).amax(1, keepdim=True)
    m, e = torch.frexp(most / 448.0)  # in (0, 1]: 2^(e - 1) < most / 448 <= 2^e unless m = 1/2
    k = (e - (m == 0.5).int()).clamp(min=-126)
    q = torch.ldexp(torch.where(finite, v, 0.0), -k)
    step = torch.ldexp(torch.ones_like(q), (torch.frexp(q).exponent - 1).clamp(min=-6) - 3)
    return torch.where(finite, torch.ldexp(torch.round(q / step) * step, k), float("nan"))  # (round: ties to even)


def rows_in_8_bits(x):
    n, c = x.shape
    full = torch.zeros(n, blocks(c) * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :c] = x.double()
    return groups_in_8_bits(full.reshape(-1, BLOCK)).reshape(n, -1)[:, :c]


def dense(pattern, shape, values):
    """values [n, 128, 128] at pattern = (block_ptr, block_col) -> the matrix, in the values' type."""
    ptr, col = pattern
    out = torch.zeros(blocks(shape[0]) * BLOCK, blocks(shape[1]) * BLOCK, dtype=values.dtype, device=values.device)
    for r in range(len(ptr) - 1):
        for j in range(int(ptr[r]), int(ptr[r + 1])):
            c = int(col[j])
            out[r * BLOCK : (r + 1) * BLOCK, c * BLOCK : (c + 1) * BLOCK] = values[j]
    return out[: shape[0], : shape[1]]


def stored(pattern, full):
    """The blocks of a matrix that the pattern has, [n, 128, 128], zero where they stick out."""
    ptr, col = pattern
    pad = torch.nn.functional.pad(full, (0, -full.shape[1] % BLOCK, 0, -full.shape[0] % BLOCK))
    got = [pad[r * BLOCK : (r + 1) * BLOCK, int(col[j]) * BLOCK : (int(col[j]) + 1) * BLOCK] for r in range(len(ptr) - 1) for j in range(int(ptr[r]), int(ptr[r + 1]))]
    return torch.stack(got) if got else pad.new_zeros(0, BLOCK, BLOCK)
