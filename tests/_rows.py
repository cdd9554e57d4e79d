"""Rows of numbers for the tests of norms and token exchanges: device tensors with guard bytes around and between the rows."""
import ctypes

import torch

import aws_ofi_nccl_amd as m

TYPES = {"bf16": (torch.bfloat16, m.BFLOAT16, 2.0 ** -8), "f16": (torch.float16, m.FLOAT16, 2.0 ** -11),
         "f32": (torch.float32, m.FLOAT32, 2.0 ** -24)}   # torch's type, the number, the unit roundoff
U32 = 2.0 ** -24
GUARD = 0xA5


class Rows:
    """n rows of `width` elements, `pad` elements apart beyond the width, `shift` elements into an allocation filled with
    guard bytes (Rows.guard).  .t is the tensor of the rows; untouched() tells whether every byte outside them is as it was."""

    guard = GUARD

    def __init__(self, n, width, dtype, pad=0, shift=0, values=None):
        size = torch.empty((), dtype=dtype).element_size()
        self.n, self.width, self.pad, self.pitch = n, width, pad, (width + pad) * size
        count = shift + n * (width + pad) + 64
        self.bytes = torch.full((count * size,), self.guard, dtype=torch.uint8, device="cuda")
        self.shift = shift
        whole = self.bytes.view(dtype) if size > 1 else self.bytes.view(torch.uint8).view(dtype)
        self.t = whole[shift:shift + n * (width + pad)].view(n, width + pad)[:, :width] if n else whole[:0].view(0, max(1, width))
        self.size = size
        if values is not None and n:
            self.t.copy_(values)

    def ptr(self):
        return self.bytes.data_ptr() + self.shift * self.size

    def untouched(self):
        rest = self.bytes.clone()
        if self.n:
            lo = self.shift * self.size
            rest[lo:lo + self.n * self.pitch].view(self.n, self.pitch)[:, :self.width * self.size] = self.guard
        return bool((rest == self.guard).all())


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def within(got, want, bound):
    """|got - want| <= bound in 64 bits, a NaN only where a NaN is wanted, infinities the same."""
    got, want = got.double().cpu(), want.double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(want)
    bad = torch.isnan(got) != torch.isnan(want)
    both = ~torch.isnan(got) & ~torch.isnan(want)
    far = both & (got != want) & ~((got - want).abs() <= bound)
    bad = bad | far
    if bool(bad.any()):
        at = torch.nonzero(bad)[0].tolist()
        raise AssertionError("%d of %d values off; first at %s: got %r, want %r, bound %r" % (
            int(bad.sum()), bad.numel(), at, got[tuple(at)].item(), want[tuple(at)].item(), bound[tuple(at)].item()))
