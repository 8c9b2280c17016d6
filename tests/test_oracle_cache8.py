"""The 64-bit restatement of the 8-bit cache: its E4M3 numbers against torch's float8 casts, and its scales."""
import torch

from oracle import cache8 as oc


def test_codes_are_those_of_torch():
    every = torch.arange(256, dtype=torch.uint8)
    want = every.view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.nan_to_num(oc.VALUES, nan=1e9), torch.nan_to_num(want, nan=1e9))
    x = torch.cat([want[torch.isfinite(want)], torch.randn(4000, generator=torch.Generator().manual_seed(1)).double() * 60,
                   torch.arange(-448 * 64, 448 * 64 + 1).double() / 64, torch.arange(-64, 65).double() * 2.0 ** -12]).clamp(-448, 448)
    codes = oc.encode(x)
    assert torch.equal(oc.VALUES[codes.long()], x.float().to(torch.float8_e4m3fn).double())
    assert oc.encode(torch.tensor([float("nan"), float("inf"), -float("inf")]).double()).tolist() == [127, 127, 255]


def test_scales_are_the_smallest_powers_of_two():
    for top, want in ((448.0, 1.0), (448.1, 2.0), (1.75, 2.0 ** -8), (1.7500001, 2.0 ** -7), (0.0, 2.0 ** -126), (3e38, 2.0 ** 120)):
        assert oc.scale_of(torch.tensor([0.1 * top, -top, float("nan"), float("inf")], dtype=torch.float64)) == want
