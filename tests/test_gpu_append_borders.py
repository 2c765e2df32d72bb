"""append_indexer_keys at the borders of e4m3's rounding: codes and scales bit for bit those of fp32's quotient x / scale, rounded to e4m3,
with scale = max(|x|, 1e-4) / 448 in fp32."""
import pytest
import torch

import paged_cases as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _codes(y):
    """From fp32 rows y [.., 128], on the host: IEEE divisions, and the conversion checked below against e4m3's values."""
    scale = y.abs().amax(dim=-1).clamp(min=1e-4) / torch.full((), 448.0)
    z = (y / scale.unsqueeze(-1)).clamp(-448, 448)
    return z.to(torch.float8_e4m3fn), scale


def _append(k, cos_sin=None, positions=None, interleaved=True, offset=0):
    """(codes, scales) that the call leaves as keys, and as queries."""
    from sparse_mla_sm120_b200 import paged
    t = len(k)
    k = k.to(DEV)
    ki, ks = torch.zeros(t, 128, device=DEV).to(torch.float8_e4m3fn), torch.zeros(t, device=DEV)
    rot = (None, None) if cos_sin is None else (positions.to(DEV), cos_sin.to(DEV))
    qi, w = paged.append_indexer_keys(k, ki, ks, torch.arange(t, device=DEV), *rot, interleaved=interleaved, rope_offset=offset, q=k.unsqueeze(1))
    return (ki.cpu(), ks.cpu()), (qi[:, 0].cpu(), w[:, 0].cpu())


def _same(got, codes, scale):
    for c, s in got:
        assert torch.equal(s.view(torch.int32), scale.view(torch.int32))
        wrong = c.view(torch.uint8) != codes.view(torch.uint8)
        assert not bool(wrong.any()), f"{int(wrong.sum())} codes differ"


def test_the_host_rounds_to_the_nearest_even_code():
    values = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middle = (values[1:] + values[:-1]) / 2
    even = torch.arange(0, 126) % 2 == 0
    got = lambda x: x.float().to(torch.float8_e4m3fn).view(torch.uint8).long()
    low = torch.arange(0, 126)
    assert torch.equal(got(middle), torch.where(even, low, low + 1))
    assert torch.equal(got(torch.nextafter(middle.float(), torch.zeros(126))), low)
    assert torch.equal(got(torch.nextafter(middle.float(), torch.full((126,), 1e9))), low + 1)


def test_every_mantissa_against_every_largest_value():
    """bf16 rows without rotation: all mantissas of a row's largest value by all mantissas of the others over twelve exponents: every tie that
    16-bit values can make, on either side of fp32's rounding of the scale and of the quotient."""
    top = torch.arange(128, 256).float()                                                  # mantissas 1.0 to 1.9921875
    rows = []
    for e in range(0, 12):
        x = top.view(1, 128, 1) * 2.0 ** -e * torch.ones(128, 1, 1)                       # [top, value, 1]
        x = x.view(128, 128).clone()
        x[x > top.unsqueeze(1)] /= 2                                                      # (not above the largest)
        x[:, 0] = top
        x[:, 1::2] *= -1
        rows.append(x)
    k = torch.cat(rows).to(torch.bfloat16)
    for shift in (0, -60, 90):
        ks = (k.float() * 2.0 ** shift).to(torch.bfloat16)
        _same(_append(ks), *_codes(ks.float()))


@pytest.mark.parametrize("interleaved,offset", [(True, 0), (False, 64)])
def test_quotients_next_to_the_borders(interleaved, offset):
    """Rotations whose sine is 0 make any fp32 value of a 1: for scales of all kinds, values whose quotient lies on the middle of two codes and
    up to four fp32 steps to either side, codes below the normal ones among them."""
    g = torch.Generator().manual_seed(3)
    t = 4096
    largest = torch.exp(torch.empty(t, dtype=torch.float64).uniform_(-8, 8, generator=g)).float()
    scale = largest / torch.full((), 448.0)
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middle = ((codes[1:] + codes[:-1]) / 2)[torch.randint(0, 126, (t, 32), generator=g)]
    x = (middle * scale.double().unsqueeze(1)).float()
    x = (x.view(torch.int32) + torch.randint(-4, 5, (t, 32), generator=g, dtype=torch.int32)).view(torch.float32)
    x[:, 0] = largest
    assert bool((x.abs() <= largest.unsqueeze(1)).all())
    table = torch.cat([x, torch.zeros(t, 32)], dim=1)
    k = torch.zeros(t, 128)
    sign = torch.where(torch.rand(t, 64, generator=g) < 0.5, -1.0, 1.0)
    k[:, offset:offset + 64] = sign
    y = torch.zeros(t, 128)
    y[:, offset:offset + 64] = sign * (x.repeat_interleave(2, dim=1) if interleaved else torch.cat([x, x], dim=1))
    # every quotient is one that a reciprocal may get wrong: within four steps of a border, or subnormal
    _same(_append(k.to(torch.bfloat16), table, torch.arange(t), interleaved, offset), *_codes(y))


@pytest.mark.parametrize("interleaved", [True, False])
def test_values_of_any_size(interleaved):
    """The same with values spread over codes at random, and rows whose scale is the least one."""
    g = torch.Generator().manual_seed(4)
    t = 4096
    x = torch.randn(t, 32, generator=g) * torch.exp(torch.randn(t, 1, generator=g) * 3)
    x[:64] *= 1e-6
    x[64:96] = 0
    table = torch.cat([x, torch.zeros(t, 32)], dim=1)
    k = torch.zeros(t, 128)
    k[:, :64] = 1
    y = torch.zeros(t, 128)
    y[:, :64] = x.repeat_interleave(2, dim=1) if interleaved else torch.cat([x, x], dim=1)
    _same(_append(k.to(torch.bfloat16), table, torch.arange(t), interleaved, 0), *_codes(y))
