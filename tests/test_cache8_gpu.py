"""An 8-bit cache: records quantised as they are written and read back, against the rule in 64 bits.

Scales are powers of two, so everything but the one rounding to e4m3 is exact and the codes are compared bit by bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from hyperion_b200 import ops
from hyperion_b200.ops.cache8 import Cache8, cache8_load, cache8_store, new_cache8

pytestmark = pytest.mark.gpu
E4M3 = np.array([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127])  # codes 0 .. 126


def quantised(x: np.ndarray):
    """Codes (bytes) and exponents of records [..., d] by the rule, in 64 bits."""
    x = x.astype(np.float64)
    largest = np.where(np.isnan(x), 0.0, np.abs(x)).max(-1)
    e = np.full(largest.shape, 40)
    for k in range(39, -41, -1):
        e = np.where(largest <= 448.0 * 2.0 ** k, k, e)
    y = x / 2.0 ** e[..., None].astype(np.float64)
    size = np.minimum(np.where(np.isnan(y), 0.0, np.abs(y)), 448.0)
    below = np.searchsorted(E4M3, size, side="right") - 1
    above = np.minimum(below + 1, 126)
    gap = size - E4M3[below], E4M3[above] - size
    code = np.where((gap[0] < gap[1]) | ((gap[0] == gap[1]) & (below % 2 == 0)), below, above)
    code = np.where(size == E4M3[below], below, code)
    code = np.where(np.isnan(y), 127, code) | np.where(np.signbit(y) & ~np.isnan(y), 128, 0)
    return code.astype(np.uint8), e.astype(np.int8)


def places(tokens, page_size, rows, seed=0):
    random = np.random.default_rng(seed)
    each = -(-tokens // rows)
    blocks = -(-each // page_size)
    table = torch.from_numpy(random.permutation(rows * blocks + 3)[: rows * blocks].reshape(rows, blocks).astype(np.int32)).cuda()
    order = random.permutation(tokens)  # in no order
    return table, torch.from_numpy((order // each).astype(np.int32)).cuda(), torch.from_numpy((order % each).astype(np.int32)).cuda(), rows * blocks + 3


def stored(x, kv, dim, page_size, k_offset, v_offset, rows=3):
    table, row, position, pages = places(x.shape[0], page_size, rows)
    cache = new_cache8(pages, kv, page_size, dim)
    cache8_store(x, k_offset, v_offset, cache, table, row, position)
    ops.raise_on_status(x.device)
    of, slot = table[row.long(), position.long() // page_size].long(), position.long() % page_size
    return cache, (table, row, position), cache.codes.view(torch.uint8)[of, :, :, slot].cpu().numpy(), cache.exponents[of, :, :, slot].cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,kv,dim,page_size", [(1, 2, 64, 16), (7, 1, 128, 8), (333, 4, 128, 64), (50, 3, 96, 16), (20, 2, 8, 32), (9, 1, 256, 16), (20011, 4, 64, 16)])
def test_records_written_and_read_back(tokens, kv, dim, page_size, dtype):
    random = torch.Generator("cuda").manual_seed(tokens)
    width = kv * dim
    x = torch.randn(tokens, 3 * width, device="cuda", generator=random) * torch.exp2(4 * torch.randn(tokens, 3 * width, device="cuda", generator=random))
    x = x.to(dtype)
    cache, where, codes, exponents = stored(x, kv, dim, page_size, width, 2 * width)
    want_codes, want_exponents = quantised(x[:, width:].float().cpu().numpy().reshape(tokens, 2, kv, dim))
    assert (exponents == want_exponents).all()
    assert (codes == want_codes).all()
    values = np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])[want_codes] * 2.0 ** want_exponents[..., None].astype(np.float64)
    for result in (torch.bfloat16, torch.float32):
        assert (cache8_load(cache, *where, dtype=result).double().cpu().numpy() == values).all()
    assert np.abs(values - x[:, width:].double().cpu().numpy().reshape(values.shape)).max(-1).max() <= 2.0 ** -4 * np.abs(values).max()


@pytest.mark.parametrize("shift", [0, 1, 3])  # columns and rows off every boundary
def test_sources_off_boundaries(shift):
    whole = torch.randn(45, 2 * 128 + 2 * shift + 5, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    _, _, codes, exponents = stored(whole, 1, 128, 16, shift, 128 + 2 * shift)
    x = torch.stack([whole[:, shift: shift + 128], whole[:, 128 + 2 * shift: 256 + 2 * shift]], 1).float().cpu().numpy().reshape(45, 2, 1, 128)
    want = quantised(x)
    assert (codes == want[0]).all() and (exponents == want[1]).all()


def test_records_at_the_rule_s_edges():
    x = torch.zeros(12, 64, device="cuda")
    x[1, :3] = torch.tensor([448.0, -448.0, 1.0])             # the largest that exponent 0 holds
    x[2, :2] = torch.tensor([448.0001, 1.0])                  # the next exponent
    x[3, 0] = 1e-30                                           # below every exponent: reads as zero
    x[4, :2] = torch.tensor([3e38, 1.0])                      # beyond every exponent
    x[5, :3] = torch.tensor([float("inf"), -float("inf"), 2.0])
    x[6, :3] = torch.tensor([float("nan"), 5.0, -0.0])
    x[7, :] = float("nan")
    x[8, :4] = torch.tensor([256.0, 17.0, 19.0, 21.0])        # ties: 17 -> 16, 19 -> 20, 21 -> 20
    x[9, :2] = torch.tensor([448.0, 2.0 ** -10])              # half the smallest: to even, which is zero
    x[10, :2] = torch.tensor([448.0, 1.5 * 2.0 ** -9])
    x[11, 0] = -1.1754944e-38
    _, _, codes, exponents = stored(torch.cat([x, x.flip(1)], 1), 1, 64, 16, 0, 64)
    want = quantised(torch.stack([x, x.flip(1)], 1).cpu().numpy().reshape(12, 2, 1, 64))
    assert (exponents == want[1]).all()
    assert (codes == want[0]).all()
    assert list(exponents[:7, 0, 0]) == [-40, 0, 1, -40, 40, 40, -6]


def test_other_slots_and_pages_stay():
    cache = new_cache8(4, 2, 16, 64)
    cache.codes.view(torch.uint8).fill_(77)
    cache.exponents.fill_(5)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    x = torch.randn(1, 4 * 64, device="cuda")
    cache8_store(x, 0, 128, cache, table, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), 19, dtype=torch.int32, device="cuda"))
    touched = (cache.codes.view(torch.uint8) != 77).any(-1) | (cache.exponents != 5)
    assert touched.nonzero()[:, 0].unique().tolist() == [0] and touched.nonzero()[:, 3].unique().tolist() == [3]


def test_a_token_without_a_page_is_left_out_and_reported():
    cache = new_cache8(2, 1, 16, 64)
    table = torch.tensor([[1, -1]], dtype=torch.int32, device="cuda")
    row = torch.zeros(4, dtype=torch.int32, device="cuda")
    position = torch.tensor([3, 17, -1, 40], dtype=torch.int32, device="cuda")
    x = torch.randn(4, 128, device="cuda")
    cache8_store(x, 0, 64, cache, table, row, position)
    with pytest.raises(ops.KernelError, match="block-table"):
        ops.raise_on_status(x.device)
    back = cache8_load(cache, table, row, position, dtype=torch.float32)
    with pytest.raises(ops.KernelError, match="block-table"):
        ops.raise_on_status(x.device)
    assert back[0].abs().max() > 0 and (back[1:] == 0).all()
    assert (cache.codes.float()[0] == 0).all()


def test_positions_behind_32_bit_offsets():
    """Pages whose codes start beyond 2^31 and 2^32 bytes."""
    pages = 2**32 // (2 * 8 * 64 * 128) + 40
    cache = Cache8(torch.empty((pages, 2, 8, 64, 128), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.empty((pages, 2, 8, 64), dtype=torch.int8, device="cuda"))
    table = torch.tensor([[pages - 1, pages // 2 + 3, 0]], dtype=torch.int32, device="cuda")
    position = torch.arange(0, 190, 3, dtype=torch.int32, device="cuda")
    x = torch.randn(len(position), 2 * 8 * 128, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(torch.bfloat16)
    row = torch.zeros_like(position)
    cache8_store(x, 0, 8 * 128, cache, table, row, position)
    ops.raise_on_status(x.device)
    values = cache8_load(cache, table, row, position, dtype=torch.float32).cpu().numpy().astype(np.float64)
    codes, exponents = quantised(x.float().cpu().numpy().reshape(-1, 2, 8, 128))
    assert (values == np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])[codes] * 2.0 ** exponents[..., None].astype(np.float64)).all()


def test_on_another_stream():
    stream = torch.cuda.Stream()
    x = torch.randn(300, 256, device="cuda").to(torch.bfloat16)
    table, row, position, pages = places(300, 16, 2)
    first, second = new_cache8(pages, 2, 16, 64), new_cache8(pages, 2, 16, 64)
    cache8_store(x, 0, 128, first, table, row, position)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        cache8_store(x, 0, 128, second, table, row, position)
        back = cache8_load(second, table, row, position)
    stream.synchronize()
    assert torch.equal(first.codes.view(torch.uint8), second.codes.view(torch.uint8)) and torch.equal(back, cache8_load(first, table, row, position))


def test_nothing_to_do():
    cache = new_cache8(1, 1, 16, 64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cache8_store(torch.empty(0, 128, device="cuda"), 0, 64, cache, table, none, none)
    assert cache8_load(cache, table, none, none).shape == (0, 2, 1, 64)


def test_refusals():
    cache = new_cache8(2, 1, 16, 64)
    table, row, position = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    x = torch.randn(3, 128, device="cuda")
    for bad in (dict(src=x.half()), dict(src=x[:2]), dict(src=x.t().contiguous().t()), dict(k_offset=65), dict(v_offset=-1), dict(src=x.cpu()), dict(positions=position.long()),
                dict(token_row=row[:2]), dict(block_table=table.long()), dict(block_table=table[0]), dict(cache=Cache8(cache.codes, cache.exponents[:, :1])),
                dict(cache=Cache8(cache.codes.view(torch.uint8), cache.exponents)), dict(cache=Cache8(cache.codes.transpose(2, 3), cache.exponents.transpose(2, 3)))):
        with pytest.raises(ops.KernelError):
            cache8_store(**{**dict(src=x, k_offset=0, v_offset=64, cache=cache, block_table=table, token_row=row, positions=position), **bad})
    with pytest.raises(ops.KernelError):
        cache8_load(cache, table, row, position, dtype=torch.float16)
    with pytest.raises(ops.KernelError):
        cache8_load(cache, table, row, position, out=torch.empty(3, 2, 1, 64, device="cuda"))
    with pytest.raises(ops.KernelError):
        new_cache8(1, 1, 16, 20)
