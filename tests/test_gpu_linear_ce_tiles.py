"""linear_cross_entropy where its products take the largest tiles, several pieces of the vocabulary, and more rows than a share of the weight's gradient may hold; which kernels ran is asked
of the profiler, so that another choice of tiles does not leave these untested."""
import re

import pytest
import torch

from tests.test_gpu_linear_ce import check, inputs, run, up_of

pytestmark = pytest.mark.gpu


def launched(call):
    """call()'s result and its kernels: ce_<name> -> (template arguments, launches)"""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as profile:
        result = call()
        torch.cuda.synchronize()
    kernels = {}
    for event in profile.events():
        found = re.search(r'sa2::(ce_\w+)<([^>]*)>', event.name)
        if found:
            arguments = tuple(found[2].replace(' ', '').split(','))
            kernels[found[1], arguments] = kernels.get((found[1], arguments), 0) + 1
    return result, kernels


def count(kernels, name, *arguments):
    return sum(n for (at, given), n in kernels.items() if at == name and given[:len(arguments)] == arguments)


TYPES = [(torch.bfloat16, '0'), (torch.float16, '1')]


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('dtype,code', TYPES, ids=['bf16', 'fp16'])
@pytest.mark.parametrize('rows,dim,vocab', [(3900, 2056, 3901), (3841, 2061, 4090)])
def test_tiles_of_256(rows, dim, vocab, dtype, code, reduction):
    """All four products in tiles of 256 x 256 whose last ones are ragged in every direction; the second shape's rows are copied."""
    hidden, weight, targets = inputs(rows, dim, vocab, dtype)
    up = up_of(reduction, rows)
    got, kernels = launched(lambda: run(hidden, weight, targets, reduction, up))
    for name in ('ce_logits_kernel', 'ce_dz_kernel', 'ce_dh_kernel', 'ce_dw_kernel'):
        assert count(kernels, name, code, '4', '4') == 1, kernels
    check(hidden, weight, targets, reduction, up, got)
    for a, b in zip(got, run(hidden, weight, targets, reduction, up)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype,code,reduction,pieces', [(torch.bfloat16, '0', 'mean', 2), (torch.float16, '1', 'sum', 2), (torch.float16, '1', 'none', 3)], ids=['bf16', 'fp16', 'fp16_none'])
def test_pieces_of_wide_rows(dtype, code, reduction, pieces):
    """The rows' gradients are added to those of the pieces before in a launch of their own, and the weight's are in shares."""
    rows, dim, vocab = 16400, 2056, 8201
    hidden, weight, targets = inputs(rows, dim, vocab, dtype)
    up = up_of(reduction, rows)
    got, kernels = launched(lambda: run(hidden, weight, targets, reduction, up))
    assert count(kernels, 'ce_dz_kernel', code, '4', '4') == count(kernels, 'ce_dh_kernel', code, '4', '4') == count(kernels, 'ce_dw_kernel', code, '4', '4') == pieces, kernels
    check(hidden, weight, targets, reduction, up, got)
    for a, b in zip(got, run(hidden, weight, targets, reduction, up)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype,reduction', [(torch.bfloat16, 'mean'), (torch.float16, 'none')], ids=['bf16', 'fp16_none'])
def test_more_rows_than_65536(dtype, reduction):
    rows = 70001
    hidden, weight, targets = inputs(rows, 8, 40, dtype)
    up = up_of(reduction, rows)
    check(hidden, weight, targets, reduction, up, run(hidden, weight, targets, reduction, up))
