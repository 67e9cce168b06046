"""What random values of one size do not show of the speculative decoding step's operators (test_speculative.py): parts of a
sequence without any row that exists.

Bounds are those of test_speculative.py, with the roundings that a test's exact values do not make left out."""
import math

import pytest
import torch

from test_serving import DT, U, Cache, cu_of, gen, half_step, ints, normal, within
from test_speculative import H16, ref_tree


# ------------------------------------------------------------------ tree
def held_rows(table, n, n_pages):
    """Which of a sequence's n rows lie on pages that exist."""
    return [r for r in range(n) if 0 <= table[r // 64] < n_pages]


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("low", [-1.0, -20.0, -110.0])
@pytest.mark.parametrize("many", [False, True])
def test_attention_tree_of_rows_behind_missing_pages(rrr, ctx, hd, kind, low, many):
    """A sequence's first pages do not exist, and the scores of all other rows are far below 0. One sequence is shared by
    CTAs block by block, of many some are a CTA's own. Keys are constant over a head, in few bits: 16-bit types, the cache
    and the operands hold them, so a score carries the sums' error alone."""
    t, g, nh, nkv, nodes = DT[kind], gen(hd), 2, 1, 3
    lens = [300, 64, 130, 520, 1] * 40 if many else [520]
    gone = [[0, 1], [0], [0, 1], [0, 1, 2, 3, 5], [0]] * 40 if many else [[0, 1, 2]]
    cache, cu = Cache(rrr, ctx, nkv, hd, lens, 3), cu_of(lens)
    n_pages = cache.pages.shape[0]
    row = torch.cat([torch.arange(n, device="cuda") for n in lens]).float()
    step = 2.0 ** math.floor(math.log2(-low)) / 32  # six bits
    level = round(low / step) * step
    k = (level + step * (row % 4))[:, None, None].expand(-1, nkv, hd).contiguous()  # scores of low .. low + 3 steps
    v = normal(g, sum(lens), nkv, hd)
    cache.c.store(k, v, cu, ints(lens))
    cache.c.load(cu, ints(lens), k, v)
    table = cache.c.page_table.cpu().numpy().copy()
    for s, pages in enumerate(gone):
        table[s, pages] = [n_pages + 5 if i % 2 else -3 for i in range(len(pages))]
    cache.c.page_table.copy_(torch.from_numpy(table))
    rows = nodes * len(lens)
    q = torch.full((rows, nh, hd), 1.0 / hd, dtype=t, device="cuda")
    kd = torch.full((rows, nkv, hd), level, dtype=t, device="cuda")
    vd = normal(g, rows, nkv, hd, dtype=t)
    out, tree = torch.empty(rows, nh, hd, dtype=t, device="cuda"), [-1, 0, 0]
    cache.c.attention_tree(q, kd, vd, cu_of([nodes] * len(lens)), ints(tree * len(lens)), ints(lens), out,
                           cache.c.tree_workspace(nh, rows), scale=1.0)
    assert ctx.device_error() == 6
    a, h = 0, half_step(t)
    for s, n in enumerate(lens):
        r, held = slice(nodes * s, nodes * (s + 1)), held_rows(table[s], n, n_pages)
        kc, vc = (x[a:a + n][held].double() for x in (k, v))
        ref, A, _ = ref_tree(q[r].double(), kd[r].double(), vd[r].double(), kc, vc, tree, 1.0)
        top = max(float(vd[r].abs().max()), float(vc.abs().max()) if held else 0.0)
        bound = (2 * torch.expm1(2 * (hd + 16) * U * A) + 2 * H16 + h + 64 * U) * top
        within(out[r], ref, ref.abs() * h * 1.01 + bound[..., None] + 2.0 ** -25)
        a += n
