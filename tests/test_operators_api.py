"""Argument checks of the operators around the GEMMs, through the C ABI and the Python layer (nothing is launched)."""
import ctypes

import pytest
import torch

import deep_gemm
from deep_gemm import _lib
from oracle import moe as om, mx as ox


@pytest.fixture(scope='module')
def lib():
    return _lib.load()


def _layout(tokens=2, topk=2, groups=4, rows=64, alignment=32, ptr=4096):
    return _lib.MoELayoutArgs(tokens, topk, groups, rows, alignment, ptr, ptr, ptr, ptr)


def _refused(lib, rc, text):
    assert rc == -1 and text in lib.dg_last_error().decode(), lib.dg_last_error()


def test_sort_refusals(lib):
    sort = lambda layout, ids=4096, size=4, ws=None, n=0: lib.dg_moe_sort(ids, size, layout, ws, n, 0, None)
    _refused(lib, sort(None), 'null layout')
    _refused(lib, sort(_layout(), size=2), 'int32 or int64')
    _refused(lib, sort(_layout(groups=0)), '1024 groups')
    _refused(lib, sort(_layout(groups=1025)), '1024 groups')
    _refused(lib, sort(_layout(rows=65)), 'multiple of the alignment')
    _refused(lib, sort(_layout(alignment=0)), 'multiple of the alignment')
    _refused(lib, sort(_layout(), ids=None), 'null tensor')
    _refused(lib, sort(_layout(ptr=None)), 'null tensor')
    _refused(lib, sort(_layout(tokens=-1)), 'invalid size')
    _refused(lib, sort(_layout(tokens=1 << 20, topk=1 << 12)), 'invalid size')
    _refused(lib, sort(_layout(tokens=1 << 28, topk=4, groups=1024, rows=0, alignment=1 << 21)), 'too many rows')
    _refused(lib, sort(_layout(tokens=1 << 15, topk=8)), 'workspace')
    need = ctypes.c_int64()
    assert lib.dg_moe_sort_workspace_size(128, 256, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.dg_moe_sort_workspace_size(1 << 18, 256, ctypes.byref(need)) == 0 and need.value > 0
    _refused(lib, lib.dg_moe_sort_workspace_size(-1, 4, ctypes.byref(need)), 'invalid size')


@pytest.mark.parametrize('pairs,rows_of_counts', [(8192, 0), (8193, 5), (1 << 21, 256), ((1 << 21) + 1, 258), (1 << 26, 8193)])
def test_sort_workspace(lib, pairs, rows_of_counts):
    """Counts of every block and, past 256 blocks, their sums."""
    need = ctypes.c_int64()
    assert lib.dg_moe_sort_workspace_size(pairs, 300, ctypes.byref(need)) == 0
    assert need.value == rows_of_counts * 300 * 4


def test_movement_refusals(lib):
    d = lambda layout=None, src=4096, sld=64, rb=64, dst=4096, dld=64, sf=None, sfo=None, oload=64: lib.dg_moe_dispatch(
        src, sld, rb, layout or _layout(), dst, dld, sf, 2, 1, sfo, oload, 1, 0, None)
    _refused(lib, d(sld=32), 'leading dimension')
    _refused(lib, d(dld=32), 'leading dimension')
    _refused(lib, d(src=None), 'null tensor')
    _refused(lib, d(dst=None), 'null tensor')
    _refused(lib, d(sf=4096, sfo=4096, oload=65), 'scale factors')
    _refused(lib, d(sf=4096, sfo=None), 'scale factors')
    c = lambda dtype=0, rows=4096, ld=64, out=4096: lib.dg_moe_combine(rows, ld, dtype, 64, _layout(), None, out, 64, 0, None)
    _refused(lib, c(dtype=2), 'bf16 or fp32')
    _refused(lib, c(ld=8), 'leading dimension')
    _refused(lib, c(rows=None), 'null tensor')
    _refused(lib, c(out=None), 'null tensor')
    b = lambda w=4096, dtype=1, ld=64: lib.dg_moe_combine_backward(4096, 64, 4096, ld, dtype, 64, _layout(), w, 4096, 64, 4096, 0, None)
    _refused(lib, b(w=None), 'null tensor')
    _refused(lib, b(dtype=2), 'bf16 or fp32')
    _refused(lib, b(ld=63), 'leading dimension')
    # nothing to do
    assert lib.dg_moe_combine(None, 64, 0, 64, _layout(tokens=0), None, None, 64, 0, None) == 0
    assert lib.dg_moe_dispatch(None, 64, 64, _layout(rows=0), None, 64, None, 0, 0, None, 0, 1, 0, None) == 0


def test_mx_refusals(lib):
    def run(fn='dg_mx_quantize', **kw):
        a = _lib.MxArgs(0, 0, 1, 4, 64, 4096, 64, 0, 4096, 32, 0, 4096, 4, 0, 0)
        for name, v in kw.items():
            setattr(a, name, v)
        return getattr(lib, fn)(a, None)
    for fn in ('dg_mx_quantize', 'dg_mx_dequantize'):
        _refused(lib, run(fn, format=2), 'unknown format')
        _refused(lib, run(fn, x_dtype=2), 'bf16 or fp32')
        _refused(lib, run(fn, k=48), 'block of 32')
        _refused(lib, run(fn, rows=-1), 'negative size')
        _refused(lib, run(fn, x=None), 'null tensor')
        _refused(lib, run(fn, x_ld=63), 'leading dimension')
        _refused(lib, run(fn, format=1), 'leading dimension')
        _refused(lib, run(fn, sf_ld=5), 'even')
        _refused(lib, run(fn, codes_ld=36), '8-byte aligned')
        assert run(fn, rows=0) == 0 and run(fn, k=0) == 0
    assert lib.dg_mx_quantize(None, None) == -1


def test_mx_gemm_refusals(lib):
    def run(m=4, n=64, k=64, x=4096, xt=0, xld=64, w=4096, wld=32, sf=4096, sfld=64, d=4096, dt=0, ldd=64):
        return lib.dg_mx_gemm(x, xt, xld, w, wld, sf, sfld, d, dt, ldd, m, n, k, 0, 0, None)
    _refused(lib, run(k=-1), 'negative size')
    _refused(lib, run(xt=2), 'x is bf16')
    _refused(lib, run(dt=2), 'D is bf16')
    assert run(m=17) == _lib.DG_ENOKERNEL and b'16 rows' in lib.dg_last_error()
    assert run(m=16, k=2080, xld=2080, wld=1040) == _lib.DG_ENOKERNEL and b'32768' in lib.dg_last_error()
    _refused(lib, run(k=48), 'block of 32')
    _refused(lib, run(k=0), 'block of 32')
    _refused(lib, run(w=None), 'null tensor')
    _refused(lib, run(wld=16), 'leading dimension')
    _refused(lib, run(xld=63), 'leading dimension')
    _refused(lib, run(ldd=32), 'leading dimension')
    _refused(lib, run(xld=65), '4-byte aligned')
    _refused(lib, run(sfld=65), 'even')
    _refused(lib, run(wld=1 << 28), 'stride too large')
    assert run(m=0) == 0 and run(n=0) == 0


def test_few_rows_to_an_expert_plan(lib):
    """M-grouped psum layouts of e2m1 rows, 64 or fewer to a group on average, take their own kernel; others do not."""
    info = _lib.LaunchInfo()
    def plan(m, kind=_lib.DG_KIND_FP4_FP4, gemm_type=_lib.DG_GEMM_MGROUPED_PSUM):
        a = _lib.GemmArgs()
        a.kind, a.gemm_type, a.m, a.n, a.k, a.num_groups, a.alignment, a.alpha = kind, gemm_type, m, 2048, 4096, 32, 32, 1.0
        a.lda = a.ldb = 2048 if kind == _lib.DG_KIND_FP4_FP4 else 4096
        a.ldd, a.batch_stride_b, a.sfa_ld, a.sfb_ld, a.num_cus = 2048, 2048 * a.ldb, m, 2048, 256
        assert lib.dg_launch_plan(ctypes.byref(a), ctypes.byref(info)) == 0, lib.dg_last_error()
        return info.skinny
    assert plan(1248) == 4 and plan(2048) == 4
    assert plan(2080) != 4 and plan(1248, _lib.DG_KIND_FP8_FP8) != 4 and plan(1248, gemm_type=_lib.DG_GEMM_MGROUPED_IDX) != 4


def _experts_args(m=1248, alignment=32):
    """A grouped e2m1 x e2m1 call over 32 experts, N = 2048, K = 4096, in a psum layout of m rows."""
    a = _lib.GemmArgs()
    a.kind, a.gemm_type, a.m, a.n, a.k, a.num_groups, a.alignment, a.alpha = \
        _lib.DG_KIND_FP4_FP4, _lib.DG_GEMM_MGROUPED_PSUM, m, 2048, 4096, 32, alignment, 1.0
    a.lda = a.ldb = a.ldd = 2048
    a.batch_stride_b, a.sfa_ld, a.sfb_ld, a.num_cus = 2048 * 2048, m, 2048, 256
    return a


@pytest.mark.parametrize('m', [1248, 4096])
def test_few_rows_to_an_expert_refuse_a_negative_split(lib, m):
    info, a = _lib.LaunchInfo(), _experts_args(m)
    assert lib.dg_launch_plan(ctypes.byref(a), ctypes.byref(info)) == 0
    a.split_k = -1
    _refused(lib, lib.dg_launch_plan(ctypes.byref(a), ctypes.byref(info)), 'split_k')


@pytest.mark.parametrize('m,alignment,cus', [(1248, 32, 256), (1248, 32, 200), (2048, 64, 256), (2240, 64, 256), (4224, 128, 256)])
def test_select_config_names_the_tile_that_runs(lib, m, alignment, cus):
    """Also where the kernel of few rows to an expert runs."""
    info, a = _lib.LaunchInfo(), _experts_args(m, alignment)
    a.num_cus = cus
    block_m, block_n = ctypes.c_int32(), ctypes.c_int32()
    assert lib.dg_launch_plan(ctypes.byref(a), ctypes.byref(info)) == 0
    assert lib.dg_select_config(ctypes.byref(a), ctypes.byref(block_m), ctypes.byref(block_n)) == 0
    assert (block_m.value, block_n.value) == (info.block_m, info.block_n)


@pytest.mark.parametrize('cus,own', [(256, True), (200, False), (64, False)])
def test_few_rows_to_an_expert_under_a_cap_take_tiles(lib, cus, own):
    """Workgroups of a wave or a few are no use of a capped number of them."""
    info, a = _lib.LaunchInfo(), _experts_args()
    a.num_cus = cus
    assert lib.dg_launch_plan(ctypes.byref(a), ctypes.byref(info)) == 0
    assert (info.skinny == 4) == own and info.grid <= (1 << 31 if own else cus)


@pytest.mark.parametrize('alignment,cus,tile', [(64, 200, (64, 128)), (128, 256, (128, 128)), (128, 200, (384, 128)), (128, 64, (384, 128))])
def test_fp4_psum_layouts_under_a_cap(lib, alignment, cus, tile):
    """128x128 tiles, which several CUs share a group's weights by, gain nothing where few CUs may run."""
    a = _experts_args(4224 if alignment == 128 else 2240, alignment)
    a.num_cus = cus
    block_m, block_n = ctypes.c_int32(), ctypes.c_int32()
    assert lib.dg_select_config(ctypes.byref(a), ctypes.byref(block_m), ctypes.byref(block_n)) == 0
    assert (block_m.value, block_n.value) == tile


@pytest.mark.parametrize('groups,n,k', [(32, 4096, 7168), (64, 2048, 2048)])
def test_fp4_masked_groups_of_fewer_rows_than_a_tile(lib, groups, n, k):
    """128 rows a group: a half-filled large tile loads half the rows, and reads the weights once."""
    a = _lib.GemmArgs()
    a.kind, a.gemm_type, a.m, a.n, a.k, a.num_groups, a.alignment, a.num_cus = \
        _lib.DG_KIND_FP4_FP4, _lib.DG_GEMM_MASKED, 128, n, k, groups, 256, 256
    block_m, block_n = ctypes.c_int32(), ctypes.c_int32()
    assert lib.dg_select_config(ctypes.byref(a), ctypes.byref(block_m), ctypes.byref(block_n)) == 0
    assert (block_m.value, block_n.value) == (256, 256)


@pytest.mark.parametrize('gemm_type,groups,m,n,k,cus', [(_lib.DG_GEMM_NORMAL, 1, 2048, 7168, 2048, 64), (_lib.DG_GEMM_NORMAL, 1, 3000, 3000, 512, 64),
                                                        (_lib.DG_GEMM_BATCHED, 16, 1024, 1024, 1024, 200)])
def test_fp4_products_under_a_cap_take_tiles_that_walk(lib, gemm_type, groups, m, n, k, cus):
    """One launch of a persistent kernel in place of launch after launch of a tile per allowed CU."""
    a = _lib.GemmArgs()
    a.kind, a.gemm_type, a.m, a.n, a.k, a.num_groups, a.alignment, a.num_cus = _lib.DG_KIND_FP4_FP4, gemm_type, m, n, k, groups, 256, cus
    block_m, block_n = ctypes.c_int32(), ctypes.c_int32()
    assert lib.dg_select_config(ctypes.byref(a), ctypes.byref(block_m), ctypes.byref(block_n)) == 0
    assert (block_m.value, block_n.value) == (256, 224)


def test_linear_xent_refusals(lib):
    def run(fn='dg_linear_xent_forward', **kw):
        a = _lib.LinearXentArgs(4, 64, 100, 4096, 4096, 64, 64, 4096, 8, -100, 4096, 4096, 4096, 4096, 4096, 64, 64, 4096, 1 << 40, 0)
        for name, v in kw.items():
            setattr(a, name, v)
        return getattr(lib, fn)(a, None)
    for fn in ('dg_linear_xent_forward', 'dg_linear_xent_backward'):
        _refused(lib, run(fn, tokens=-1), 'invalid size')
        _refused(lib, run(fn, vocab=0), 'invalid size')
        _refused(lib, run(fn, tokens=(1 << 20) + 1), '2^20 tokens')
        _refused(lib, run(fn, width=60), 'multiple of 8')
        _refused(lib, run(fn, target_bytes=2), 'int32 or int64')
        _refused(lib, run(fn, x_ld=32), '16-byte aligned')
        _refused(lib, run(fn, w=4100), '16-byte aligned')
        _refused(lib, run(fn, w_ld=1 << 22), 'stride too large')
        _refused(lib, run(fn, x=None), 'null tensor')
        _refused(lib, run(fn, lse=None), 'null tensor')
        _refused(lib, run(fn, workspace=None), 'workspace')
        _refused(lib, run(fn, workspace_bytes=16), 'workspace')
    _refused(lib, run('dg_linear_xent_backward', d_w_ld=32), 'gradients')
    _refused(lib, run('dg_linear_xent_backward', d_loss=None), 'null tensor')
    _refused(lib, run('dg_linear_xent_backward', tokens=0), 'no tokens')
    assert run(tokens=0) == 0
    need = ctypes.c_int64()
    a = _lib.LinearXentArgs(8192, 4096, 131072, 4096, 4096, 4096, 4096, 4096, 8)
    assert lib.dg_linear_xent_workspace_size(a, 1, ctypes.byref(need)) == 0
    assert 0 < need.value < 8192 * 131072 * 2          # (a piece of the vocabulary, not all of it)
    assert lib.dg_linear_xent_workspace_size(a, 0, ctypes.byref(need)) == 0 and need.value < 8192 * 131072 // 8


@pytest.mark.parametrize('tokens,x_ld,pieces', [(262143, 4096, False), (262144, 4096, True), (1023, 1 << 20, False), (1100, 1 << 20, True)])
def test_linear_xent_sums_pieces_of_tokens_past_2_gib(lib, tokens, x_ld, pieces):
    """Where the rows of x span 2 GiB, the gradient's workspace holds fp32 sums of d_w besides d and d_x."""
    need, small = ctypes.c_int64(), 64 * 1024
    a = _lib.LinearXentArgs(tokens, 256, 512, 4096, 4096, x_ld, 256, 4096, 8)
    a.num_cus = 8   # (no ranges of K)
    assert lib.dg_linear_xent_workspace_size(a, 1, ctypes.byref(need)) == 0
    rest = need.value - (tokens + 8) * 512 * 2 - tokens * 256 * 4 - tokens * 4
    assert (rest > 512 * 256 * 4 - small) == pieces and rest < 512 * 256 * 4 + small


@pytest.mark.parametrize('tokens', [1, 9, 1001])
def test_linear_xent_holds_no_rows_past_the_tokens(lib, tokens):
    """The gradient's workspace: d over the tokens, d_x's fp32 sums, the tokens' rests, and little else."""
    need = ctypes.c_int64()
    a = _lib.LinearXentArgs(tokens, 64, 1 << 17, 4096, 4096, 64, 64, 4096, 8)
    a.num_cus = 1   # (no ranges of K)
    assert lib.dg_linear_xent_workspace_size(a, 1, ctypes.byref(need)) == 0
    least = tokens * (1 << 17) * 2 + tokens * 64 * 4 + tokens * 4
    assert least <= need.value < least + 5 * 256


def test_python_refusals():
    with pytest.raises(RuntimeError, match='int32 or int64'):
        deep_gemm.moe_sort(torch.zeros(2, 2), 4)
    with pytest.raises(RuntimeError, match='device tensor'):
        deep_gemm.moe_sort(torch.zeros(2, 2, dtype=torch.int32), 4)
    with pytest.raises(RuntimeError, match='device tensor'):
        deep_gemm.mx_quantize(torch.zeros(2, 64))
    with pytest.raises(RuntimeError, match='unknown format'):
        deep_gemm.mx_quantize(torch.zeros(2, 64), 'e5m2')
    with pytest.raises(RuntimeError, match='e2m1 weights'):
        deep_gemm.mx_gemm_nt(torch.zeros(2, 64), (torch.zeros(4, 64, dtype=torch.float8_e4m3fn), None), torch.zeros(2, 4))
    x, w, t = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(9, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match='device tensors'):
        deep_gemm.linear_cross_entropy(x, w, t)
    layout = deep_gemm.MoELayout(*(torch.zeros(s, dtype=torch.int32) for s in ((2, 2), (64,), (4,), (64,))))
    with pytest.raises(RuntimeError, match='device tensor'):
        deep_gemm.moe_dispatch(torch.zeros(2, 64), layout)
    with pytest.raises(RuntimeError, match='device tensor'):
        deep_gemm.moe_combine(torch.zeros(64, 64), layout)
    with pytest.raises(RuntimeError, match='contiguous int32'):
        deep_gemm.moe_combine(torch.zeros(64, 64), layout._replace(source=torch.zeros(64)))


def test_num_rows_bounds_every_routing():
    g = torch.Generator().manual_seed(0)
    for pairs, groups, alignment in ((0, 4, 32), (1, 4, 32), (5, 9, 64), (100, 7, 32), (1000, 300, 128)):
        deep_gemm.set_mk_alignment_for_contiguous_layout(alignment)
        try:
            m = deep_gemm.moe_num_rows(pairs, groups)
        finally:
            deep_gemm.set_mk_alignment_for_contiguous_layout(256)
        assert m % alignment == 0
        for kind in range(3):
            ids = torch.randint(0, groups, (pairs, 1), generator=g) if kind == 0 else torch.arange(pairs).view(-1, 1) % groups if kind == 1 \
                else (torch.arange(pairs).view(-1, 1) % groups).clamp(max=min(groups, pairs) - 1)
            counts = torch.bincount(ids.reshape(-1), minlength=groups)
            assert int(((counts + alignment - 1) // alignment * alignment).sum()) <= m
            assert (om.sort(ids, groups, alignment, m)[0] >= 0).all()


def test_oracle_quantisation_is_nearest():
    """No value of the format lies nearer than the one the oracle takes, and its codes decode to multiples of the step."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 64, generator=g) * torch.exp(2 * torch.randn(6, 1, generator=g))
    for fmt, table in (('e2m1', ox.E2M1), ('e4m3', ox.E4M3)):
        codes, scales = ox.quantize(x, fmt)
        got = ox.values(codes, scales, fmt)
        s = torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)
        near = (x.double().abs().unsqueeze(-1) - s.unsqueeze(-1) * torch.tensor(table, dtype=torch.float64)).abs().amin(-1)
        assert torch.equal((x.double() - got).abs(), near)
        top = 6.0 if fmt == 'e2m1' else 448.0
        amax = x.double().abs().view(6, 2, 32).amax(-1)
        blocks = torch.exp2(scales.double() - 127)
        assert (amax <= top * blocks).all() and (amax > top * blocks / 2).all()


@pytest.mark.parametrize('m,n,k,bm', [(200, 4096, 4096, 128), (512, 2112, 7168, 128), (4096, 7168, 2048, 256)])
def test_fp4_products_of_few_rows_take_small_tiles(lib, m, n, k, bm):
    """A large tile would leave most CUs idle at a few hundred rows."""
    args = _lib.GemmArgs()
    args.kind, args.m, args.n, args.k, args.num_groups, args.num_cus = 2, m, n, k, 1, 256
    block_m, block_n = ctypes.c_int32(), ctypes.c_int32()
    assert lib.dg_select_config(ctypes.byref(args), ctypes.byref(block_m), ctypes.byref(block_n)) == 0
    assert block_m.value <= bm if bm < 256 else block_m.value == bm


@pytest.mark.parametrize('m,alignment,tile', [(2240, 64, (64, 128)), (4224, 128, (128, 128)), (8192, 128, (384, 128)), (4096, 96, (384, 128))])
def test_fp4_psum_layouts_of_little_more_than_a_tile_a_group(lib, m, alignment, tile):
    args = _lib.GemmArgs()
    args.kind, args.gemm_type, args.m, args.n, args.k, args.num_groups = 2, 2, m, 2048, 4096, 32
    args.alignment, args.num_cus = alignment, 256
    block_m, block_n = ctypes.c_int32(), ctypes.c_int32()
    assert lib.dg_select_config(ctypes.byref(args), ctypes.byref(block_m), ctypes.byref(block_n)) == 0
    assert (block_m.value, block_n.value) == tile


def test_extents_past_2_to_the_30(lib):
    """Indices of tiles that end past an extent are 32-bit: larger extents are refused before anything is launched."""
    big = (1 << 30) + 32
    layout = _layout(tokens=big, topk=1)
    _refused(lib, lib.dg_moe_sort(4096, 4, layout, None, 0, 0, None), 'invalid size')
    _refused(lib, lib.dg_moe_combine(4096, 64, 0, 64, _layout(rows=big), None, 4096, 64, 0, None), 'invalid size')
    _refused(lib, lib.dg_moe_dispatch(4096, 64, 64, layout, 4096, 64, None, 0, 0, None, 0, 1, 0, None), 'invalid size')
    for kw in (dict(rows=big, sf_ld=big), dict(k=big, x_ld=big, codes_ld=big)):
        a = _lib.MxArgs(0, 0, 1, 4, 64, 4096, 64, 0, 4096, 32, 0, 4096, 4, 0, 0)
        for name, v in kw.items():
            setattr(a, name, v)
        _refused(lib, lib.dg_mx_quantize(a, None), '2^30')
        _refused(lib, lib.dg_mx_dequantize(a, None), '2^30')
    _refused(lib, lib.dg_mx_gemm(4096, 0, 64, 4096, 32, 4096, big, 4096, 0, big, 1, big, 64, 0, 0, None), '2^30')
    a = _lib.LinearXentArgs(4, 64, 100, 4096, 4096, 64, 64, 4096, 8, -100, 4096, 4096, 4096, 4096, 4096, 64, 64, 4096, 1 << 60, 0)
    a.vocab = (1 << 30) + 1
    _refused(lib, lib.dg_linear_xent_forward(a, None), '2^30')
    _refused(lib, lib.dg_linear_xent_backward(a, None), '2^30')
