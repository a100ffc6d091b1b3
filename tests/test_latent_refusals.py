"""Calls of latent attention that are refused before any launch, without a GPU."""
import pytest
import torch

from stepquant_amd import _native as N
from stepquant_amd.kernels.latent_cache import _output, _scale
from tests.test_latent_surface import _cache, _schedule

ABSORBED = dict(q=16, q_rope=16, out=16, workspace=16, table=16, requests=2, tokens=16, q_stride=4096, q_head_stride=512,
                rope_stride=512, rope_head_stride=64, width=4, scale=1.)
EXPANDED = dict(q=16, k=16, v=16, rope=16, out=16, workspace=16, cu=16, starts=16, tokens=16, rows=16, q_stride=1536,
                q_head_stride=192, k_stride=1024, k_head_stride=128, v_stride=1024, v_head_stride=128, rope_stride=64, batch=2,
                dim=128, dtype=N.F16, scale=1.)


@pytest.mark.parametrize("scale", [2.4e38, -2.9e38])
def test_scales_that_pass_32_bits_times_log2_e_are_refused(scale):
    """Scores are powers of two: scale * log2(e) would be infinite, and no number where a score is 0."""
    a = N.LatentAttend(**{**ABSORBED, "scale": scale}, schedule=_schedule())
    assert N.lib().sq_latent_attend(_cache(), a, None) == -22 and b"scale" in N.lib().sq_last_error()
    a = N.ExpandedAttend(**{**EXPANDED, "scale": scale}, schedule=_schedule(kv_heads=8, rows=256))
    assert N.lib().sq_expanded_attend(a, None) == -22 and b"scale" in N.lib().sq_last_error()
    with pytest.raises(ValueError, match="scale"):
        _scale(scale)
    assert _scale(1.9e38) == 1.9e38


def test_appends_of_no_tokens_check_the_rows_that_they_turn():
    """Rows may be turned beside an empty append, as beside the 8-bit cache's."""
    L = N.lib()
    rotary = lambda **kw: N.Rotary(**{**dict(turns=16, dim=64, magnitude=1.), **kw})
    rows = lambda **kw: N.RotaryRows(**{**dict(x=16, out=16, positions=16, tokens=4, x_stride=512, x_head_stride=64,
                                               out_stride=512, out_head_stride=64, heads=8, head_dim=64, dtype=N.BF16,
                                               positions_dtype=N.I32), **kw})
    call = lambda r, q: L.sq_latent_append(_cache(), N.LatentAppend(tokens=0), r, q, None)
    assert call(None, rows()) == -22 and call(rotary(turns=None), rows()) == -22 and call(rotary(dim=80), rows(head_dim=80)) == -23
    assert call(rotary(), rows(dtype=N.F16)) == -22 and call(rotary(), rows(x=None)) == -22 and call(rotary(), rows(tokens=-1)) == -22
    assert call(rotary(), rows(tokens=0)) == 0 and call(rotary(), None) == 0 and call(None, None) == 0


def test_sets_of_128_rows_have_two_workgroups_to_count():
    """A launch has fewer than 2^32 threads: 512 a workgroup, two workgroups a worker."""
    fits = dict(rows=128, slots=128, max_workers=1 << 22, max_units=600, max_merges=256, max_partials=512, merge_rows=128)
    a = N.LatentAttend(**ABSORBED, schedule=_schedule(**fits))
    assert N.lib().sq_latent_attend(_cache(), a, None) == -22 and b"workers" in N.lib().sq_last_error()


def test_outputs_that_lie_over_operands_are_refused():
    """Workgroups still read the operands while others write; only absorbed queries, a row of
    which no other row's workgroups read, may be where their outputs go."""
    x = torch.zeros(6, 4, 192, dtype=torch.bfloat16)
    out = x.view(-1)[:6 * 4 * 128].view(6, 4, 128)
    other = torch.zeros(6, 4, 128, dtype=torch.bfloat16)
    assert _output(other, (6, 4, 128), x, x, out) is other
    for y in (x, x[..., 64:], x[3:], out, x[2:3, :, :8]):
        with pytest.raises(ValueError, match="overlap"):
            _output(out, (6, 4, 128), x, other, y)
    assert _output(out, (6, 4, 128), x, x[:0], x[1:1]) is out and _output(out, (6, 4, 128), x, x.view(-1)[6 * 4 * 128:]) is out
    assert _output(out, (6, 4, 128), x, in_place=out) is out
    for y in (x.view(-1)[8:8 + 6 * 4 * 128].view(6, 4, 128), x[..., :128]):
        with pytest.raises(ValueError, match="overlap"):
            _output(out, (6, 4, 128), x, in_place=y)
