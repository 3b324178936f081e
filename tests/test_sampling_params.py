"""The filters of a request's sampling parameters: what they accept, and when they count."""
import pytest

from swifttransformer_amd.sampling import SamplingParams


def test_defaults_filter_nothing():
    assert not SamplingParams().filtered and not SamplingParams(temperature=1.0).filtered
    assert not SamplingParams(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0).filtered
    # greedy requests are greedy with them too
    assert not SamplingParams(top_k=5, top_p=0.5, min_p=0.5).filtered


@pytest.mark.parametrize("kw", [dict(top_k=1), dict(top_p=0.99), dict(min_p=0.01)])
def test_each_filters(kw):
    assert SamplingParams(temperature=0.5, **kw).filtered


@pytest.mark.parametrize("kw", [dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.1)])
def test_refused(kw):
    with pytest.raises(ValueError):
        SamplingParams(temperature=1.0, **kw)


def test_command_line_takes_them():
    from swifttransformer_amd.cli.run_opt import build_parser
    args = build_parser().parse_args(["m", "auto", "bf16", "p", "--top-k", "7", "--top-p", "0.9", "--min-p", "0.1"])
    assert (args.top_k, args.top_p, args.min_p) == (7, 0.9, 0.1)
