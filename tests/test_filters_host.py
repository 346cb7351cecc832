"""The filters of sampled tokens as a request gives them: what is refused, without a GPU."""
import pytest


def test_filters_of_requests_are_checked():
    from imparo_b200.engine.engine import checked_filters
    assert checked_filters(2, [0, 0], [1.0, 1], [0.0, 0]) == ()
    assert checked_filters(2, [0, 5], [1.0, 0.5], [0.0, 0.1]) == ([0, 5], [1.0, 0.5], [0.0, 0.1])
    for bad in (([0], [1.0, 1.0], [0, 0]), ([0, -1], [1.0, 1.0], [0, 0]), ([0, 0.5], [1.0, 1.0], [0, 0]), ([0, 0], [0.0, 1.0], [0, 0]),
                ([0, 0], [1.0, 1.5], [0, 0]), ([0, 0], [float("nan"), 1.0], [0, 0]), ([0, 0], [1.0, 1.0], [-0.1, 0]), ([0, 0], [1.0, 1.0], [0, 1.1])):
        with pytest.raises(ValueError):
            checked_filters(2, *bad)


def test_command_line_takes_the_filters():
    from imparo_b200.cli import build_parser
    args = build_parser().parse_args(["-m", "x", "--top-k", "5", "--top-p", "0.5", "--min-p", "0.1", "1"])
    assert (args.top_k, args.top_p, args.min_p) == (5, 0.5, 0.1)
    args = build_parser().parse_args(["-m", "x", "1"])
    assert (args.top_k, args.top_p, args.min_p) == (0, 1.0, 0.0)


def test_a_top_k_that_is_no_whole_number_is_refused_by_name():
    from imparo_b200.engine.engine import checked_filters
    for k in (float("inf"), float("-inf"), float("nan"), 2.5):
        with pytest.raises(ValueError, match="top_k must be a whole number"):
            checked_filters(1, [k], [1.0], [0.0])
    assert checked_filters(1, [7.0], [1.0], [0.0]) == ([7.0], [1.0], [0.0])
