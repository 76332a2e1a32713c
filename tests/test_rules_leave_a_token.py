"""Rules that leave no token are refused, whichever of them it is that leaves none."""
import math

import pytest

import wick_b200 as wick

OUT = -math.inf


@pytest.mark.parametrize("rules", [wick.LogitRules(allowed=[]), wick.LogitRules(allowed=[3], bias={3: OUT}),
                                   wick.LogitRules(allowed=[3, 5, 3], bias={3: OUT, 5: OUT, 6: 1.0}), wick.LogitRules(bias={t: OUT for t in range(8)})])
def test_no_token_left(rules):
    with pytest.raises(ValueError, match="no token is allowed"):
        rules.check(8)


def test_one_token_left():
    wick.LogitRules(allowed=[3, 5], bias={3: OUT, 6: OUT}).check(8)
    wick.LogitRules(bias={t: OUT for t in range(7)}).check(8)
    wick.LogitRules(allowed=[3], bias={3: math.inf}).check(8)
