"""The benchmark's time of a token, from generations whose times have outliers."""
import pytest

from hyperattention_b200.llm_bench import token_ms


@pytest.mark.parametrize('late', [(), (0,), (1, 3), (0, 1, 2, 4), (7, 8, 10)])
def test_token_ms_without_the_outliers(late):
    runs = []

    def measure(n):
        runs.append(n)
        return 600 + 5 * n + (700 if len(runs) - 1 in late else 0)

    assert token_ms(measure, 64) == 5
    assert sorted(set(runs)) == [4, 68]
