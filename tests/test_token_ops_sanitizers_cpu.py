"""The operators of a token step, recorded, lowered, stored and loaded with damaged records, under AddressSanitizer and
UndefinedBehaviorSanitizer."""
import test_host_sanitizers_cpu as host


def test_token_operators_are_clean_under_asan_and_ubsan(monkeypatch):
    monkeypatch.setattr(host, "CASES", ["tests/test_token_ops_cpu.py"])
    host.test_cpu_suites_are_clean_under_asan_and_ubsan()
