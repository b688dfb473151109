"""The tests that conftest.py skips where the reference-built programs are
missing, and only there."""
import ast
import os

import conftest


def test_named_tests_exist_and_run_the_named_programs():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "test_gpu_llama2.py")
    text = open(path).read()
    tests = {f.name: ast.get_source_segment(text, f) for f in ast.parse(text).body if isinstance(f, ast.FunctionDef)}
    for name, programs in conftest.REFERENCE_PROGRAMS.items():
        for p in programs:
            place, program = p.split("/")
            assert f'"{place}"' in tests[name] and f'"{program}"' in text
    # no other test of that file runs a reference-built program
    assert {n for n, source in tests.items() if n.startswith("test_") and "REF" in source} == set(conftest.REFERENCE_PROGRAMS)


def test_tests_are_skipped_only_without_their_programs(tmp_path):
    for name, programs in conftest.REFERENCE_PROGRAMS.items():
        built = tmp_path / name
        assert conftest.missing_reference_programs(name, str(built)) == list(programs)
        for p in programs:
            (built / p).parent.mkdir(parents=True, exist_ok=True)
            (built / p).touch()
        assert conftest.missing_reference_programs(name, str(built)) == []
        os.remove(built / programs[0])
        assert conftest.missing_reference_programs(name, str(built)) == [programs[0]]
    assert conftest.missing_reference_programs("test_llama2_matmul_matches_oracle", str(tmp_path)) == []
