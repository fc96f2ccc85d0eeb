"""The hooks of conftest.py, in a test run of their own."""
import os
import subprocess
import sys
import textwrap


def test_a_modules_fixtures_are_collected_before_the_next_module(tmp_path):
    """A dead cycle that a module's fixture held is gone when the next module's first test runs, without a collection of its own."""
    hooks = os.path.join(os.path.dirname(os.path.abspath(__file__)), "conftest.py")
    (tmp_path / "conftest.py").write_text(textwrap.dedent(f"""
        import gc
        import importlib.util
        spec = importlib.util.spec_from_file_location("hooks", {hooks!r})
        hooks = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(hooks)
        globals().update({{n: f for n, f in vars(hooks).items() if n.startswith("pytest_runtest")}})
        gc.disable()
        refs = []
        """))
    (tmp_path / "test_a.py").write_text(textwrap.dedent("""
        import weakref
        import pytest
        from conftest import refs

        class Cycle:
            pass

        @pytest.fixture(scope="module")
        def cycle():
            c = Cycle()
            c.me = c
            refs.append(weakref.ref(c))
            return c

        def test_one(cycle):
            assert refs[0]() is cycle

        def test_two(cycle):
            assert refs[0]() is cycle
        """))
    (tmp_path / "test_b.py").write_text(textwrap.dedent("""
        from conftest import refs

        def test_three():
            assert len(refs) == 1 and refs[0]() is None
        """))
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", str(tmp_path)], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "3 passed" in r.stdout
