# one-off GPU batch: the new staging / path tests
mkdir -p gpurun_out/r6b gpurun_out/race
timeout -k 10 700 python -u -m pytest tests/test_gpu_allreduce.py -m gpu -x -v -s --timeout 300 --timeout-method thread \
  -k "reference_framing_staging or above_arena or staging_bounded_by_segment" > gpurun_out/r6b/staging.log 2>&1
rc=$?; echo "staging rc=$rc" > gpurun_out/r6b/rcs.txt
[ $rc -eq 0 ] || exit $rc
