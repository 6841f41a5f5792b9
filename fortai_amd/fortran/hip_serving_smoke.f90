! hip_serving_smoke.f90 -- a Fortran caller of the serving operators through
! fortai_hip_serving.
!
! Without an argument: page bookkeeping and refused calls, which need no GPU.
! With the argument "gpu" also one step on device 0 with known answers: a vector
! at position 0 is not rotated, a query that sees a single token gets that
! token's value, greedy verification keeps a draft that is the largest logit,
! and a token that the text has loses what the rules say.
! Exit status 0 and "fortran serving smoke ok" on success.
program hip_serving_smoke
    use, intrinsic :: iso_c_binding, only: c_double, c_float, c_int, c_int8_t, c_int32_t, c_int64_t, c_null_ptr, c_ptr, &
        c_size_t
    use fortai_status, only: FORTAI_INVALID, status_t
    use fortai_backend_hip, only: hip_q8_context_t
    use fortai_hip_serving
    implicit none

    type(status_t) :: stat
    integer :: failures
    character(len=8) :: mode

    failures = 0
    call pages_part()
    mode = ''
    if (command_argument_count() > 0) call get_command_argument(1, mode)
    if (mode == 'gpu') call gpu_part()
    if (failures /= 0) error stop 1
    print '(a)', 'fortran serving smoke ok'

contains

    subroutine pages_part()
        type(hip_kv8_pages_t) :: pool
        type(hip_kv8_cache_t) :: cache
        type(hip_kv8_batch_t) :: batch
        type(hip_gdn_cache_t) :: states
        type(hip_gdn_batch_t) :: rows
        integer(c_int32_t) :: from, to, table(4, 2), moved_from(8), moved_to(8), starts(3), shared(2), group_of(2)
        integer :: copies, groups

        call need(hip_kv8_bytes(3, 5, 16, 2, 64) == int(3 * 5 * 2 * (2 * 16 * 64 + 8), c_size_t), 'bytes')
        call need(hip_kv8_bytes(3, 5, 24, 2, 64) == 0_c_size_t, 'bytes of no such cache')
        call pool%extend(0, 1, from, to, copies, stat)
        call need(stat%code == FORTAI_INVALID, 'extend before create')
        call cache%append(0, batch, HIP_DTYPE_F32, c_null_ptr, 0_c_int64_t, c_null_ptr, 0_c_int64_t, stat)
        call need(stat%code == FORTAI_INVALID, 'append before create')
        call pool%create(8, 16, 2, 4, stat)
        call need(stat%is_ok() .and. pool%free_count() == 8, 'pool create')
        call pool%extend(0, 20, from, to, copies, stat)
        call need(stat%is_ok() .and. copies == 0 .and. pool%length(0) == 20, 'extend')
        call pool%fork(0, 1, 18_c_int64_t, stat)
        call need(stat%is_ok() .and. pool%free_count() == 6, 'fork')
        call pool%extend(1, 1, from, to, copies, stat)
        call need(stat%is_ok() .and. copies == 1 .and. pool%free_count() == 5, 'a shared page is replaced')
        call pool%tables([0_c_int, 1_c_int], table, stat)
        call need(stat%is_ok() .and. table(1, 1) == table(1, 2), 'the full page stays shared')
        call need(table(2, 1) == from .and. table(2, 2) == to .and. all(table(3:, :) == -1), 'tables')
        call pool%groups([0_c_int, 1_c_int], starts, shared, group_of, groups, stat)
        call need(stat%is_ok() .and. groups == 1 .and. shared(1) == 0 .and. all(starts(:2) == [0, 2]), 'groups')
        call need(all(group_of == 0), 'sequences that share less than a tile lie together')
        call pool%groups([0_c_int, 1_c_int], starts(:2), shared, group_of, groups, stat)
        call need(stat%code == FORTAI_INVALID, 'groups without room for the last start')
        call need(hip_gdn_bytes(1, 2, 1, 2, 64, 4, 3) == int(4 * (2 * 2 * 64 * 64 + 2 * 6 * 256 + 2 * 3 * (64 + 128 + 2) + 2), &
            c_size_t), 'bytes of states')
        call need(hip_gdn_bytes(1, 2, 2, 3, 64, 4, 3) == 0_c_size_t, 'bytes of no such states')
        call states%run(0, rows, HIP_DTYPE_F32, c_null_ptr, 0_c_int64_t, c_null_ptr, 0_c_int64_t, c_null_ptr, 0_c_int64_t, &
            c_null_ptr, c_null_ptr, c_null_ptr, 0.0_c_float, c_null_ptr, 0_c_int64_t, stat)
        call need(stat%code == FORTAI_INVALID, 'rows before create')
        call states%copy_slots([0_c_int32_t], [1_c_int32_t], stat)
        call need(stat%code == FORTAI_INVALID, 'slots before create')
        call pool%extend(0, 1000, from, to, copies, stat)
        call need(stat%code == FORTAI_INVALID .and. pool%length(0) == 20, 'refused without a change')
        call pool%truncate(0, 0_c_int64_t, stat)
        call need(stat%is_ok() .and. pool%length(0) == 0 .and. pool%length(7) == -1, 'truncate')
        call pool%compact(moved_from, moved_to, copies, stat)
        call need(stat%is_ok() .and. copies == 1 .and. moved_from(1) > moved_to(1), 'compact')
        call pool%destroy(stat)
        call pool%destroy(stat)
        call need(stat%is_ok(), 'destroy, twice')
    end subroutine pages_part

    subroutine gpu_part()
        type(hip_q8_context_t) :: ctx
        type(hip_rope_t) :: rope
        type(hip_kv8_cache_t) :: cache
        type(hip_verifier_t) :: verifier
        type(hip_kv8_batch_t) :: batch
        type(hip_gdn_cache_t) :: states
        type(hip_gdn_batch_t) :: state_rows
        type(hip_logit_rules_t) :: rules
        type(c_ptr) :: quants, qkv
        type(c_ptr) :: x, y, positions, starts, lengths, tables, logits, tokens, uniforms, temperatures, emitted, accepted
        real(c_float) :: keys(64), values(64), got(64), rows(8)
        integer(c_int8_t) :: bytes(16)
        integer :: i

        keys = [(real(i, c_float) / 64.0_c_float, i = 1, 64)]
        values = [(real(2 * i - 65, c_float) * 127.0_c_float / 63.0_c_float, i = 1, 64)]
        values = anint(values)
        call ctx%create(0, stat)
        call need(stat%is_ok(), 'context create')
        x = room(ctx, 256)
        y = room(ctx, 256)
        positions = room(ctx, 4)
        starts = room(ctx, 8)
        lengths = room(ctx, 4)
        tables = room(ctx, 4)
        call ctx%upload_real(x, keys, stat)
        call put(ctx, positions, [0_c_int32_t])
        call put(ctx, starts, [0_c_int32_t, 1_c_int32_t])
        call put(ctx, lengths, [0_c_int32_t])
        call put(ctx, tables, [2_c_int32_t])

        call rope%create(ctx, 63, 10000.0_c_double, stat)
        call need(stat%code == FORTAI_INVALID .and. allocated(stat%message), 'an odd rope dimension is refused')
        call rope%create(ctx, 64, 10000.0_c_double, stat)
        call need(stat%is_ok(), 'rope create')
        call rope%apply(HIP_DTYPE_F32, x, 64_c_int64_t, 64_c_int64_t, 1, 1, 64, positions, c_null_ptr, 0.0_c_float, x, &
            64_c_int64_t, 64_c_int64_t, stat)
        call need(stat%is_ok(), 'rope')
        call ctx%download_real(x, got, stat)
        call need(all(got == keys), 'position 0 is not rotated')

        call cache%create(ctx, 1, 4, 16, 1, 64, stat)
        call need(stat%is_ok(), 'cache create')
        batch%sequences = 1
        batch%rows = 1
        batch%max_rows = 1
        batch%table_pitch = 1
        batch%row_starts = starts
        batch%lengths = lengths
        batch%tables = tables
        call ctx%upload_real(y, values, stat)
        call cache%append(0, batch, HIP_DTYPE_F32, x, 64_c_int64_t, y, 64_c_int64_t, stat)
        call need(stat%is_ok(), 'append')
        call cache%copy_pages([2_c_int32_t], [1_c_int32_t], stat)
        call need(stat%is_ok(), 'copy pages')
        call put(ctx, tables, [1_c_int32_t])
        call cache%attention(0, batch, HIP_DTYPE_F32, x, 64_c_int64_t, 64_c_int64_t, c_null_ptr, 1, 0.125_c_float, 1, y, &
            64_c_int64_t, stat)
        call need(stat%is_ok(), 'attention')
        call ctx%download_real(y, got, stat)
        ! integers up to 127 are codes as they are; fp32 queries give fp32's accuracy
        call need(all(abs(got - values) <= 127.0_c_float * 2.0_c_float**(-20)), 'a single token gives its value')
        call cache%read(0, batch, HIP_DTYPE_F32, x, 64_c_int64_t, y, 64_c_int64_t, stat)
        call ctx%download_real(y, got, stat)
        call need(all(abs(got - values) <= 127.0_c_float * 2.0_c_float**(-22)), 'values read back')
        call cache%attention(1, batch, HIP_DTYPE_F32, x, 64_c_int64_t, 64_c_int64_t, c_null_ptr, 1, 0.125_c_float, 1, y, &
            64_c_int64_t, stat)
        call need(stat%code == FORTAI_INVALID, 'no such layer')

        call verifier%create(ctx, 2, 1, 4, stat)
        call need(stat%is_ok(), 'verifier create')
        logits = room(ctx, 32)
        tokens = room(ctx, 16)
        uniforms = room(ctx, 12)
        quants = room(ctx, 128 * 4 * 36)
        qkv = room(ctx, 3 * 192 * 4)
        temperatures = room(ctx, 4)
        emitted = room(ctx, 16)
        accepted = room(ctx, 4)
        rows = [0.0_c_float, 1.0_c_float, 5.0_c_float, 2.0_c_float, 9.0_c_float, 1.0_c_float, 1.0_c_float, 9.0_c_float]
        call ctx%upload_real(logits, rows, stat)
        call ctx%upload_real(uniforms, [0.5_c_float, 0.5_c_float], stat)
        call ctx%upload_real(temperatures, [0.0_c_float], stat)
        call put(ctx, starts, [0_c_int32_t, 2_c_int32_t])
        call ctx%upload(tokens, transfer([1_c_int64_t, 2_c_int64_t], bytes), 16_c_size_t, stat)
        call verifier%run(HIP_DTYPE_F32, logits, 4_c_int64_t, c_null_ptr, 0_c_int64_t, tokens, uniforms, temperatures, 1, &
            starts, 2, emitted, accepted, c_null_ptr, stat)
        call need(stat%is_ok(), 'verify')
        call ctx%download(emitted, bytes, 16_c_size_t, stat)
        call need(all(transfer(bytes, [0_c_int64_t], 2) == [2_c_int64_t, 0_c_int64_t]), 'the draft stands, then the first largest')
        call ctx%download(accepted, bytes(:4), 4_c_size_t, stat)
        call need(transfer(bytes(:4), 0_c_int32_t) == 1_c_int32_t, 'one draft stands')

        ! the second row's token stands twice in its text; the first row's only once
        call ctx%upload_real(uniforms, [2.0_c_float, 0.5_c_float, 0.25_c_float], stat)
        rules%penalties = uniforms
        rules%tokens = tokens
        call ctx%upload(tokens, transfer([2_c_int64_t, 2_c_int64_t], bytes), 16_c_size_t, stat)
        call hip_logits_adjust(ctx, HIP_DTYPE_F32, logits, 4_c_int64_t, 2, 4, 1, starts, rules, logits, 4_c_int64_t, stat)
        call need(stat%is_ok(), 'rules on logits')
        call ctx%download_real(logits, rows, stat)
        call need(all(rows == [0.0_c_float, 1.0_c_float, 1.75_c_float, 2.0_c_float, 9.0_c_float, 1.0_c_float, -0.75_c_float, &
            9.0_c_float]), 'a token that was there loses')
        call hip_logits_adjust(ctx, HIP_DTYPE_F32, logits, 3_c_int64_t, 2, 4, 1, starts, rules, logits, 4_c_int64_t, stat)
        call need(stat%code == FORTAI_INVALID, 'a pitch below the vocabulary')

        ! codes that are integers: +-127 and whole numbers between them
        call ctx%upload_real(x, values, stat)
        call hip_norm_tokens(ctx, HIP_DTYPE_F32, x, 64_c_int64_t, c_null_ptr, 0_c_int64_t, c_null_ptr, 0_c_int64_t, c_null_ptr, &
            64, 0.0_c_float, c_null_ptr, 0_c_int64_t, 1, 64, c_null_ptr, 0_c_int64_t, quants, stat)
        call need(stat%is_ok(), 'norm into tokens')
        call hip_tokens_read(ctx, HIP_DTYPE_F32, quants, 1, 64, y, 64_c_int64_t, stat)
        call need(stat%is_ok(), 'read tokens')
        call ctx%download_real(y, got, stat)
        call need(all(abs(got - values) <= 0.51_c_float), 'tokens hold their values')
        call hip_norm_tokens(ctx, HIP_DTYPE_F32, x, 64_c_int64_t, c_null_ptr, 0_c_int64_t, c_null_ptr, 0_c_int64_t, c_null_ptr, &
            64, 0.0_c_float, c_null_ptr, 0_c_int64_t, 1, 63, c_null_ptr, 0_c_int64_t, quants, stat)
        call need(stat%code == FORTAI_INVALID, 'half a block')

        ! without keys and values the state stays zero, and so do the outputs
        call states%create(ctx, 1, 2, 1, 1, 64, 2, 0, 1, stat)
        call need(stat%is_ok(), 'states')
        call ctx%upload_real(qkv, [(0.0_c_float, i = 1, 576)], stat)
        state_rows%sequences = 1
        state_rows%rows = 1
        state_rows%max_rows = 1
        state_rows%row_starts = starts
        state_rows%slots = lengths
        call put(ctx, starts, [0_c_int32_t, 1_c_int32_t])
        call put(ctx, lengths, [0_c_int32_t])
        call states%run(0, state_rows, HIP_DTYPE_F32, qkv, 192_c_int64_t, qkv, 1_c_int64_t, qkv, 1_c_int64_t, qkv, qkv, qkv, &
            1.0e-6_c_float, y, 64_c_int64_t, stat)
        call need(stat%is_ok(), 'delta rule')
        call ctx%download_real(y, got, stat)
        call need(all(got == 0.0_c_float), 'zeros in, zeros out')
        call states%copy_slots([0_c_int32_t], [1_c_int32_t], stat)
        call need(stat%is_ok(), 'copy slots')
        call states%run(1, state_rows, HIP_DTYPE_F32, qkv, 192_c_int64_t, qkv, 1_c_int64_t, qkv, 1_c_int64_t, qkv, qkv, qkv, &
            1.0e-6_c_float, y, 64_c_int64_t, stat)
        call need(stat%code == FORTAI_INVALID, 'no such layer of states')

        call states%destroy(stat)
        call verifier%destroy(stat)
        call cache%destroy(stat)
        call rope%destroy(stat)
        call need(stat%is_ok(), 'destroy')
        call ctx%destroy(stat)
        call need(stat%is_ok(), 'context destroy')
    end subroutine gpu_part

    function room(ctx, bytes) result(buffer)
        type(hip_q8_context_t), intent(in) :: ctx
        integer, intent(in) :: bytes
        type(c_ptr) :: buffer

        call ctx%allocate_buffer(int(bytes, c_size_t), buffer, stat)
        call need(stat%is_ok(), 'allocate')
    end function room

    subroutine put(ctx, buffer, numbers)
        type(hip_q8_context_t), intent(in) :: ctx
        type(c_ptr), intent(in) :: buffer
        integer(c_int32_t), intent(in) :: numbers(:)
        integer(c_int8_t) :: bytes(4 * size(numbers))

        bytes = transfer(numbers, bytes)
        call ctx%upload(buffer, bytes, int(size(bytes), c_size_t), stat)
        call need(stat%is_ok(), 'upload')
    end subroutine put

    subroutine need(ok, what)
        logical, intent(in) :: ok
        character(len=*), intent(in) :: what
        if (.not. ok) then
            failures = failures + 1
            print '(a)', 'FAILED: ' // what
            if (allocated(stat%message)) print '(a)', '  status: ' // stat%message
        end if
    end subroutine need

end program hip_serving_smoke
