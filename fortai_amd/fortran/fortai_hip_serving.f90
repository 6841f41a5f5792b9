! fortai_hip_serving.f90 -- the serving operators of libfortai_hip.so from
! Fortran: rotary positions, the 8-bit paged key/value cache with its attention,
! its page bookkeeping, the verification of drafted tokens, the gated delta rule
! over rows, norms into 8-bit tokens and rules on logits.
!
! The reference runs one token of one sequence at a time and has none of these;
! the module keeps the manner of fortai_backend_hip: derived types that hold a
! handle, a status_t for every call, device arrays as c_ptr.  What the arguments
! mean is said at the C entry points (include/fortai_hip_backend.h).
!
! Status contract: a handle that was not created gives FORTAI_INVALID before any
! C call, arguments that the library refuses give FORTAI_INVALID and device
! errors FORTAI_UNSUPPORTED, both with the library's own text where there is a
! context to ask for it.  Destroying a null handle is a no-op.
module fortai_hip_serving
    use, intrinsic :: iso_c_binding, only: c_associated, c_double, c_float, c_int, c_int32_t, c_int64_t, &
        c_null_ptr, c_ptr, c_size_t
    use fortai_status, only: FORTAI_INVALID, FORTAI_UNSUPPORTED, status_t
    use fortai_backend_hip, only: FORTAI_HIP_OK, hip_q8_context_t
    implicit none
    private

    integer, parameter, public :: HIP_DTYPE_F32 = 0, HIP_DTYPE_F16 = 1, HIP_DTYPE_BF16 = 2
    integer, parameter, public :: HIP_ROPE_PLAIN = 0, HIP_ROPE_LINEAR = 1, HIP_ROPE_YARN = 2

    ! fortai_hip_kv8_batch: the rows of a call and where their tokens lie
    type, bind(C), public :: hip_kv8_batch_t
        integer(c_int) :: sequences = 0, rows = 0, max_rows = 0, table_pitch = 0
        type(c_ptr) :: row_starts = c_null_ptr
        type(c_ptr) :: lengths = c_null_ptr
        type(c_ptr) :: tables = c_null_ptr
    end type hip_kv8_batch_t

    ! fortai_hip_kv8_groups: which sequences of a batch share their first pages
    type, bind(C), public :: hip_kv8_groups_t
        integer(c_int) :: groups = 0, max_rows = 0
        type(c_ptr) :: starts = c_null_ptr
        type(c_ptr) :: shared = c_null_ptr
        type(c_ptr) :: group_of = c_null_ptr
    end type hip_kv8_groups_t

    ! fortai_hip_gdn_batch: the rows of a call, whose they are and how many of the last ones stand
    type, bind(C), public :: hip_gdn_batch_t
        integer(c_int) :: sequences = 0, rows = 0, max_rows = 0
        type(c_ptr) :: row_starts = c_null_ptr
        type(c_ptr) :: slots = c_null_ptr
        type(c_ptr) :: standing = c_null_ptr
    end type hip_gdn_batch_t

    ! fortai_hip_logit_rules
    type, bind(C), public :: hip_logit_rules_t
        integer(c_int) :: window = 0, mask_count = 0
        type(c_ptr) :: penalties = c_null_ptr
        type(c_ptr) :: tokens = c_null_ptr
        type(c_ptr) :: history = c_null_ptr
        type(c_ptr) :: history_lengths = c_null_ptr
        type(c_ptr) :: bias = c_null_ptr
        type(c_ptr) :: masks = c_null_ptr
        type(c_ptr) :: mask_of = c_null_ptr
        integer(c_int64_t) :: history_pitch = 0, bias_pitch = 0, mask_pitch = 0
    end type hip_logit_rules_t

    type, public :: hip_rope_t
        type(c_ptr) :: handle = c_null_ptr
        type(hip_q8_context_t) :: context
    contains
        procedure :: create => rope_create
        procedure :: destroy => rope_destroy
        procedure :: apply => rope_apply
    end type hip_rope_t

    type, public :: hip_kv8_cache_t
        type(c_ptr) :: handle = c_null_ptr
        type(hip_q8_context_t) :: context
    contains
        procedure :: create => cache_create
        procedure :: destroy => cache_destroy
        procedure :: append => cache_append
        procedure :: read => cache_read
        procedure :: attention => cache_attention
        procedure :: shared_attention => cache_shared_attention
        procedure :: copy_pages => cache_copy_pages
    end type hip_kv8_cache_t

    type, public :: hip_kv8_pages_t
        type(c_ptr) :: handle = c_null_ptr
    contains
        procedure :: create => pages_create
        procedure :: destroy => pages_destroy
        procedure :: extend => pages_extend
        procedure :: fork => pages_fork
        procedure :: truncate => pages_truncate
        procedure :: compact => pages_compact
        procedure :: length => pages_length
        procedure :: free_count => pages_free_count
        procedure :: tables => pages_tables
        procedure :: groups => pages_groups
    end type hip_kv8_pages_t

    type, public :: hip_verifier_t
        type(c_ptr) :: handle = c_null_ptr
        type(hip_q8_context_t) :: context
    contains
        procedure :: create => verifier_create
        procedure :: destroy => verifier_destroy
        procedure :: run => verifier_run
    end type hip_verifier_t

    type, public :: hip_gdn_cache_t
        type(c_ptr) :: handle = c_null_ptr
        type(hip_q8_context_t) :: context
    contains
        procedure :: create => gdn_create
        procedure :: destroy => gdn_destroy
        procedure :: run => gdn_run
        procedure :: copy_slots => gdn_copy_slots
    end type hip_gdn_cache_t

    public :: hip_kv8_bytes, hip_gdn_bytes, hip_norm_tokens, hip_tokens_read, hip_logits_adjust

    interface
        integer(c_int) function fh_rope_create(context, rope_dimension, interleaved, base, scaling, factor, &
            original_context, beta_fast, beta_slow, attention_factor, rope) bind(C, name='fortai_hip_rope_create')
            import :: c_double, c_int, c_ptr
            type(c_ptr), value :: context
            integer(c_int), value :: rope_dimension, interleaved, scaling, original_context
            real(c_double), value :: base, factor, beta_fast, beta_slow, attention_factor
            type(c_ptr), intent(out) :: rope
        end function fh_rope_create
        integer(c_int) function fh_rope_destroy(rope) bind(C, name='fortai_hip_rope_destroy')
            import :: c_int, c_ptr
            type(c_ptr), value :: rope
        end function fh_rope_destroy
        integer(c_int) function fh_rope(rope, dtype, input, input_row_pitch, input_head_pitch, rows, heads, head_size, &
            positions, norm, epsilon, output, output_row_pitch, output_head_pitch) bind(C, name='fortai_hip_rope_device')
            import :: c_float, c_int, c_int64_t, c_ptr
            type(c_ptr), value :: rope, input, positions, norm, output
            integer(c_int), value :: dtype, rows, heads, head_size
            integer(c_int64_t), value :: input_row_pitch, input_head_pitch, output_row_pitch, output_head_pitch
            real(c_float), value :: epsilon
        end function fh_rope
        integer(c_size_t) function fh_kv8_bytes(layers, pages, page_tokens, kv_heads, head_size) &
            bind(C, name='fortai_hip_kv8_bytes')
            import :: c_int, c_size_t
            integer(c_int), value :: layers, pages, page_tokens, kv_heads, head_size
        end function fh_kv8_bytes
        integer(c_int) function fh_kv8_create(context, layers, pages, page_tokens, kv_heads, head_size, storage, &
            storage_bytes, cache) bind(C, name='fortai_hip_kv8_create')
            import :: c_int, c_ptr, c_size_t
            type(c_ptr), value :: context, storage
            integer(c_int), value :: layers, pages, page_tokens, kv_heads, head_size
            integer(c_size_t), value :: storage_bytes
            type(c_ptr), intent(out) :: cache
        end function fh_kv8_create
        integer(c_int) function fh_kv8_destroy(cache) bind(C, name='fortai_hip_kv8_destroy')
            import :: c_int, c_ptr
            type(c_ptr), value :: cache
        end function fh_kv8_destroy
        integer(c_int) function fh_kv8_append(cache, layer, batch, dtype, keys, key_pitch, values, value_pitch) &
            bind(C, name='fortai_hip_kv8_append_device')
            import :: c_int, c_int64_t, c_ptr, hip_kv8_batch_t
            type(c_ptr), value :: cache, keys, values
            type(hip_kv8_batch_t), intent(in) :: batch
            integer(c_int), value :: layer, dtype
            integer(c_int64_t), value :: key_pitch, value_pitch
        end function fh_kv8_append
        integer(c_int) function fh_kv8_read(cache, layer, batch, dtype, keys, key_pitch, values, value_pitch) &
            bind(C, name='fortai_hip_kv8_read_device')
            import :: c_int, c_int64_t, c_ptr, hip_kv8_batch_t
            type(c_ptr), value :: cache, keys, values
            type(hip_kv8_batch_t), intent(in) :: batch
            integer(c_int), value :: layer, dtype
            integer(c_int64_t), value :: key_pitch, value_pitch
        end function fh_kv8_read
        integer(c_int) function fh_kv8_attention(cache, layer, batch, dtype, query, query_pitch, query_head_pitch, gate, &
            heads, scale, max_length, output, output_pitch) bind(C, name='fortai_hip_kv8_attention_device')
            import :: c_float, c_int, c_int64_t, c_ptr, hip_kv8_batch_t
            type(c_ptr), value :: cache, query, gate, output
            type(hip_kv8_batch_t), intent(in) :: batch
            integer(c_int), value :: layer, dtype, heads, max_length
            integer(c_int64_t), value :: query_pitch, query_head_pitch, output_pitch
            real(c_float), value :: scale
        end function fh_kv8_attention
        integer(c_int) function fh_kv8_shared_attention(cache, layer, batch, sharing, dtype, query, query_pitch, &
            query_head_pitch, gate, heads, scale, max_length, max_shared, output, output_pitch) &
            bind(C, name='fortai_hip_kv8_shared_attention_device')
            import :: c_float, c_int, c_int64_t, c_ptr, hip_kv8_batch_t, hip_kv8_groups_t
            type(c_ptr), value :: cache, query, gate, output
            type(hip_kv8_batch_t), intent(in) :: batch
            type(hip_kv8_groups_t), intent(in) :: sharing
            integer(c_int), value :: layer, dtype, heads, max_length, max_shared
            integer(c_int64_t), value :: query_pitch, query_head_pitch, output_pitch
            real(c_float), value :: scale
        end function fh_kv8_shared_attention
        integer(c_int) function fh_pages_groups(pool, sequences, count, starts, shared, group_of, groups) &
            bind(C, name='fortai_hip_kv8_pages_groups')
            import :: c_int, c_int32_t, c_ptr
            type(c_ptr), value :: pool
            integer(c_int), intent(in) :: sequences(*)
            integer(c_int), value :: count
            integer(c_int32_t), intent(inout) :: starts(*), shared(*), group_of(*)
            integer(c_int32_t), intent(out) :: groups
        end function fh_pages_groups
        integer(c_int) function fh_norm_tokens(context, dtype, x, x_pitch, residual, residual_pitch, total, sum_pitch, norm, &
            group, epsilon, gate, gate_pitch, rows, width, output, output_pitch, tokens) &
            bind(C, name='fortai_hip_norm_tokens_device')
            import :: c_float, c_int, c_int64_t, c_ptr
            type(c_ptr), value :: context, x, residual, total, norm, gate, output, tokens
            integer(c_int), value :: dtype, group, rows, width
            integer(c_int64_t), value :: x_pitch, residual_pitch, sum_pitch, gate_pitch, output_pitch
            real(c_float), value :: epsilon
        end function fh_norm_tokens
        integer(c_int) function fh_tokens_read(context, dtype, tokens, rows, width, output, output_pitch) &
            bind(C, name='fortai_hip_q8_tokens_read_device')
            import :: c_int, c_int64_t, c_ptr
            type(c_ptr), value :: context, tokens, output
            integer(c_int), value :: dtype, rows, width
            integer(c_int64_t), value :: output_pitch
        end function fh_tokens_read
        integer(c_int) function fh_logits_adjust(context, dtype, logits, logits_pitch, rows, vocab, sequences, row_starts, &
            rules, output, output_pitch) bind(C, name='fortai_hip_logits_adjust_device')
            import :: c_int, c_int64_t, c_ptr, hip_logit_rules_t
            type(c_ptr), value :: context, logits, row_starts, output
            type(hip_logit_rules_t), intent(in) :: rules
            integer(c_int), value :: dtype, rows, vocab, sequences
            integer(c_int64_t), value :: logits_pitch, output_pitch
        end function fh_logits_adjust
        integer(c_size_t) function fh_gdn_bytes(layers, slots, key_heads, value_heads, head_size, conv_kernel, pending) &
            bind(C, name='fortai_hip_gdn_bytes')
            import :: c_int, c_size_t
            integer(c_int), value :: layers, slots, key_heads, value_heads, head_size, conv_kernel, pending
        end function fh_gdn_bytes
        integer(c_int) function fh_gdn_create(context, layers, slots, key_heads, value_heads, head_size, conv_kernel, pending, &
            max_rows, storage, storage_bytes, cache) bind(C, name='fortai_hip_gdn_create')
            import :: c_int, c_ptr, c_size_t
            type(c_ptr), value :: context, storage
            integer(c_int), value :: layers, slots, key_heads, value_heads, head_size, conv_kernel, pending, max_rows
            integer(c_size_t), value :: storage_bytes
            type(c_ptr), intent(out) :: cache
        end function fh_gdn_create
        integer(c_int) function fh_gdn_destroy(cache) bind(C, name='fortai_hip_gdn_destroy')
            import :: c_int, c_ptr
            type(c_ptr), value :: cache
        end function fh_gdn_destroy
        integer(c_int) function fh_gdn_run(cache, layer, batch, dtype, qkv, qkv_pitch, alpha, alpha_pitch, beta, beta_pitch, &
            conv, ssm_a, ssm_dt, epsilon, output, output_pitch) bind(C, name='fortai_hip_gdn_run_device')
            import :: c_float, c_int, c_int64_t, c_ptr, hip_gdn_batch_t
            type(c_ptr), value :: cache, qkv, alpha, beta, conv, ssm_a, ssm_dt, output
            type(hip_gdn_batch_t), intent(in) :: batch
            integer(c_int), value :: layer, dtype
            integer(c_int64_t), value :: qkv_pitch, alpha_pitch, beta_pitch, output_pitch
            real(c_float), value :: epsilon
        end function fh_gdn_run
        integer(c_int) function fh_gdn_copy_slots(cache, from, to, count) bind(C, name='fortai_hip_gdn_copy_slots')
            import :: c_int, c_int32_t, c_ptr
            type(c_ptr), value :: cache
            integer(c_int32_t), intent(in) :: from(*), to(*)
            integer(c_int), value :: count
        end function fh_gdn_copy_slots
        integer(c_int) function fh_kv8_copy_pages(cache, from, to, count) bind(C, name='fortai_hip_kv8_copy_pages')
            import :: c_int, c_int32_t, c_ptr
            type(c_ptr), value :: cache
            integer(c_int32_t), intent(in) :: from(*), to(*)
            integer(c_int), value :: count
        end function fh_kv8_copy_pages
        integer(c_int) function fh_pages_create(pages, page_tokens, sequences, table_pitch, pool) &
            bind(C, name='fortai_hip_kv8_pages_create')
            import :: c_int, c_ptr
            integer(c_int), value :: pages, page_tokens, sequences, table_pitch
            type(c_ptr), intent(out) :: pool
        end function fh_pages_create
        integer(c_int) function fh_pages_destroy(pool) bind(C, name='fortai_hip_kv8_pages_destroy')
            import :: c_int, c_ptr
            type(c_ptr), value :: pool
        end function fh_pages_destroy
        integer(c_int) function fh_pages_extend(pool, sequence, tokens, from, to, copies) &
            bind(C, name='fortai_hip_kv8_pages_extend')
            import :: c_int, c_int32_t, c_ptr
            type(c_ptr), value :: pool
            integer(c_int), value :: sequence, tokens
            integer(c_int32_t), intent(inout) :: from, to
            integer(c_int), intent(inout) :: copies
        end function fh_pages_extend
        integer(c_int) function fh_pages_fork(pool, sequence, fork, length) bind(C, name='fortai_hip_kv8_pages_fork')
            import :: c_int, c_int64_t, c_ptr
            type(c_ptr), value :: pool
            integer(c_int), value :: sequence, fork
            integer(c_int64_t), value :: length
        end function fh_pages_fork
        integer(c_int) function fh_pages_truncate(pool, sequence, length) bind(C, name='fortai_hip_kv8_pages_truncate')
            import :: c_int, c_int64_t, c_ptr
            type(c_ptr), value :: pool
            integer(c_int), value :: sequence
            integer(c_int64_t), value :: length
        end function fh_pages_truncate
        integer(c_int) function fh_pages_compact(pool, from, to, capacity, copies) &
            bind(C, name='fortai_hip_kv8_pages_compact')
            import :: c_int, c_int32_t, c_ptr
            type(c_ptr), value :: pool
            integer(c_int32_t), intent(inout) :: from(*), to(*)
            integer(c_int), value :: capacity
            integer(c_int), intent(inout) :: copies
        end function fh_pages_compact
        integer(c_int64_t) function fh_pages_length(pool, sequence) bind(C, name='fortai_hip_kv8_pages_length')
            import :: c_int, c_int64_t, c_ptr
            type(c_ptr), value :: pool
            integer(c_int), value :: sequence
        end function fh_pages_length
        integer(c_int) function fh_pages_free_count(pool) bind(C, name='fortai_hip_kv8_pages_free_count')
            import :: c_int, c_ptr
            type(c_ptr), value :: pool
        end function fh_pages_free_count
        integer(c_int) function fh_pages_tables(pool, sequences, count, tables, table_pitch) &
            bind(C, name='fortai_hip_kv8_pages_tables')
            import :: c_int, c_int32_t, c_ptr
            type(c_ptr), value :: pool
            integer(c_int), intent(in) :: sequences(*)
            integer(c_int), value :: count, table_pitch
            integer(c_int32_t), intent(inout) :: tables(*)
        end function fh_pages_tables
        integer(c_int) function fh_verifier_create(context, max_rows, max_sequences, vocab, verifier) &
            bind(C, name='fortai_hip_verifier_create')
            import :: c_int, c_ptr
            type(c_ptr), value :: context
            integer(c_int), value :: max_rows, max_sequences, vocab
            type(c_ptr), intent(out) :: verifier
        end function fh_verifier_create
        integer(c_int) function fh_verifier_destroy(verifier) bind(C, name='fortai_hip_verifier_destroy')
            import :: c_int, c_ptr
            type(c_ptr), value :: verifier
        end function fh_verifier_destroy
        integer(c_int) function fh_verify(verifier, dtype, target, target_pitch, draft, draft_pitch, tokens, uniforms, &
            temperatures, sequences, row_starts, rows, emitted, accepted, logprobs) &
            bind(C, name='fortai_hip_verify_drafts_device')
            import :: c_int, c_int64_t, c_ptr
            type(c_ptr), value :: verifier, target, draft, tokens, uniforms, temperatures, row_starts, emitted, accepted, &
                logprobs
            integer(c_int), value :: dtype, sequences, rows
            integer(c_int64_t), value :: target_pitch, draft_pitch
        end function fh_verify
    end interface

contains

    ! the status of a C call: 1 is a refused argument, 2 a device error
    subroutine settle(code, context, what, stat)
        integer(c_int), intent(in) :: code
        type(hip_q8_context_t), intent(in) :: context
        character(len=*), intent(in) :: what
        type(status_t), intent(inout) :: stat
        character(len=:), allocatable :: message

        if (code == FORTAI_HIP_OK) return
        message = 'HIP ' // what // ' failed'
        if (c_associated(context%handle)) message = message // ': ' // context%last_error()
        if (code == 1_c_int) then
            call stat%set(FORTAI_INVALID, message)
        else
            call stat%set(FORTAI_UNSUPPORTED, message)
        end if
    end subroutine settle

    ! clears the status; whether the handle may be used, with FORTAI_INVALID if not
    logical function usable(handle, what, stat)
        type(c_ptr), intent(in) :: handle
        character(len=*), intent(in) :: what
        type(status_t), intent(inout) :: stat

        call stat%clear()
        usable = c_associated(handle)
        if (.not. usable) call stat%set(FORTAI_INVALID, 'invalid HIP ' // what)
    end function usable

    type(hip_q8_context_t) function nowhere()
        nowhere%handle = c_null_ptr
    end function nowhere

    ! ---- rotary positions ----

    subroutine rope_create(self, context, rope_dimension, base, stat, interleaved, scaling, factor, original_context, &
        beta_fast, beta_slow, attention_factor)
        class(hip_rope_t), intent(inout) :: self
        type(hip_q8_context_t), intent(in) :: context
        integer, intent(in) :: rope_dimension
        real(c_double), intent(in) :: base
        type(status_t), intent(out) :: stat
        logical, intent(in), optional :: interleaved
        integer, intent(in), optional :: scaling, original_context
        real(c_double), intent(in), optional :: factor, beta_fast, beta_slow, attention_factor
        integer(c_int) :: pairs, kind, original
        real(c_double) :: f, fast, slow, attention

        if (.not. usable(context%handle, 'context', stat)) return
        call self%destroy(stat)
        pairs = 0
        if (present(interleaved)) pairs = merge(1_c_int, 0_c_int, interleaved)
        kind = HIP_ROPE_PLAIN
        if (present(scaling)) kind = int(scaling, c_int)
        original = 0
        if (present(original_context)) original = int(original_context, c_int)
        f = 1.0_c_double
        if (present(factor)) f = factor
        fast = 32.0_c_double
        if (present(beta_fast)) fast = beta_fast
        slow = 1.0_c_double
        if (present(beta_slow)) slow = beta_slow
        attention = 1.0_c_double
        if (present(attention_factor)) attention = attention_factor
        self%context = context
        call settle(fh_rope_create(context%handle, int(rope_dimension, c_int), pairs, base, kind, f, original, fast, slow, &
            attention, self%handle), context, 'rotary position creation', stat)
    end subroutine rope_create

    subroutine rope_destroy(self, stat)
        class(hip_rope_t), intent(inout) :: self
        type(status_t), intent(out) :: stat

        call stat%clear()
        if (.not. c_associated(self%handle)) return
        call settle(fh_rope_destroy(self%handle), self%context, 'rotary position destruction', stat)
        self%handle = c_null_ptr
    end subroutine rope_destroy

    subroutine rope_apply(self, dtype, input, input_row_pitch, input_head_pitch, rows, heads, head_size, positions, norm, &
        epsilon, output, output_row_pitch, output_head_pitch, stat)
        class(hip_rope_t), intent(in) :: self
        integer, intent(in) :: dtype, rows, heads, head_size
        type(c_ptr), intent(in) :: input, positions, norm, output
        integer(c_int64_t), intent(in) :: input_row_pitch, input_head_pitch, output_row_pitch, output_head_pitch
        real(c_float), intent(in) :: epsilon
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, 'rotary positions', stat)) return
        call settle(fh_rope(self%handle, int(dtype, c_int), input, input_row_pitch, input_head_pitch, int(rows, c_int), &
            int(heads, c_int), int(head_size, c_int), positions, norm, epsilon, output, output_row_pitch, &
            output_head_pitch), self%context, 'rotary positions', stat)
    end subroutine rope_apply

    ! ---- the 8-bit cache ----

    ! bytes of a cache's storage; 0 where there is no such cache
    function hip_kv8_bytes(layers, pages, page_tokens, kv_heads, head_size) result(bytes)
        integer, intent(in) :: layers, pages, page_tokens, kv_heads, head_size
        integer(c_size_t) :: bytes

        bytes = fh_kv8_bytes(int(layers, c_int), int(pages, c_int), int(page_tokens, c_int), int(kv_heads, c_int), &
            int(head_size, c_int))
    end function hip_kv8_bytes

    ! over the caller's device storage of storage_bytes, or over storage of its own
    subroutine cache_create(self, context, layers, pages, page_tokens, kv_heads, head_size, stat, storage, storage_bytes)
        class(hip_kv8_cache_t), intent(inout) :: self
        type(hip_q8_context_t), intent(in) :: context
        integer, intent(in) :: layers, pages, page_tokens, kv_heads, head_size
        type(status_t), intent(out) :: stat
        type(c_ptr), intent(in), optional :: storage
        integer(c_size_t), intent(in), optional :: storage_bytes
        type(c_ptr) :: place
        integer(c_size_t) :: bytes

        if (.not. usable(context%handle, 'context', stat)) return
        call self%destroy(stat)
        place = c_null_ptr
        if (present(storage)) place = storage
        bytes = 0_c_size_t
        if (present(storage_bytes)) bytes = storage_bytes
        self%context = context
        call settle(fh_kv8_create(context%handle, int(layers, c_int), int(pages, c_int), int(page_tokens, c_int), &
            int(kv_heads, c_int), int(head_size, c_int), place, bytes, self%handle), context, '8-bit cache creation', stat)
    end subroutine cache_create

    subroutine cache_destroy(self, stat)
        class(hip_kv8_cache_t), intent(inout) :: self
        type(status_t), intent(out) :: stat

        call stat%clear()
        if (.not. c_associated(self%handle)) return
        call settle(fh_kv8_destroy(self%handle), self%context, '8-bit cache destruction', stat)
        self%handle = c_null_ptr
    end subroutine cache_destroy

    ! layers count from 0, as everywhere in the C interface
    subroutine cache_append(self, layer, batch, dtype, keys, key_pitch, values, value_pitch, stat)
        class(hip_kv8_cache_t), intent(in) :: self
        integer, intent(in) :: layer, dtype
        type(hip_kv8_batch_t), intent(in) :: batch
        type(c_ptr), intent(in) :: keys, values
        integer(c_int64_t), intent(in) :: key_pitch, value_pitch
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, '8-bit cache', stat)) return
        call settle(fh_kv8_append(self%handle, int(layer, c_int), batch, int(dtype, c_int), keys, key_pitch, values, &
            value_pitch), self%context, '8-bit cache append', stat)
    end subroutine cache_append

    subroutine cache_read(self, layer, batch, dtype, keys, key_pitch, values, value_pitch, stat)
        class(hip_kv8_cache_t), intent(in) :: self
        integer, intent(in) :: layer, dtype
        type(hip_kv8_batch_t), intent(in) :: batch
        type(c_ptr), intent(in) :: keys, values
        integer(c_int64_t), intent(in) :: key_pitch, value_pitch
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, '8-bit cache', stat)) return
        call settle(fh_kv8_read(self%handle, int(layer, c_int), batch, int(dtype, c_int), keys, key_pitch, values, &
            value_pitch), self%context, '8-bit cache read', stat)
    end subroutine cache_read

    subroutine cache_attention(self, layer, batch, dtype, query, query_pitch, query_head_pitch, gate, heads, scale, &
        max_length, output, output_pitch, stat)
        class(hip_kv8_cache_t), intent(in) :: self
        integer, intent(in) :: layer, dtype, heads, max_length
        type(hip_kv8_batch_t), intent(in) :: batch
        type(c_ptr), intent(in) :: query, gate, output
        integer(c_int64_t), intent(in) :: query_pitch, query_head_pitch, output_pitch
        real(c_float), intent(in) :: scale
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, '8-bit cache', stat)) return
        call settle(fh_kv8_attention(self%handle, int(layer, c_int), batch, int(dtype, c_int), query, query_pitch, &
            query_head_pitch, gate, int(heads, c_int), scale, int(max_length, c_int), output, output_pitch), self%context, &
            '8-bit cache attention', stat)
    end subroutine cache_attention

    ! the tokens of sequences that share their first pages are read once for a group
    subroutine cache_shared_attention(self, layer, batch, sharing, dtype, query, query_pitch, query_head_pitch, gate, heads, &
        scale, max_length, max_shared, output, output_pitch, stat)
        class(hip_kv8_cache_t), intent(in) :: self
        integer, intent(in) :: layer, dtype, heads, max_length, max_shared
        type(hip_kv8_batch_t), intent(in) :: batch
        type(hip_kv8_groups_t), intent(in) :: sharing
        type(c_ptr), intent(in) :: query, gate, output
        integer(c_int64_t), intent(in) :: query_pitch, query_head_pitch, output_pitch
        real(c_float), intent(in) :: scale
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, '8-bit cache', stat)) return
        call settle(fh_kv8_shared_attention(self%handle, int(layer, c_int), batch, sharing, int(dtype, c_int), query, &
            query_pitch, query_head_pitch, gate, int(heads, c_int), scale, int(max_length, c_int), int(max_shared, c_int), &
            output, output_pitch), self%context, '8-bit cache shared attention', stat)
    end subroutine cache_shared_attention

    subroutine cache_copy_pages(self, from, to, stat)
        class(hip_kv8_cache_t), intent(in) :: self
        integer(c_int32_t), intent(in) :: from(:), to(:)
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, '8-bit cache', stat)) return
        if (size(from) /= size(to)) then
            call stat%set(FORTAI_INVALID, 'HIP page copy: as many pages to as from')
            return
        end if
        call settle(fh_kv8_copy_pages(self%handle, from, to, int(size(from), c_int)), self%context, 'page copy', stat)
    end subroutine cache_copy_pages

    ! ---- page bookkeeping (no GPU) ----

    subroutine pages_create(self, pages, page_tokens, sequences, table_pitch, stat)
        class(hip_kv8_pages_t), intent(inout) :: self
        integer, intent(in) :: pages, page_tokens, sequences, table_pitch
        type(status_t), intent(out) :: stat

        call self%destroy(stat)
        call settle(fh_pages_create(int(pages, c_int), int(page_tokens, c_int), int(sequences, c_int), &
            int(table_pitch, c_int), self%handle), nowhere(), 'page pool creation', stat)
    end subroutine pages_create

    subroutine pages_destroy(self, stat)
        class(hip_kv8_pages_t), intent(inout) :: self
        type(status_t), intent(out) :: stat

        call stat%clear()
        if (.not. c_associated(self%handle)) return
        call settle(fh_pages_destroy(self%handle), nowhere(), 'page pool destruction', stat)
        self%handle = c_null_ptr
    end subroutine pages_destroy

    ! copies is 1 where the page `from` has to be copied to `to` before the next append
    subroutine pages_extend(self, sequence, tokens, from, to, copies, stat)
        class(hip_kv8_pages_t), intent(in) :: self
        integer, intent(in) :: sequence, tokens
        integer(c_int32_t), intent(out) :: from, to
        integer, intent(out) :: copies
        type(status_t), intent(out) :: stat
        integer(c_int) :: count

        from = -1
        to = -1
        count = 0
        copies = 0
        if (.not. usable(self%handle, 'page pool', stat)) return
        call settle(fh_pages_extend(self%handle, int(sequence, c_int), int(tokens, c_int), from, to, count), nowhere(), &
            'page pool extension', stat)
        if (stat%is_ok()) copies = int(count)
    end subroutine pages_extend

    subroutine pages_fork(self, sequence, fork, length, stat)
        class(hip_kv8_pages_t), intent(in) :: self
        integer, intent(in) :: sequence, fork
        integer(c_int64_t), intent(in) :: length
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, 'page pool', stat)) return
        call settle(fh_pages_fork(self%handle, int(sequence, c_int), int(fork, c_int), length), nowhere(), &
            'sequence fork', stat)
    end subroutine pages_fork

    subroutine pages_truncate(self, sequence, length, stat)
        class(hip_kv8_pages_t), intent(in) :: self
        integer, intent(in) :: sequence
        integer(c_int64_t), intent(in) :: length
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, 'page pool', stat)) return
        call settle(fh_pages_truncate(self%handle, int(sequence, c_int), length), nowhere(), 'sequence truncation', stat)
    end subroutine pages_truncate

    ! up to size(from) moves; the first `copies` of from and to say which
    subroutine pages_compact(self, from, to, copies, stat)
        class(hip_kv8_pages_t), intent(in) :: self
        integer(c_int32_t), intent(inout) :: from(:), to(:)
        integer, intent(out) :: copies
        type(status_t), intent(out) :: stat
        integer(c_int) :: count

        count = 0
        copies = 0
        if (.not. usable(self%handle, 'page pool', stat)) return
        call settle(fh_pages_compact(self%handle, from, to, int(min(size(from), size(to)), c_int), count), nowhere(), &
            'page pool compaction', stat)
        if (stat%is_ok()) copies = int(count)
    end subroutine pages_compact

    ! -1: no such sequence
    integer(c_int64_t) function pages_length(self, sequence)
        class(hip_kv8_pages_t), intent(in) :: self
        integer, intent(in) :: sequence

        pages_length = -1
        if (c_associated(self%handle)) pages_length = fh_pages_length(self%handle, int(sequence, c_int))
    end function pages_length

    integer function pages_free_count(self)
        class(hip_kv8_pages_t), intent(in) :: self

        pages_free_count = 0
        if (c_associated(self%handle)) pages_free_count = int(fh_pages_free_count(self%handle))
    end function pages_free_count

    ! tables(:, i): the pages of sequences(i), -1 behind the last
    subroutine pages_tables(self, sequences, tables, stat)
        class(hip_kv8_pages_t), intent(in) :: self
        integer(c_int), intent(in) :: sequences(:)
        integer(c_int32_t), intent(inout), contiguous :: tables(:, :)
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, 'page pool', stat)) return
        if (size(tables, 2) < size(sequences)) then
            call stat%set(FORTAI_INVALID, 'HIP page tables: a column for every sequence')
            return
        end if
        call settle(fh_pages_tables(self%handle, sequences, int(size(sequences), c_int), tables, &
            int(size(tables, 1), c_int)), nowhere(), 'page tables', stat)
    end subroutine pages_tables

    ! the groups 0 .. groups - 1 of these sequences, in this order; starts has one more than sequences
    subroutine pages_groups(self, sequences, starts, shared, group_of, groups, stat)
        class(hip_kv8_pages_t), intent(in) :: self
        integer(c_int), intent(in) :: sequences(:)
        integer(c_int32_t), intent(inout) :: starts(:), shared(:), group_of(:)
        integer, intent(out) :: groups
        type(status_t), intent(out) :: stat
        integer(c_int32_t) :: count

        groups = 0
        if (.not. usable(self%handle, 'page pool', stat)) return
        if (size(starts) <= size(sequences) .or. size(shared) < size(sequences) .or. size(group_of) < size(sequences)) then
            call stat%set(FORTAI_INVALID, 'HIP page groups: a place for every sequence, and one more start')
            return
        end if
        call settle(fh_pages_groups(self%handle, sequences, int(size(sequences), c_int), starts, shared, group_of, count), &
            nowhere(), 'page groups', stat)
        if (stat%is_ok()) groups = int(count)
    end subroutine pages_groups

    ! ---- draft verification ----

    subroutine verifier_create(self, context, max_rows, max_sequences, vocab, stat)
        class(hip_verifier_t), intent(inout) :: self
        type(hip_q8_context_t), intent(in) :: context
        integer, intent(in) :: max_rows, max_sequences, vocab
        type(status_t), intent(out) :: stat

        if (.not. usable(context%handle, 'context', stat)) return
        call self%destroy(stat)
        self%context = context
        call settle(fh_verifier_create(context%handle, int(max_rows, c_int), int(max_sequences, c_int), &
            int(vocab, c_int), self%handle), context, 'verifier creation', stat)
    end subroutine verifier_create

    subroutine verifier_destroy(self, stat)
        class(hip_verifier_t), intent(inout) :: self
        type(status_t), intent(out) :: stat

        call stat%clear()
        if (.not. c_associated(self%handle)) return
        call settle(fh_verifier_destroy(self%handle), self%context, 'verifier destruction', stat)
        self%handle = c_null_ptr
    end subroutine verifier_destroy

    ! draft, temperatures and logprobs may be c_null_ptr
    subroutine verifier_run(self, dtype, target, target_pitch, draft, draft_pitch, tokens, uniforms, temperatures, &
        sequences, row_starts, rows, emitted, accepted, logprobs, stat)
        class(hip_verifier_t), intent(in) :: self
        integer, intent(in) :: dtype, sequences, rows
        type(c_ptr), intent(in) :: target, draft, tokens, uniforms, temperatures, row_starts, emitted, accepted, logprobs
        integer(c_int64_t), intent(in) :: target_pitch, draft_pitch
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, 'verifier', stat)) return
        call settle(fh_verify(self%handle, int(dtype, c_int), target, target_pitch, draft, draft_pitch, tokens, uniforms, &
            temperatures, int(sequences, c_int), row_starts, int(rows, c_int), emitted, accepted, logprobs), self%context, &
            'draft verification', stat)
    end subroutine verifier_run

    ! ---- norms into 8-bit tokens ----

    ! residual, total (the sum), norm, gate, output and tokens may be c_null_ptr
    subroutine hip_norm_tokens(context, dtype, x, x_pitch, residual, residual_pitch, total, sum_pitch, norm, group, epsilon, &
        gate, gate_pitch, rows, width, output, output_pitch, tokens, stat)
        type(hip_q8_context_t), intent(in) :: context
        integer, intent(in) :: dtype, group, rows, width
        type(c_ptr), intent(in) :: x, residual, total, norm, gate, output, tokens
        integer(c_int64_t), intent(in) :: x_pitch, residual_pitch, sum_pitch, gate_pitch, output_pitch
        real(c_float), intent(in) :: epsilon
        type(status_t), intent(out) :: stat

        if (.not. usable(context%handle, 'context', stat)) return
        call settle(fh_norm_tokens(context%handle, int(dtype, c_int), x, x_pitch, residual, residual_pitch, total, sum_pitch, &
            norm, int(group, c_int), epsilon, gate, gate_pitch, int(rows, c_int), int(width, c_int), output, output_pitch, &
            tokens), context, 'norm into tokens', stat)
    end subroutine hip_norm_tokens

    subroutine hip_tokens_read(context, dtype, tokens, rows, width, output, output_pitch, stat)
        type(hip_q8_context_t), intent(in) :: context
        integer, intent(in) :: dtype, rows, width
        type(c_ptr), intent(in) :: tokens, output
        integer(c_int64_t), intent(in) :: output_pitch
        type(status_t), intent(out) :: stat

        if (.not. usable(context%handle, 'context', stat)) return
        call settle(fh_tokens_read(context%handle, int(dtype, c_int), tokens, int(rows, c_int), int(width, c_int), output, &
            output_pitch), context, 'reading tokens', stat)
    end subroutine hip_tokens_read

    ! ---- rules on logits ----

    subroutine hip_logits_adjust(context, dtype, logits, logits_pitch, rows, vocab, sequences, row_starts, rules, output, &
        output_pitch, stat)
        type(hip_q8_context_t), intent(in) :: context
        integer, intent(in) :: dtype, rows, vocab, sequences
        type(c_ptr), intent(in) :: logits, row_starts, output
        integer(c_int64_t), intent(in) :: logits_pitch, output_pitch
        type(hip_logit_rules_t), intent(in) :: rules
        type(status_t), intent(out) :: stat

        if (.not. usable(context%handle, 'context', stat)) return
        call settle(fh_logits_adjust(context%handle, int(dtype, c_int), logits, logits_pitch, int(rows, c_int), &
            int(vocab, c_int), int(sequences, c_int), row_starts, rules, output, output_pitch), context, 'rules on logits', &
            stat)
    end subroutine hip_logits_adjust

    ! ---- the gated delta rule over rows ----

    ! 0: no such cache
    integer(c_size_t) function hip_gdn_bytes(layers, slots, key_heads, value_heads, head_size, conv_kernel, pending)
        integer, intent(in) :: layers, slots, key_heads, value_heads, head_size, conv_kernel, pending

        hip_gdn_bytes = fh_gdn_bytes(int(layers, c_int), int(slots, c_int), int(key_heads, c_int), int(value_heads, c_int), &
            int(head_size, c_int), int(conv_kernel, c_int), int(pending, c_int))
    end function hip_gdn_bytes

    ! without storage the cache has its own, cleared
    subroutine gdn_create(self, context, layers, slots, key_heads, value_heads, head_size, conv_kernel, pending, max_rows, &
        stat, storage, storage_bytes)
        class(hip_gdn_cache_t), intent(inout) :: self
        type(hip_q8_context_t), intent(in) :: context
        integer, intent(in) :: layers, slots, key_heads, value_heads, head_size, conv_kernel, pending, max_rows
        type(status_t), intent(out) :: stat
        type(c_ptr), intent(in), optional :: storage
        integer(c_size_t), intent(in), optional :: storage_bytes
        type(c_ptr) :: memory
        integer(c_size_t) :: bytes

        memory = c_null_ptr
        bytes = 0
        if (present(storage)) memory = storage
        if (present(storage_bytes)) bytes = storage_bytes
        if (.not. usable(context%handle, 'context', stat)) return
        call self%destroy(stat)
        self%context = context
        call settle(fh_gdn_create(context%handle, int(layers, c_int), int(slots, c_int), int(key_heads, c_int), &
            int(value_heads, c_int), int(head_size, c_int), int(conv_kernel, c_int), int(pending, c_int), &
            int(max_rows, c_int), memory, bytes, self%handle), context, 'delta rule cache creation', stat)
    end subroutine gdn_create

    subroutine gdn_destroy(self, stat)
        class(hip_gdn_cache_t), intent(inout) :: self
        type(status_t), intent(out) :: stat

        call stat%clear()
        if (.not. c_associated(self%handle)) return
        call settle(fh_gdn_destroy(self%handle), self%context, 'delta rule cache destruction', stat)
        self%handle = c_null_ptr
    end subroutine gdn_destroy

    subroutine gdn_run(self, layer, batch, dtype, qkv, qkv_pitch, alpha, alpha_pitch, beta, beta_pitch, conv, ssm_a, ssm_dt, &
        epsilon, output, output_pitch, stat)
        class(hip_gdn_cache_t), intent(in) :: self
        integer, intent(in) :: layer, dtype
        type(hip_gdn_batch_t), intent(in) :: batch
        type(c_ptr), intent(in) :: qkv, alpha, beta, conv, ssm_a, ssm_dt, output
        integer(c_int64_t), intent(in) :: qkv_pitch, alpha_pitch, beta_pitch, output_pitch
        real(c_float), intent(in) :: epsilon
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, 'delta rule cache', stat)) return
        call settle(fh_gdn_run(self%handle, int(layer, c_int), batch, int(dtype, c_int), qkv, qkv_pitch, alpha, alpha_pitch, &
            beta, beta_pitch, conv, ssm_a, ssm_dt, epsilon, output, output_pitch), self%context, 'delta rule', stat)
    end subroutine gdn_run

    subroutine gdn_copy_slots(self, from, to, stat)
        class(hip_gdn_cache_t), intent(in) :: self
        integer(c_int32_t), intent(in) :: from(:), to(:)
        type(status_t), intent(out) :: stat

        if (.not. usable(self%handle, 'delta rule cache', stat)) return
        if (size(from) /= size(to)) then
            call stat%set(FORTAI_INVALID, 'HIP slot copy: as many slots to as from')
            return
        end if
        call settle(fh_gdn_copy_slots(self%handle, from, to, int(size(from), c_int)), self%context, 'slot copy', stat)
    end subroutine gdn_copy_slots

end module fortai_hip_serving
